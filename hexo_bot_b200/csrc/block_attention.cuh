// Softmax attention of every query over the key blocks it has chosen.
//
//   s_t = scale q . k_t over the live keys t of row i's blocks,
//   p = exp(s - lse), out = sum p_t v_t, lse = log sum exp(s)
//   backward: dv_t += p_t do, ds_t = p_t (do . v_t - do . out),
//             dq = scale sum ds_t k_t, dk_t += scale ds_t q
//
// Neighbouring queries choose different blocks, so a tile of queries shares no
// key block and a query alone fills one row of a matrix instruction. The work
// is turned round: a CTA owns one key block (in shared memory) and a segment
// of the queries, lists the queries that chose the block, and runs them 16
// rows at a time through mma.sync. Each (query, block) pair leaves a partial
// result (max, sum and unnormalised output row in fp32) at the place of the
// block in the query's list; a second kernel joins a row's parts. Nothing is
// added up in an order that varies: results are the same from run to run.
//
// A part is written and read once (8 D bytes a pair against 4 D block flops),
// so for D >= 32 the traffic of the parts is the cost. The host therefore runs
// windows of rows whose parts fit the L2 cache, the buffer of the window
// before being written over while it is still cached.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "block_select.cuh"
#include "ptx.cuh"

namespace sb {

constexpr int kBaMaxTopk = 64;
constexpr int kBaMaxDim = 128;
constexpr int kBaMark = 256;     // queries of a mark word group (8 words)
constexpr int kBaMaxSeg = 4096;  // queries of a segment
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct BaArgs {
  HeadsView q, k, v, o, go, dq, dk, dv;  // o: out (forward: written); go: gradient of out
  float* lse;             // (B, Hq, Sq)
  const int* idx;         // (B, Hkv, Sq, topk)
  const int* kv_lens;
  const int* q_lens;
  uint32_t* bits;         // (B Hkv, marks, nb, 8): bit i of a block's words = query i of the group chose it
  unsigned long long* slots;  // (B Hkv, Sq): bit s = entry s of the row's list counts
  float* part;            // window's parts: [row][topk][dim], row = (local bh * wq + local i) * group + g
  float2* ml;             // forward: [row][topk] (max in log2 units, sum)
  float* delta;           // backward: (B Hkv, Sq, group) do . out
  float* kv_part;         // backward, more than one segment: [bh][nb][nseg][2][block][dim]
  int batch, kv_heads, group, q_rows, kv_rows, dim, nb, block, topk, marks;
  int bh0, nbh;           // window: first (batch, kv head) pair and their count
  int w0, wq;             // window: first query and count (w0 a multiple of kBaMark)
  int seg, nseg;          // queries of a segment, segments of the window
  int seg0, nseg_all;     // backward: index of the window's first segment, segments in all
  float scale, scale_log2;
  uint32_t group_magic;   // ceil(2^32 / group), 0 for group 1
};

__device__ __forceinline__ int ba_kv_len(const BaArgs& a, int b) {
  const int n = a.kv_lens ? a.kv_lens[b] : a.kv_rows;
  return n < 0 ? 0 : n > a.kv_rows ? a.kv_rows : n;
}
__device__ __forceinline__ int ba_q_len(const BaArgs& a, int b) {
  const int n = a.q_lens ? a.q_lens[b] : a.q_rows;
  return n < 0 ? 0 : n > a.q_rows ? a.q_rows : n;
}

// ---- who chose what -----------------------------------------------------------
// One CTA per 256 queries of a (batch, kv head): a bit per (block, query), and
// per query the entries of its list that count (in range, not a repetition).
constexpr int kBaMarkWindow = 1024;  // blocks whose bits are in shared memory at once

__global__ __launch_bounds__(kBaMark) void block_mark_kernel(const BaArgs a) {
  __shared__ uint32_t sm[kBaMarkWindow * 8];
  const int mark = blockIdx.x % a.marks, bh = blockIdx.x / a.marks;
  const int b = bh / a.kv_heads;
  const int i = mark * kBaMark + threadIdx.x;
  const int live = (ba_kv_len(a, b) + a.block - 1) / a.block;
  const bool on = i < ba_q_len(a, b);
  const int* row = a.idx + ((long long)bh * a.q_rows + i) * a.topk;
  unsigned long long counts = 0;
  for (int j0 = 0; j0 < a.nb; j0 += kBaMarkWindow) {
    const int n = a.nb - j0 < kBaMarkWindow ? a.nb - j0 : kBaMarkWindow;
    for (int x = threadIdx.x; x < n * 8; x += kBaMark) sm[x] = 0;
    __syncthreads();
    if (on)
      for (int s = 0; s < a.topk; ++s) {
        const int j = row[s];
        if (j < j0 || j >= j0 + n || j >= live) continue;
        const uint32_t bit = 1u << (threadIdx.x & 31);
        // this thread alone touches its bit, so the old value tells of a repetition
        if (!(atomicOr(&sm[(j - j0) * 8 + (threadIdx.x >> 5)], bit) & bit)) counts |= 1ull << s;
      }
    __syncthreads();
    uint32_t* dst = a.bits + (((long long)bh * a.marks + mark) * a.nb + j0) * 8;
    for (int x = threadIdx.x; x < n * 8; x += kBaMark) dst[x] = sm[x];
    __syncthreads();
  }
  if (i < a.q_rows) a.slots[(long long)bh * a.q_rows + i] = counts;
}

// ---- shared-memory tiles ---------------------------------------------------------
// Rows of DP 16-bit values in 16-byte chunks; the chunk index is XORed with the
// row so that ldmatrix (eight rows of one chunk column) meets every bank once.
template <int DP>
__device__ __forceinline__ uint32_t ba_at(uint32_t base, int row, int chunk) {
  constexpr int CH = DP / 8;
  constexpr int PER = CH >= 8 ? 1 : 8 / CH;  // rows of a 128-byte line
  constexpr int MASK = (CH >= 8 ? 8 : CH) - 1;
  return base + row * (DP * 2) + ((chunk ^ ((row / PER) & MASK)) << 4);
}

// cp.async of `rows` rows (zero past `have` rows and past dim), by `n` threads.
template <typename T, int DP>
__device__ __forceinline__ void ba_load_rows(uint32_t dst, const T* src, long long stride, int rows, int have, int dim,
                                             int t, int n) {
  constexpr int CH = DP / 8;
  for (int x = t; x < rows * CH; x += n) {
    const int r = x / CH, c = x - r * CH;
    const bool ok = r < have && c * 8 < dim;
    cp_async16(ba_at<DP>(dst, r, c), ok ? src + r * stride + c * 8 : src, ok ? 16 : 0);
  }
}

// The listed queries of a segment: ascending indices into list[], returns their
// count. Every thread of the CTA calls it; it ends with a barrier.
template <int THREADS>
__device__ __forceinline__ int ba_list(const BaArgs& a, int bh, int j, int q_first, int q_count, uint16_t* list) {
  __shared__ int warp_sum[THREADS / 32];
  const int words = (q_count + 31) / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t* bits = a.bits + (((long long)bh * a.marks + q_first / kBaMark) * a.nb + j) * 8;
  int total = 0;
  for (int w0 = 0; w0 < words; w0 += THREADS) {
    const int w = w0 + threadIdx.x;
    uint32_t m = 0;
    if (w < words) m = bits[(long long)(w >> 3) * a.nb * 8 + (w & 7)];
    const int mine = __popc(m);
    int pre = mine;
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, pre, d);
      if (lane >= d) pre += o;
    }
    if (lane == 31) warp_sum[warp] = pre;
    __syncthreads();
    int at = total + pre - mine;
    int all = 0;
    for (int x = 0; x < THREADS / 32; ++x) {
      if (x < warp) at += warp_sum[x];
      all += warp_sum[x];
    }
    for (; m; m &= m - 1) list[at++] = (uint16_t)(w * 32 + __ffs(m) - 1);
    total += all;
    __syncthreads();
  }
  return total;
}

// Place of block j in a row's list: its first entry that counts.
__device__ __forceinline__ int ba_slot(const BaArgs& a, long long row, int j) {
  const int* p = a.idx + row * a.topk;
  for (int s = 0; s < a.topk; ++s)
    if (p[s] == j) return s;
  return 0;
}

__device__ __forceinline__ int ba_div_group(const BaArgs& a, int x) {
  return a.group_magic ? (int)__umulhi((uint32_t)x, a.group_magic) : x;
}

// Scores of 16 rows against BK keys, their row maxima and sums, and the output
// rows, all in registers (mma.sync accumulator layout: lane / 4 and + 8 the
// rows, 2 (lane % 4) and + 1 the columns of each 8-wide tile).
template <typename T, int DP, int BK>
struct BaTile {
  float o[DP / 8][4];
  float m[2], l[2];

  __device__ __forceinline__ void run(uint32_t q, uint32_t k, uint32_t v, int live_keys, float scale_log2) {
    const int lane = threadIdx.x & 31;
    float s[BK / 8][4];
#pragma unroll
    for (int n = 0; n < BK / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      uint32_t fa[4];
      ldmatrix_x4(fa, ba_at<DP>(q, lane & 15, 2 * kk + (lane >> 4)));
#pragma unroll
      for (int n = 0; n < BK / 16; ++n) {
        uint32_t fb[4];
        ldmatrix_x4(fb, ba_at<DP>(k, 16 * n + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)));
        const uint32_t b0[2] = {fb[0], fb[1]}, b1[2] = {fb[2], fb[3]};
        MmaTraits<T>::mma(s[2 * n], fa, b0);
        MmaTraits<T>::mma(s[2 * n + 1], fa, b1);
      }
    }
    m[0] = m[1] = -INFINITY;
#pragma unroll
    for (int n = 0; n < BK / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] *= scale_log2;
        if (n * 8 + 2 * (lane & 3) + (e & 1) >= live_keys) s[n][e] = -INFINITY;
      }
#pragma unroll
    for (int n = 0; n < BK / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) m[e >> 1] = fmaxf(m[e >> 1], s[n][e]);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 1));
      m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 2));
      l[r] = 0.f;
    }
    // a row of nothing but -inf scores keeps weight 0
    const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
    for (int n = 0; n < BK / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = exp2f(s[n][e] - (e >> 1 ? m1 : m0));
        l[e >> 1] += s[n][e];
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
    // weights go to the matrix unit in the inputs' 16-bit type (half a step of
    // rounding each, averaged over the keys); their sum l stays in 32 bits
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      const uint32_t fa[4] = {MmaTraits<T>::pack(s[2 * kk][0], s[2 * kk][1]),
                              MmaTraits<T>::pack(s[2 * kk][2], s[2 * kk][3]),
                              MmaTraits<T>::pack(s[2 * kk + 1][0], s[2 * kk + 1][1]),
                              MmaTraits<T>::pack(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        uint32_t fb[4];
        ldmatrix_x4_trans(fb, ba_at<DP>(v, 16 * kk + (lane & 15), 2 * n + (lane >> 4)));
        const uint32_t b0[2] = {fb[0], fb[1]}, b1[2] = {fb[2], fb[3]};
        MmaTraits<T>::mma(o[2 * n], fa, b0);
        MmaTraits<T>::mma(o[2 * n + 1], fa, b1);
      }
    }
  }
};

// ---- forward, many queries -----------------------------------------------------
constexpr int kBaFwdThreads = 128;
constexpr int kBaFwdWarps = kBaFwdThreads / 32;

template <int DP, int BK>
constexpr int ba_fwd_smem() {
  return 2 * BK * DP * 2 + kBaFwdWarps * 2 * 16 * DP * 2 + kBaMaxSeg * 2;
}

template <typename T, int DP, int BK>
__global__ __launch_bounds__(kBaFwdThreads) void block_attn_kernel(const BaArgs a) {
  extern __shared__ __align__(128) char ba_smem[];
  const uint32_t ks = smem_u32(ba_smem), vs = ks + BK * DP * 2;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t qs = vs + BK * DP * 2 + warp * (2 * 16 * DP * 2);
  uint16_t* list = reinterpret_cast<uint16_t*>(ba_smem + 2 * BK * DP * 2 + kBaFwdWarps * 2 * 16 * DP * 2);
  const long long u = blockIdx.x;
  const int sg = (int)(u % a.nseg);
  const int j = (int)((u / a.nseg) % a.nb);
  const int lbh = (int)(u / a.nseg / a.nb), bh = a.bh0 + lbh;
  const int b = bh / a.kv_heads, h = bh - b * a.kv_heads;
  const int q_first = a.w0 + sg * a.seg;
  const int q_count = min(a.seg, a.w0 + a.wq - q_first);
  const int have = min(BK, ba_kv_len(a, b) - j * BK);
  if (have <= 0) return;
  const int n = ba_list<kBaFwdThreads>(a, bh, j, q_first, q_count, list);
  if (n == 0) return;
  const T* kp = (const T*)a.k.p + b * a.k.b + h * a.k.h + (long long)j * BK * a.k.s;
  const T* vp = (const T*)a.v.p + b * a.v.b + h * a.v.h + (long long)j * BK * a.v.s;
  ba_load_rows<T, DP>(ks, kp, a.k.s, BK, have, a.dim, threadIdx.x, kBaFwdThreads);
  ba_load_rows<T, DP>(vs, vp, a.v.s, BK, have, a.dim, threadIdx.x, kBaFwdThreads);
  cp_async_commit();

  const int rows = n * a.group;
  const int G = a.group;
  const T* qp = (const T*)a.q.p + b * a.q.b + (long long)h * G * a.q.h;
  constexpr int CH = DP / 8;
  auto load_q = [&](int tile, uint32_t dst) {
    for (int x = lane; x < 16 * CH; x += 32) {
      const int r = x / CH, c = x - r * CH;
      const int row = tile * 16 + r;
      const bool ok = row < rows && c * 8 < a.dim;
      const T* src = qp;
      if (ok) {
        const int li = ba_div_group(a, row), g = row - li * G;
        src = qp + g * a.q.h + (long long)(q_first + list[li]) * a.q.s + c * 8;
      }
      cp_async16(ba_at<DP>(dst, r, c), src, ok ? 16 : 0);
    }
  };
  const int tiles = (rows + 15) / 16;
  if (warp < tiles) load_q(warp, qs);
  cp_async_commit();
  cp_async_wait<1>();
  __syncthreads();
  int buf = 0;
  for (int t = warp; t < tiles; t += kBaFwdWarps, buf ^= 1) {
    const uint32_t qt = qs + buf * (16 * DP * 2);
    if (t + kBaFwdWarps < tiles) load_q(t + kBaFwdWarps, qs + (buf ^ 1) * (16 * DP * 2));
    cp_async_commit();
    // this lane's two rows: where their parts go
    long long at[2];
    bool ok[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = t * 16 + (lane >> 2) + 8 * r;
      ok[r] = row < rows;
      at[r] = 0;
      if (ok[r]) {
        const int li = ba_div_group(a, row), g = row - li * G;
        const int i = q_first + list[li];
        const int slot = ba_slot(a, (long long)bh * a.q_rows + i, j);
        at[r] = (((long long)lbh * a.wq + (i - a.w0)) * G + g) * a.topk + slot;
      }
    }
    cp_async_wait<1>();
    __syncwarp();
    BaTile<T, DP, BK> tile;
    tile.run(qt, ks, vs, have, a.scale_log2);
    __syncwarp();  // the buffer is free for the tile after next
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (!ok[r]) continue;
      if ((lane & 3) == 0) a.ml[at[r]] = make_float2(tile.m[r], tile.l[r]);
      float* p = a.part + at[r] * a.dim;
#pragma unroll
      for (int nn = 0; nn < DP / 8; ++nn)
        if (nn * 8 < a.dim)
          *reinterpret_cast<float2*>(p + nn * 8 + 2 * (lane & 3)) = make_float2(tile.o[nn][2 * r], tile.o[nn][2 * r + 1]);
    }
  }
}

// Joins the parts of each row: 8 channels a thread.
template <typename T>
__global__ __launch_bounds__(256) void block_attn_join_kernel(const BaArgs a) {
  const int chunks = a.dim / 8;
  const long long total = (long long)a.nbh * a.wq * a.group * chunks;
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  if (x >= total) return;
  const long long row = x / chunks;
  const int c = (int)(x - row * chunks);
  const long long iq = row / a.group;
  const int g = (int)(row - iq * a.group);
  const int lbh = (int)(iq / a.wq), i = a.w0 + (int)(iq - (long long)lbh * a.wq);
  const int bh = a.bh0 + lbh, b = bh / a.kv_heads, h = (bh - b * a.kv_heads) * a.group + g;
  const unsigned long long slots = a.slots[(long long)bh * a.q_rows + i];
  const float2* ml = a.ml + row * a.topk;
  float top = -INFINITY;
  for (unsigned long long m = slots; m; m &= m - 1) top = fmaxf(top, ml[__ffsll(m) - 1].x);
  const float ref = top == -INFINITY ? 0.f : top;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
  for (unsigned long long m = slots; m; m &= m - 1) {
    const int s = __ffsll(m) - 1;
    const float2 p = ml[s];
    const float w = exp2f(p.x - ref);
    sum += w * p.y;
    const float4* src = reinterpret_cast<const float4*>(a.part + (row * a.topk + s) * a.dim + c * 8);
    const float4 u = src[0], v = src[1];
    acc[0] += w * u.x; acc[1] += w * u.y; acc[2] += w * u.z; acc[3] += w * u.w;
    acc[4] += w * v.x; acc[5] += w * v.y; acc[6] += w * v.z; acc[7] += w * v.w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  RotVec<T, 8> y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y.v[e] = rot_cast<T>(acc[e] * inv);
  *reinterpret_cast<RotVec<T, 8>*>((T*)a.o.p + b * a.o.b + h * a.o.h + i * a.o.s + c * 8) = y;
  if (c == 0) a.lse[((long long)b * a.kv_heads * a.group + h) * a.q_rows + i] = (ref + log2f(sum)) * kLn2;
}

// ---- forward, few queries --------------------------------------------------------
// One CTA per (batch, kv head, query): its warps take the row's blocks in turn,
// each with a key block of its own in shared memory, and keep running maxima,
// sums and output rows; the warps' results are joined in shared memory. The
// group's heads are the rows of the 16-row tile.
template <int DP, int BK>
constexpr int ba_few_warps() {
  return DP * BK >= 16384 ? 2 : DP * BK >= 8192 ? 4 : 8;
}
template <int DP, int BK>
constexpr int ba_few_smem() {
  return ba_few_warps<DP, BK>() * (2 * BK * DP * 2) + 16 * DP * 2;
}

template <typename T, int DP, int BK>
__global__ __launch_bounds__(ba_few_warps<DP, BK>() * 32) void block_attn_few_kernel(const BaArgs a) {
  constexpr int W = ba_few_warps<DP, BK>();
  extern __shared__ __align__(128) char ba_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t base = smem_u32(ba_smem);
  const uint32_t ks = base + warp * (2 * BK * DP * 2), vs = ks + BK * DP * 2;
  const uint32_t qs = base + W * (2 * BK * DP * 2);
  __shared__ int chosen[kBaMaxTopk];
  __shared__ int num;
  __shared__ float2 sml[W][16];
  const int G = a.group, gt = (G + 15) / 16;
  const long long u = blockIdx.x;
  const int gi = (int)(u % gt);
  const int i = (int)(u / gt % a.q_rows);
  const int bh = (int)(u / gt / a.q_rows), b = bh / a.kv_heads, h = bh - b * a.kv_heads;
  const int kv = ba_kv_len(a, b), live = (kv + BK - 1) / BK;
  const bool on = i < ba_q_len(a, b);
  const int rows = min(16, G - gi * 16);
  const T* qp = (const T*)a.q.p + b * a.q.b + (long long)(h * G + gi * 16) * a.q.h + (long long)i * a.q.s;
  ba_load_rows<T, DP>(qs, qp, a.q.h, 16, rows, a.dim, threadIdx.x, W * 32);
  cp_async_commit();
  if (warp == 0) {
    const int* row = a.idx + ((long long)bh * a.q_rows + i) * a.topk;
    int n = 0;
    for (int s0 = 0; s0 < a.topk; s0 += 32) {
      const int s = s0 + lane;
      const int j = s < a.topk ? row[s] : -1;
      bool ok = on && j >= 0 && j < live;
      for (int e = 0; e < n; ++e) ok &= chosen[e] != j;  // kept by the 32 before
      const unsigned same = __match_any_sync(0xffffffffu, j);
      ok &= (same & ((1u << lane) - 1u)) == 0;
      const unsigned m = __ballot_sync(0xffffffffu, ok);
      if (ok) chosen[n + __popc(m & ((1u << lane) - 1u))] = j;
      n += __popc(m);
      __syncwarp();
    }
    if (lane == 0) num = n;
  }
  cp_async_wait_all();
  __syncthreads();
  const int n = num;
  float o[DP / 8][4];
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
  for (int x = 0; x < DP / 8; ++x)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[x][e] = 0.f;
  for (int c = warp; c < n; c += W) {
    const int j = chosen[c];
    const int have = min(BK, kv - j * BK);
    const T* kp = (const T*)a.k.p + b * a.k.b + h * a.k.h + (long long)j * BK * a.k.s;
    const T* vp = (const T*)a.v.p + b * a.v.b + h * a.v.h + (long long)j * BK * a.v.s;
    ba_load_rows<T, DP>(ks, kp, a.k.s, BK, have, a.dim, lane, 32);
    ba_load_rows<T, DP>(vs, vp, a.v.s, BK, have, a.dim, lane, 32);
    cp_async_wait_all();
    __syncwarp();
    BaTile<T, DP, BK> tile;
    tile.run(qs, ks, vs, have, a.scale_log2);
    __syncwarp();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float t = fmaxf(top[r], tile.m[r]);
      const float ref = t == -INFINITY ? 0.f : t;
      const float wo = exp2f(top[r] - ref), wn = exp2f(tile.m[r] - ref);
      top[r] = t;
      sum[r] = sum[r] * wo + tile.l[r] * wn;
#pragma unroll
      for (int x = 0; x < DP / 8; ++x) {
        o[x][2 * r] = o[x][2 * r] * wo + tile.o[x][2 * r] * wn;
        o[x][2 * r + 1] = o[x][2 * r + 1] * wo + tile.o[x][2 * r + 1] * wn;
      }
    }
  }
  // join over the warps: parts in the key buffers (16 x DP fp32 each)
  __syncthreads();
  float* mine = reinterpret_cast<float*>(ba_smem) + warp * (16 * DP);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = (lane >> 2) + 8 * r;
    if ((lane & 3) == 0) sml[warp][row] = make_float2(top[r], sum[r]);
#pragma unroll
    for (int x = 0; x < DP / 8; ++x)
      *reinterpret_cast<float2*>(mine + row * DP + x * 8 + 2 * (lane & 3)) = make_float2(o[x][2 * r], o[x][2 * r + 1]);
  }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(ba_smem);
  for (int x = threadIdx.x; x < rows * a.dim; x += W * 32) {
    const int row = x / a.dim, d = x - row * a.dim;
    float t = -INFINITY;
    for (int w = 0; w < W; ++w) t = fmaxf(t, sml[w][row].x);
    const float ref = t == -INFINITY ? 0.f : t;
    float acc = 0.f, s = 0.f;
    for (int w = 0; w < W; ++w) {
      const float f = exp2f(sml[w][row].x - ref);
      s += f * sml[w][row].y;
      acc += f * all[w * (16 * DP) + row * DP + d];
    }
    const int hq = h * G + gi * 16 + row;
    ((T*)a.o.p)[b * a.o.b + hq * a.o.h + i * a.o.s + d] = rot_cast<T>(s == 0.f ? 0.f : acc / s);
    if (d == 0) a.lse[((long long)b * a.kv_heads * G + hq) * a.q_rows + i] = (ref + log2f(s)) * kLn2;
  }
}

// ---- backward --------------------------------------------------------------------
// delta = do . out of every row, 8 channels a lane.
template <typename T>
__global__ __launch_bounds__(256) void block_attn_delta_kernel(const BaArgs a) {
  const int chunks = a.dim / 8;
  int lanes = 1;
  while (lanes < chunks) lanes <<= 1;
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = x / lanes;
  const int c = (int)(x - row * lanes);
  const long long rows = (long long)a.batch * a.kv_heads * a.q_rows * a.group;
  float s = 0.f;
  if (row < rows && c < chunks) {
    const long long iq = row / a.group;
    const int g = (int)(row - iq * a.group);
    const long long bh = iq / a.q_rows;
    const int i = (int)(iq - bh * a.q_rows), b = (int)(bh / a.kv_heads);
    const int h = (int)(bh - (long long)b * a.kv_heads) * a.group + g;
    if (i < ba_q_len(a, b)) {
      const RotVec<T, 8> u = *reinterpret_cast<const RotVec<T, 8>*>((const T*)a.o.p + b * a.o.b + h * a.o.h + i * a.o.s + c * 8);
      const RotVec<T, 8> v = *reinterpret_cast<const RotVec<T, 8>*>((const T*)a.go.p + b * a.go.b + h * a.go.h + i * a.go.s + c * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += rot_f32(u.v[e]) * rot_f32(v.v[e]);
    }
  }
  for (int m = 1; m < lanes; m <<= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
  if (row < rows && c == 0) a.delta[row] = s;
}

// One CTA per (segment, key block): BK / 16 warps, each owning 16 keys and
// their dk, dv rows in registers over all listed rows. Row tiles of TR rows
// pass through shared memory; scores are computed transposed (keys x rows), so
// that p and ds are the left operands of dv += p do and dk += ds q without
// leaving the registers; ds also goes through shared memory, from where the
// warps form dq = ds k, a part of each (row, block) pair as in the forward.
template <int DP>
constexpr int ba_bwd_rows() {
  return DP == 128 ? 32 : 64;
}
template <int DP, int BK>
constexpr int ba_bwd_smem() {
  constexpr int TR = ba_bwd_rows<DP>();
  return 2 * BK * DP * 2 + 2 * 2 * TR * DP * 2 + BK * TR * 2 + 2 * TR * 16 + kBaMaxSeg * 2;
}

template <typename T, int DP, int BK>
__global__ __launch_bounds__(BK * 2) void block_attn_bwd_kernel(const BaArgs a) {
  constexpr int NW = BK / 16, THREADS = NW * 32, TR = ba_bwd_rows<DP>();
  constexpr int TILE = TR * DP * 2;
  extern __shared__ __align__(128) char ba_smem[];
  const uint32_t ks = smem_u32(ba_smem), vs = ks + BK * DP * 2;
  const uint32_t qs = vs + BK * DP * 2;        // [2][TR][DP]
  const uint32_t gs = qs + 2 * TILE;           // [2][TR][DP]
  const uint32_t ds = gs + 2 * TILE;           // [BK][TR]
  char* tail = ba_smem + 2 * BK * DP * 2 + 4 * TILE + BK * TR * 2;
  // per row of a tile: (lse in log2 units, delta) and where its dq part goes
  float2* stat = reinterpret_cast<float2*>(tail);                    // [2][TR]
  long long* dst = reinterpret_cast<long long*>(tail + 2 * TR * 8);  // [2][TR]
  uint16_t* list = reinterpret_cast<uint16_t*>(tail + 2 * TR * 16);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long u = blockIdx.x;
  const int sg = (int)(u % a.nseg);
  const int j = (int)((u / a.nseg) % a.nb);
  const int lbh = (int)(u / a.nseg / a.nb), bh = a.bh0 + lbh;
  const int b = bh / a.kv_heads, h = bh - b * a.kv_heads;
  const int q_first = a.w0 + sg * a.seg;
  const int q_count = min(a.seg, a.w0 + a.wq - q_first);
  const int G = a.group;
  const int have = max(0, min(BK, ba_kv_len(a, b) - j * BK));
  const int n = ba_list<THREADS>(a, bh, j, q_first, q_count, list);
  const int rows = n * G;
  const T* kp = (const T*)a.k.p + b * a.k.b + h * a.k.h + (long long)j * BK * a.k.s;
  const T* vp = (const T*)a.v.p + b * a.v.b + h * a.v.h + (long long)j * BK * a.v.s;
  if (n > 0) {
    ba_load_rows<T, DP>(ks, kp, a.k.s, BK, have, a.dim, threadIdx.x, THREADS);
    ba_load_rows<T, DP>(vs, vp, a.v.s, BK, have, a.dim, threadIdx.x, THREADS);
  }
  const T* qp = (const T*)a.q.p + b * a.q.b + (long long)h * G * a.q.h;
  const T* gp = (const T*)a.go.p + b * a.go.b + (long long)h * G * a.go.h;
  constexpr int CH = DP / 8;
  auto load_tile = [&](int t, int buf) {
    for (int x = threadIdx.x; x < TR * CH; x += THREADS) {
      const int r = x / CH, c = x - r * CH;
      const int row = t * TR + r;
      const bool ok = row < rows && c * 8 < a.dim;
      const T *sq = qp, *sgr = gp;
      if (ok) {
        const int li = ba_div_group(a, row), g = row - li * G;
        const long long i = q_first + list[li];
        sq = qp + g * a.q.h + i * a.q.s + c * 8;
        sgr = gp + g * a.go.h + i * a.go.s + c * 8;
      }
      cp_async16(ba_at<DP>(qs + buf * TILE, r, c), sq, ok ? 16 : 0);
      cp_async16(ba_at<DP>(gs + buf * TILE, r, c), sgr, ok ? 16 : 0);
    }
    for (int r = threadIdx.x; r < TR; r += THREADS) {
      const int row = t * TR + r;
      float2 st = make_float2(INFINITY, 0.f);  // rows that are not there: weight 0
      long long to = -1;
      if (row < rows) {
        const int li = ba_div_group(a, row), g = row - li * G;
        const int i = q_first + list[li];
        const long long qrow = (long long)bh * a.q_rows + i;
        // a row all of whose scores are -inf has no weights
        const float l = a.lse[((long long)b * a.kv_heads * G + h * G + g) * a.q_rows + i];
        st = make_float2(l == -INFINITY ? INFINITY : l * kLog2e, a.delta[qrow * G + g]);
        to = (((long long)lbh * a.wq + (i - a.w0)) * G + g) * a.topk + ba_slot(a, qrow, j);
      }
      stat[buf * TR + r] = st;
      dst[buf * TR + r] = to;
    }
  };
  float dk[DP / 8][4], dv[DP / 8][4];
#pragma unroll
  for (int x = 0; x < DP / 8; ++x)
#pragma unroll
    for (int e = 0; e < 4; ++e) dk[x][e] = dv[x][e] = 0.f;
  const int tiles = (rows + TR - 1) / TR;
  if (tiles > 0) load_tile(0, 0);
  cp_async_commit();
  const int k0 = warp * 16;
  const bool live0 = k0 + (lane >> 2) < have, live1 = k0 + (lane >> 2) + 8 < have;
  for (int t = 0; t < tiles; ++t) {
    const int buf = t & 1;
    if (t + 1 < tiles) load_tile(t + 1, buf ^ 1);
    cp_async_commit();
    cp_async_wait<1>();
    __syncthreads();
    const uint32_t qt = qs + buf * TILE, gt = gs + buf * TILE;
    float s[TR / 8][4], dp[TR / 8][4];
#pragma unroll
    for (int x = 0; x < TR / 8; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[x][e] = dp[x][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      uint32_t fk[4], fv[4];
      ldmatrix_x4(fk, ba_at<DP>(ks, k0 + (lane & 15), 2 * kk + (lane >> 4)));
      ldmatrix_x4(fv, ba_at<DP>(vs, k0 + (lane & 15), 2 * kk + (lane >> 4)));
#pragma unroll
      for (int x = 0; x < TR / 16; ++x) {
        uint32_t f[4];
        ldmatrix_x4(f, ba_at<DP>(qt, 16 * x + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)));
        const uint32_t b0[2] = {f[0], f[1]}, b1[2] = {f[2], f[3]};
        MmaTraits<T>::mma(s[2 * x], fk, b0);
        MmaTraits<T>::mma(s[2 * x + 1], fk, b1);
        ldmatrix_x4(f, ba_at<DP>(gt, 16 * x + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)));
        const uint32_t c0[2] = {f[0], f[1]}, c1[2] = {f[2], f[3]};
        MmaTraits<T>::mma(dp[2 * x], fv, c0);
        MmaTraits<T>::mma(dp[2 * x + 1], fv, c1);
      }
    }
    // p = 2^(s - lse), ds = p (dp - delta): columns are rows of the tile
#pragma unroll
    for (int x = 0; x < TR / 8; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 st = stat[buf * TR + 8 * x + 2 * (lane & 3) + (e & 1)];
        const bool live = e >> 1 ? live1 : live0;
        s[x][e] = live ? exp2f(s[x][e] * a.scale_log2 - st.x) : 0.f;
        dp[x][e] = live ? s[x][e] * (dp[x][e] - st.y) : 0.f;
      }
    // p and ds are rounded to the inputs' type for the matrix unit (as the
    // forward rounds p); their products are added in 32 bits
    uint32_t fp[TR / 16][4], fd[TR / 16][4];
#pragma unroll
    for (int x = 0; x < TR / 16; ++x) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        fp[x][2 * hf] = MmaTraits<T>::pack(s[2 * x + hf][0], s[2 * x + hf][1]);
        fp[x][2 * hf + 1] = MmaTraits<T>::pack(s[2 * x + hf][2], s[2 * x + hf][3]);
        fd[x][2 * hf] = MmaTraits<T>::pack(dp[2 * x + hf][0], dp[2 * x + hf][1]);
        fd[x][2 * hf + 1] = MmaTraits<T>::pack(dp[2 * x + hf][2], dp[2 * x + hf][3]);
        // ds to shared memory as [key][row]
        const uint32_t a0 = ba_at<TR>(ds, k0 + (lane >> 2), 2 * x + hf) + 4 * (lane & 3);
        const uint32_t a1 = ba_at<TR>(ds, k0 + (lane >> 2) + 8, 2 * x + hf) + 4 * (lane & 3);
        asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(a0), "r"(fd[x][2 * hf]) : "memory");
        asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(a1), "r"(fd[x][2 * hf + 1]) : "memory");
      }
    }
#pragma unroll
    for (int x = 0; x < TR / 16; ++x)
#pragma unroll
      for (int nn = 0; nn < DP / 16; ++nn) {
        uint32_t f[4];
        ldmatrix_x4_trans(f, ba_at<DP>(gt, 16 * x + (lane & 15), 2 * nn + (lane >> 4)));
        const uint32_t b0[2] = {f[0], f[1]}, b1[2] = {f[2], f[3]};
        MmaTraits<T>::mma(dv[2 * nn], fp[x], b0);
        MmaTraits<T>::mma(dv[2 * nn + 1], fp[x], b1);
        ldmatrix_x4_trans(f, ba_at<DP>(qt, 16 * x + (lane & 15), 2 * nn + (lane >> 4)));
        const uint32_t c0[2] = {f[0], f[1]}, c1[2] = {f[2], f[3]};
        MmaTraits<T>::mma(dk[2 * nn], fd[x], c0);
        MmaTraits<T>::mma(dk[2 * nn + 1], fd[x], c1);
      }
    __syncthreads();
    // dq parts: units of 16 rows x 16 channels, spread over the warps
    for (int unit = warp; unit < (TR / 16) * (DP / 16); unit += NW) {
      const int mt = unit % (TR / 16), nt = unit / (TR / 16);
      if (nt * 16 >= a.dim || t * TR + mt * 16 >= rows) continue;
      float acc[2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[x][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < BK / 16; ++kk) {
        uint32_t fa[4], fb[4];
        ldmatrix_x4_trans(fa, ba_at<TR>(ds, 16 * kk + (lane & 7) + ((lane >> 4) << 3), 2 * mt + ((lane >> 3) & 1)));
        ldmatrix_x4_trans(fb, ba_at<DP>(ks, 16 * kk + (lane & 15), 2 * nt + (lane >> 4)));
        const uint32_t b0[2] = {fb[0], fb[1]}, b1[2] = {fb[2], fb[3]};
        MmaTraits<T>::mma(acc[0], fa, b0);
        MmaTraits<T>::mma(acc[1], fa, b1);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const long long to = dst[buf * TR + mt * 16 + (lane >> 2) + 8 * r];
        if (to < 0) continue;
        float* p = a.part + to * a.dim + nt * 16 + 2 * (lane & 3);
        *reinterpret_cast<float2*>(p) = make_float2(acc[0][2 * r], acc[0][2 * r + 1]);
        if (nt * 16 + 8 < a.dim) *reinterpret_cast<float2*>(p + 8) = make_float2(acc[1][2 * r], acc[1][2 * r + 1]);
      }
    }
    __syncthreads();  // ds, the tile and its stats are written over from here on
  }
  cp_async_wait_all();
  // keys of this block: final rows, or this segment's part
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int key = k0 + (lane >> 2) + 8 * r;
    if (a.nseg_all > 1) {
      float* p = a.kv_part + ((((long long)bh * a.nb + j) * a.nseg_all + a.seg0 + sg) * 2 * BK + key) * a.dim;
#pragma unroll
      for (int x = 0; x < DP / 8; ++x)
        if (x * 8 < a.dim) {
          *reinterpret_cast<float2*>(p + x * 8 + 2 * (lane & 3)) = make_float2(dk[x][2 * r], dk[x][2 * r + 1]);
          *reinterpret_cast<float2*>(p + (long long)BK * a.dim + x * 8 + 2 * (lane & 3)) =
              make_float2(dv[x][2 * r], dv[x][2 * r + 1]);
        }
    } else if (j * BK + key < a.kv_rows) {
      T* pk = (T*)a.dk.p + b * a.dk.b + h * a.dk.h + (long long)(j * BK + key) * a.dk.s;
      T* pv = (T*)a.dv.p + b * a.dv.b + h * a.dv.h + (long long)(j * BK + key) * a.dv.s;
#pragma unroll
      for (int x = 0; x < DP / 8; ++x)
        if (x * 8 < a.dim) {
          *reinterpret_cast<uint32_t*>(pk + x * 8 + 2 * (lane & 3)) =
              MmaTraits<T>::pack(dk[x][2 * r] * a.scale, dk[x][2 * r + 1] * a.scale);
          *reinterpret_cast<uint32_t*>(pv + x * 8 + 2 * (lane & 3)) = MmaTraits<T>::pack(dv[x][2 * r], dv[x][2 * r + 1]);
        }
    }
  }
}

// dq of the window: the sum of each row's parts.
template <typename T>
__global__ __launch_bounds__(256) void block_attn_dq_kernel(const BaArgs a) {
  const int chunks = a.dim / 8;
  const long long total = (long long)a.nbh * a.wq * a.group * chunks;
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  if (x >= total) return;
  const long long row = x / chunks;
  const int c = (int)(x - row * chunks);
  const long long iq = row / a.group;
  const int g = (int)(row - iq * a.group);
  const int lbh = (int)(iq / a.wq), i = a.w0 + (int)(iq - (long long)lbh * a.wq);
  const int bh = a.bh0 + lbh, b = bh / a.kv_heads, h = (bh - b * a.kv_heads) * a.group + g;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (unsigned long long m = a.slots[(long long)bh * a.q_rows + i]; m; m &= m - 1) {
    const float4* src = reinterpret_cast<const float4*>(a.part + (row * a.topk + __ffsll(m) - 1) * a.dim + c * 8);
    const float4 u = src[0], v = src[1];
    acc[0] += u.x; acc[1] += u.y; acc[2] += u.z; acc[3] += u.w;
    acc[4] += v.x; acc[5] += v.y; acc[6] += v.z; acc[7] += v.w;
  }
  RotVec<T, 8> y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y.v[e] = rot_cast<T>(acc[e] * a.scale);
  *reinterpret_cast<RotVec<T, 8>*>((T*)a.dq.p + b * a.dq.b + h * a.dq.h + i * a.dq.s + c * 8) = y;
}

// dk, dv: the sum of the segments' parts, in segment order.
template <typename T>
__global__ __launch_bounds__(256) void block_attn_dkv_kernel(const BaArgs a) {
  const int chunks = a.dim / 8;
  const long long total = (long long)a.batch * a.kv_heads * a.kv_rows * chunks;
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  if (x >= total) return;
  const long long row = x / chunks;
  const int c = (int)(x - row * chunks);
  const int bh = (int)(row / a.kv_rows), t = (int)(row - (long long)bh * a.kv_rows);
  const int b = bh / a.kv_heads, h = bh - b * a.kv_heads;
  const int j = t / a.block, key = t - j * a.block;
  const long long step = 2ll * a.block * a.dim;
  const float* p = a.kv_part + ((long long)bh * a.nb + j) * a.nseg_all * step + (long long)key * a.dim + c * 8;
  float acc[2][8] = {};
  for (int s = 0; s < a.nseg_all; ++s, p += step)
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const float4* src = reinterpret_cast<const float4*>(p + (long long)w * a.block * a.dim);
      const float4 u = src[0], v = src[1];
      acc[w][0] += u.x; acc[w][1] += u.y; acc[w][2] += u.z; acc[w][3] += u.w;
      acc[w][4] += v.x; acc[w][5] += v.y; acc[w][6] += v.z; acc[w][7] += v.w;
    }
  RotVec<T, 8> yk, yv;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    yk.v[e] = rot_cast<T>(acc[0][e] * a.scale);
    yv.v[e] = rot_cast<T>(acc[1][e]);
  }
  *reinterpret_cast<RotVec<T, 8>*>((T*)a.dk.p + b * a.dk.b + h * a.dk.h + (long long)t * a.dk.s + c * 8) = yk;
  *reinterpret_cast<RotVec<T, 8>*>((T*)a.dv.p + b * a.dv.b + h * a.dv.h + (long long)t * a.dv.s + c * 8) = yv;
}

}  // namespace sb
