// Softmax attention of every query over the key blocks it has chosen.
//
//   s_t = scale q . k_t over the live keys t of row i's blocks,
//   p = exp(s - lse), out = sum p_t v_t, lse = log sum exp(s)
//   backward: dv_t += p_t do, ds_t = p_t (do . v_t - do . out),
//             dq = scale sum ds_t k_t, dk_t += scale ds_t q
//
// Neighbouring queries need not choose the same blocks: a tile of queries may share
// no key block, and a query alone fills one row of a matrix instruction. The work
// is turned round: a work item is one key block (in shared memory) and a segment
// of the queries; its CTA lists the queries that chose the block and runs them in
// tiles of 128 rows through the tensor cores. Each (query, block) pair leaves a partial
// result (max, sum and unnormalised output row in fp32) at the place of the
// block in the query's list; a second kernel joins a row's parts. Nothing is
// added up in an order that varies: results are the same from run to run.
//
// A part is written and read once: 8 D bytes a pair against 4 D block flops,
// five times as long at HBM's rate as the products at the tensor cores' (D = 64,
// block 64): the parts and the chain of a tile's steps bound the kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "block_select.cuh"
#include "ptx.cuh"

namespace sb {

constexpr int kBaMaxTopk = 64;
constexpr int kBaMaxDim = 128;
constexpr int kBaMark = 256;    // queries of a list group
constexpr int kBaChunk = 1024;  // listed queries that a CTA holds at once
constexpr int kBaJoinThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct BaArgs {
  HeadsView q, k, v, o, go, dq, dk, dv;  // o: out (forward: written); go: gradient of out
  float* lse;             // (B, Hq, Sq)
  const int* idx;         // (B, Hkv, Sq, topk)
  const int* kv_lens;
  const int* q_lens;
  uint16_t* entries;      // window's (local bh, marks, kBaMark topk): per group, by block: place in the row's list << 8 | query
  uint32_t* spans;        // (local bh, nb, marks): first entry of the group's queries that chose the block | count << 16
  uint32_t* ticket;       // work items that the persistent CTAs have taken; 0 before each launch
  unsigned long long* slots;  // (B Hkv, Sq): bit s = entry s of the row's list counts
  float* part;            // window's parts: [row][topk][dim], row = (local bh * wq + local i) * group + g
  float2* ml;             // forward: [row][topk] (max in log2 units, sum)
  float2* delta;          // backward: (B Hkv, Sq, group) do . out, and the norm of do (f16 alone reads it)
  float* kv_part;         // backward, more than one segment or window: [local bh][nb][sums][2][block][dim]
  int batch, kv_heads, group, q_rows, kv_rows, dim, nb, block, topk;
  int marks;              // list groups of a full window
  int bh0, nbh;           // window: first (batch, kv head) pair and their count
  int w0, wq;             // window: first query and count (w0 a multiple of kBaMark)
  int seg, nseg;          // list groups of a segment, segments of the window
  int sums;               // backward: sums of dk and dv that a block has, one a segment; 0: results at once
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
// One CTA per 256 queries of a window's (batch, kv head) turns their lists round:
// for every block the queries that chose it, ascending, with the place of the block
// in each query's list. A bit per (block, query) in shared memory counts and
// orders them (a counting sort whose result no scheduling changes) and shows
// repeated entries: `slots` marks the entries that count.
constexpr int kBaListWindow = 1024;  // blocks whose bits are in shared memory at once

__host__ __device__ inline int ba_list_window(int nb) { return nb < kBaListWindow ? (nb + 3) / 4 * 4 : kBaListWindow; }
__host__ __device__ inline int ba_list_smem(int nb, int topk) {
  return ba_list_window(nb) * 8 * (4 + 2) + kBaMark * topk * 2;
}

// KR: entries of a list that a thread holds in registers (topk <= KR).
template <int KR>
__global__ __launch_bounds__(kBaMark) void block_list_kernel(const BaArgs a) {
  extern __shared__ __align__(16) char list_smem[];
  const int W = ba_list_window(a.nb), K = a.topk;
  uint32_t* bits = reinterpret_cast<uint32_t*>(list_smem);       // [8][W]
  uint16_t* offs = reinterpret_cast<uint16_t*>(bits + 8 * W);    // [8][W]: first entry of a word's queries
  uint16_t* sorted = offs + 8 * W;                               // [256 topk]
  __shared__ uint32_t warp_sum[kBaMark / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int marks = (a.wq + kBaMark - 1) / kBaMark;
  const int lbh = blockIdx.x / marks, mark = blockIdx.x - lbh * marks, bh = a.bh0 + lbh;
  const int b = bh / a.kv_heads;
  const int i = a.w0 + mark * kBaMark + tid;
  const bool on = i < a.w0 + a.wq;
  const int* src = a.idx + ((long long)bh * a.q_rows + i) * K;
  int e[KR];
#pragma unroll
  for (int s = 0; s < KR; ++s) e[s] = on && s < K ? src[s] : -1;
  const int live = i < ba_q_len(a, b) ? (ba_kv_len(a, b) + a.block - 1) / a.block : 0;
  // lists as block_select writes them ascend; in any other a block may be named twice
  bool ascends = true;
  int last = -1;
#pragma unroll
  for (int s = 0; s < KR; ++s) {
    if (e[s] < 0 || e[s] >= live) {
      e[s] = -1;
    } else {
      ascends = ascends && e[s] > last;
      last = e[s];
    }
  }
  uint32_t base = 0;
  const uint32_t bit = 1u << lane;
  for (int j0 = 0; j0 < a.nb; j0 += W) {
    const int n = min(a.nb - j0, W), n4 = W / 4;
    for (int x = tid; x < 8 * n4; x += kBaMark) reinterpret_cast<uint4*>(bits)[x] = uint4{};
    __syncthreads();
    if (ascends) {
#pragma unroll
      for (int s = 0; s < KR; ++s)
        if (e[s] >= j0 && e[s] < j0 + n) atomicOr(&bits[warp * W + e[s] - j0], bit);
    } else {
      // this thread alone touches its bit, so the old value tells of a repetition
#pragma unroll
      for (int s = 0; s < KR; ++s)
        if (e[s] >= j0 && e[s] < j0 + n && (atomicOr(&bits[warp * W + e[s] - j0], bit) & bit)) e[s] = -1;
    }
    __syncthreads();
    // four blocks a thread: counts, and their exclusive sums over the window
    uint32_t c[8][4], sum[4] = {0, 0, 0, 0}, total = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const uint4 v = tid < n4 ? reinterpret_cast<const uint4*>(bits + w * W)[tid] : uint4{};
      c[w][0] = __popc(v.x); c[w][1] = __popc(v.y); c[w][2] = __popc(v.z); c[w][3] = __popc(v.w);
#pragma unroll
      for (int y = 0; y < 4; ++y) sum[y] += c[w][y];
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) total += sum[y];
    uint32_t pre = total;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, pre, d);
      if (lane >= d) pre += o;
    }
    if (lane == 31) warp_sum[warp] = pre;
    __syncthreads();
    uint32_t at = base + pre - total;
#pragma unroll
    for (int w = 0; w < kBaMark / 32; ++w) {
      if (w < warp) at += warp_sum[w];
      base += warp_sum[w];
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int j = tid * 4 + y;
      if (j < n) a.spans[((long long)lbh * a.nb + j0 + j) * a.marks + mark] = at | sum[y] << 16;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        if (j < n) offs[w * W + j] = (uint16_t)at;
        at += c[w][y];
      }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < KR; ++s) {
      const int j = e[s] - j0;
      if (e[s] >= 0 && j >= 0 && j < n)
        sorted[offs[warp * W + j] + __popc(bits[warp * W + j] & (bit - 1))] = (uint16_t)(s << 8 | tid);
    }
    __syncthreads();
  }
  // out in 16-byte pieces (the group's place holds 256 topk entries)
  uint4* dst = reinterpret_cast<uint4*>(a.entries + ((long long)lbh * a.marks + mark) * kBaMark * K);
  for (int x = tid; x < ((int)base + 7) / 8; x += kBaMark) dst[x] = reinterpret_cast<const uint4*>(sorted)[x];
  unsigned long long counts = 0;
#pragma unroll
  for (int s = 0; s < KR; ++s) counts |= (unsigned long long)(e[s] >= 0) << s;
  if (on) a.slots[(long long)bh * a.q_rows + i] = counts;
  if (blockIdx.x == 0 && tid == 0) *a.ticket = 0;
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

// The queries that chose block j in the window's list groups from g on (up to `end`), as
// many whole groups as fit kBaChunk: list[] gets query << 6 | place in its list,
// ascending. Moves g past the groups taken; returns the number listed. Every
// thread of the CTA calls it; it begins and ends with a barrier.
template <int THREADS>
__device__ __forceinline__ int ba_fill(const BaArgs& a, int lbh, int j, int& g, int end, uint32_t* list) {
  __shared__ uint32_t pos[THREADS + 1], first[THREADS];
  __shared__ uint32_t warp_sum[THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool in = g + tid < end;
  const uint32_t sp = in ? a.spans[((long long)lbh * a.nb + j) * a.marks + g + tid] : 0u;
  const uint32_t cnt = sp >> 16;
  uint32_t pre = cnt;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, pre, d);
    if (lane >= d) pre += o;
  }
  __syncthreads();  // the list and these arrays may still be in use
  if (lane == 31) warp_sum[warp] = pre;
  __syncthreads();
  for (int w = 0; w < warp; ++w) pre += warp_sum[w];
  pos[tid + 1] = pre;
  first[tid] = sp & 0xffffu;
  if (tid == 0) pos[0] = 0;
  const int taken = __syncthreads_count(in && pre <= kBaChunk);
  const int n = (int)pos[taken];
  const uint16_t* entries = a.entries + ((long long)lbh * a.marks + g) * kBaMark * a.topk;
  for (int e0 = tid; e0 < n; e0 += 4 * THREADS) {  // four entries in flight
    int lo[4];
    uint32_t x[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int e = min(e0 + y * THREADS, n - 1);
      int l = 0, hi = taken - 1;  // the group that holds entry e
      while (l < hi) {
        const int mid = (l + hi + 1) >> 1;
        if (pos[mid] <= (uint32_t)e) l = mid;
        else hi = mid - 1;
      }
      lo[y] = l;
      x[y] = entries[(long long)l * kBaMark * a.topk + first[l] + (e - pos[l])];
    }
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (e0 + y * THREADS < n) list[e0 + y * THREADS] = (uint32_t)(a.w0 + (g + lo[y]) * kBaMark + (x[y] & 255)) << 6 | x[y] >> 8;
  }
  g += taken;
  __syncthreads();
  return n;
}

__device__ __forceinline__ float ba_exp2(float x) {  // 2^x, relative error 2^-22, 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What rounding two values to the packed 16-bit pair `hi` left of them, packed
// the same way: hi + rest holds a value to u^2 (u one rounding of the type).
template <typename T>
__device__ __forceinline__ float2 ba_unpack(uint32_t v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <typename T>
__device__ __forceinline__ uint32_t ba_rest(float a, float b, uint32_t hi) {
  const float2 h = ba_unpack<T>(hi);
  return MmaTraits<T>::pack(a - h.x, b - h.y);
}

__device__ __forceinline__ int ba_div_group(const BaArgs& a, int x) {
  return a.group_magic ? (int)__umulhi((uint32_t)x, a.group_magic) : x;
}

// Scores of 16 rows against BK keys, their row maxima and sums, and the output
// rows, all in registers (mma.sync accumulator layout: lane / 4 and + 8 the
// rows, 2 (lane % 4) and + 1 the columns of each 8-wide tile).
template <typename T, int DP, int BK>
struct BaTile {
  float s[BK / 8][4], o[DP / 8][4];
  float m[2], l[2];

  // weights, row maxima and sums; the keys are free afterwards
  __device__ __forceinline__ void scores(uint32_t q, uint32_t k, int live_keys, float scale_log2) {
    const int lane = threadIdx.x & 31;
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
    if (scale_log2 < 0.f) {
#pragma unroll
      for (int n = 0; n < BK / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = -s[n][e];
    }
    const float sc = fmaxf(fabsf(scale_log2), 1e-38f);  // not 0: masked scores stay -inf
    if (live_keys < BK) {
#pragma unroll
      for (int n = 0; n < BK / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n * 8 + 2 * (lane & 3) + (e & 1) >= live_keys) s[n][e] = -INFINITY;
    }
    m[0] = m[1] = -INFINITY;
#pragma unroll
    for (int n = 0; n < BK / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) m[e >> 1] = fmaxf(m[e >> 1], s[n][e]);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 1));
      m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 2));
      // -inf (no score above it: the row keeps weight 0) or the maximum in log2 units
      m[r] = m[r] == -INFINITY ? m[r] : m[r] * sc;
      l[r] = 0.f;
    }
    const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
    for (int n = 0; n < BK / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = ba_exp2(fmaf(s[n][e], sc, e >> 1 ? -m1 : -m0));
        l[e >> 1] += s[n][e];
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
  }
  __device__ __forceinline__ void output(uint32_t v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
    // weights go to the matrix unit as pairs of the inputs' 16-bit type, so that
    // the result is rounded once; their sum l is one of 32-bit weights
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      uint32_t fa[4], fr[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float* w = &s[2 * kk + (x >> 1)][2 * (x & 1)];
        fa[x] = MmaTraits<T>::pack(w[0], w[1]);
        fr[x] = ba_rest<T>(w[0], w[1], fa[x]);
      }
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        uint32_t fb[4];
        ldmatrix_x4_trans(fb, ba_at<DP>(v, 16 * kk + (lane & 15), 2 * n + (lane >> 4)));
        const uint32_t b0[2] = {fb[0], fb[1]}, b1[2] = {fb[2], fb[3]};
        MmaTraits<T>::mma(o[2 * n], fr, b0);
        MmaTraits<T>::mma(o[2 * n + 1], fr, b1);
        MmaTraits<T>::mma(o[2 * n], fa, b0);
        MmaTraits<T>::mma(o[2 * n + 1], fa, b1);
      }
    }
  }
};

// ---- forward, many queries -----------------------------------------------------
// Tiles of 128 listed rows on the fifth-generation tensor cores, one row a
// thread: S = Q K^T into TMEM; each thread reads its row of S, takes maximum,
// exponentials and sum without any exchange and writes the weights back over S as
// pairs of 16-bit numbers; O = P V with P as the TMEM operand; O leaves through the
// tile's own Q buffer (transposed there, so that a part goes out in whole 128-byte
// lines). Four CTAs an SM (128 TMEM columns each at D = 64) cover one another's waits.
// 8192 rows, 8 heads of 64, 16 of 128 blocks: 129 us, 118 with single 16-bit weights;
// an mma.sync form, 16 rows a warp, took 134 with those: it issued 48 instructions
// a row and read every key and value fragment from shared memory once per 16 rows
// (74 % of that pipe).
//
// Shared memory, rows of 128 bytes (64 channels; DP = 128: two panels) in the
// 128-byte swizzle: K, V [panels][BK], Q [2][panels][128]. As a left or right
// operand whose rows run over channels (Q, K) they are K-major; V, whose rows
// run over keys of the sum, is an N-major operand of the same bytes.
constexpr int kBaFwdThreads = 128;
constexpr int kBaFwdRows = 128;

__host__ __device__ constexpr int ba_panels(int dp) { return dp > 64 ? 2 : 1; }
template <int DP, int BK>
constexpr int ba_fwd_tmem() {
  return BK + DP <= 64 ? 64 : BK + DP <= 128 ? 128 : 256;
}
template <int DP, int BK>
constexpr int ba_fwd_smem() {
  constexpr int need = 1024 + ba_panels(DP) * (2 * BK + 2 * kBaFwdRows) * 128 + kBaChunk * 4 + kBaFwdRows * 12;
  // no more CTAs on an SM than its 512 TMEM columns serve: an allocation never waits
  constexpr int least = 232448 / (512 / ba_fwd_tmem<DP, BK>() + 1) + 1;
  return need > least ? need : least;
}
__device__ __forceinline__ uint32_t ba_panel_at(uint32_t base, int rows, int row, int chunk) {
  return base + (chunk >> 3) * rows * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}
// cp.async of key rows into panels (zero past `have` rows and past dim).
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void ba_load_panels(uint32_t dst, const T* src, long long stride, int have, int dim) {
  constexpr int CH = DP / 8;
#pragma unroll
  for (int x0 = 0; x0 < ROWS * CH; x0 += kBaFwdThreads) {
    const int x = x0 + threadIdx.x, r = x / CH, c = x % CH;
    if (ROWS * CH % kBaFwdThreads && x >= ROWS * CH) break;
    const bool ok = r < have && c * 8 < dim;
    cp_async16(ba_panel_at(dst, ROWS, r, c), ok ? src + r * stride + c * 8 : src, ok ? 16 : 0);
  }
}
// N columns of this thread's TMEM lane.
template <int N>
__device__ __forceinline__ void ba_tmem_ld(uint32_t taddr, float* v) {
  static_assert(N == 16 || N == 32, "");
  uint32_t r[N];
  __syncwarp();
  if constexpr (N == 32) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void ba_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Descriptor of an operand whose rows of 64 elements run along M or N (swizzled
// 128-byte rows, one row per K index): 8 K rows every 1024 bytes, further 64
// elements of M / N `panel` bytes on.
__device__ __forceinline__ uint64_t ba_mn_desc(uint32_t addr, uint32_t panel) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)((panel >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
constexpr uint32_t kIdescBMn = 1u << 16;  // right operand N-major

template <int DP, int BK>
constexpr int ba_fwd_ctas() {  // of an SM: by TMEM columns, and by its 228 KB (2 KB a CTA beside the dynamic part)
  constexpr int t = 512 / ba_fwd_tmem<DP, BK>(), m = 233472 / (ba_fwd_smem<DP, BK>() + 2048);
  return t < m ? t : m;
}

template <typename T, int DP, int BK>
__global__ __launch_bounds__(kBaFwdThreads, ba_fwd_ctas<DP, BK>()) void block_attn_kernel(const BaArgs a) {
  constexpr int PAN = ba_panels(DP), CH = DP / 8, ROWS = kBaFwdRows;
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t KB = PAN * BK * 128, QB = PAN * ROWS * 128;
  constexpr int SH = BK < 64 ? BK : 64;  // scores a thread holds at a time
  constexpr int OW = DP < 32 ? DP : 32;  // output channels staged at a time
  extern __shared__ char ba_smem_raw[];
  char* ba_smem = ba_smem_raw + (1024 - (smem_u32(ba_smem_raw) & 1023)) % 1024;
  const uint32_t ks = smem_u32(ba_smem), vs = ks + KB, qs = vs + KB;
  uint32_t* list = reinterpret_cast<uint32_t*>(ba_smem + 2 * KB + 2 * QB);
  long long* qoff = reinterpret_cast<long long*>(list + kBaChunk);  // [128]: rows of the tile being loaded
  int* dst = reinterpret_cast<int*>(qoff + ROWS);                    // [128]: parts of the tile being stored
  __shared__ __align__(8) uint64_t bars[2];
  __shared__ uint32_t tmem_slot;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ uint32_t next_item;
  const uint32_t items = (uint32_t)a.nbh * (uint32_t)a.nb * (uint32_t)a.nseg;
  const int G = a.group;
  const uint32_t bar_s = smem_u32(&bars[0]), bar_o = smem_u32(&bars[1]);
  if (warp == 0) {
    tmem_alloc(smem_u32(&tmem_slot), ba_fwd_tmem<DP, BK>());
    tmem_relinquish();
  }
  if (tid == 0) {
    mbar_init(bar_s, 1);
    mbar_init(bar_o, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  bool ok = true;
  uint32_t phase = 0;
  for (uint32_t u = blockIdx.x; u < items;) {
    const int sg = (int)(u % (uint32_t)a.nseg);
    const int j = (int)(u / (uint32_t)a.nseg % (uint32_t)a.nb);
    const int lbh = (int)(u / (uint32_t)a.nseg / (uint32_t)a.nb), bh = a.bh0 + lbh;
    const int b = bh / a.kv_heads, h = bh - b * a.kv_heads;
    int g = sg * a.seg;
    const int end = min(g + a.seg, (a.wq + kBaMark - 1) / kBaMark);
    const int have = min(BK, ba_kv_len(a, b) - j * BK);
    __syncthreads();  // the item before is done with the keys, and its successor has been read
    if (tid == 0) next_item = gridDim.x + atomicAdd(a.ticket, 1u);
    if (have <= 0) g = end;
    const T* qp = (const T*)a.q.p + b * a.q.b + (long long)h * G * a.q.h;
    // on their way while the list is made
    if (have > 0) {
    ba_load_panels<T, DP, BK>(ks, (const T*)a.k.p + b * a.k.b + h * a.k.h + (long long)j * BK * a.k.s, a.k.s, have, a.dim);
    ba_load_panels<T, DP, BK>(vs, (const T*)a.v.p + b * a.v.b + h * a.v.h + (long long)j * BK * a.v.s, a.v.s, have, a.dim);
    }
    while (g < end) {
      const int n = ba_fill<kBaFwdThreads>(a, lbh, j, g, end, list);
      if (n == 0) continue;
      const int rows = n * G, tiles = (rows + ROWS - 1) / ROWS;
      // a warp loads the 32 rows whose offsets its lanes worked out
      auto load_q = [&](int tile, uint32_t to) {
        const int row = tile * ROWS + tid;
        long long off = -1;
        if (row < rows) {
          const int li = ba_div_group(a, row);
          off = (row - li * G) * a.q.h + (long long)(list[li] >> 6) * a.q.s;
        }
        qoff[tid] = off;
        __syncwarp();
#pragma unroll
        for (int x0 = 0; x0 < 32 * CH; x0 += 32) {
          const int r = warp * 32 + (x0 + lane) / CH, c = (x0 + lane) % CH;
          const long long o = qoff[r];
          const bool in = o >= 0 && c * 8 < a.dim;
          cp_async16(ba_panel_at(to, ROWS, r, c), in ? qp + o + c * 8 : qp, in ? 16 : 0);
        }
        __syncwarp();
      };
      load_q(0, qs);
      cp_async_commit();
      for (int t = 0; t < tiles; ++t) {
        const uint32_t qt = qs + (t & 1) * QB;
        cp_async_wait_all();
        fence_proxy_async_smem();
        tc_fence_before();
        __syncthreads();  // Q of this tile is there; every thread has read the O of the one before
        tc_fence_after();
        const uint32_t s_tm = tmem, o_tm = tmem + BK, lanes = (uint32_t)(warp * 32) << 16;
        if (tid == 0) {
          constexpr uint32_t id = mma_idesc(BK, BF);
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk)
            tc_mma_f16(s_tm, sw128_desc(qt + kk / 4 * ROWS * 128 + kk % 4 * 32), sw128_desc(ks + kk / 4 * BK * 128 + kk % 4 * 32),
                       id, kk > 0);
          tc_commit(bar_s);
        }
        if (t + 1 < tiles) load_q(t + 1, qs + ((t + 1) & 1) * QB);
        cp_async_commit();
        ok = ok && mbar_wait(bar_s, phase);
        tc_fence_after();
        // this thread's row: maximum, weights, sum
        const float sc = fmaxf(fabsf(a.scale_log2), 1e-38f);  // not 0: masked scores stay -inf
        const bool flip = a.scale_log2 < 0.f;
        float s[SH], m = -INFINITY, l = 0.f;
        auto load_s = [&](int c0) {
#pragma unroll
          for (int x = 0; x < SH; x += 32) ba_tmem_ld<32>(s_tm + lanes + c0 + x, s + x);
          if (flip) {
#pragma unroll
            for (int x = 0; x < SH; ++x) s[x] = -s[x];
          }
          if (have < BK) {
#pragma unroll
            for (int x = 0; x < SH; ++x)
              if (c0 + x >= have) s[x] = -INFINITY;
          }
        };
#pragma unroll
        for (int c0 = 0; c0 < BK; c0 += SH) {
          load_s(c0);
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int x = 0; x < SH; ++x) m4[x & 3] = fmaxf(m4[x & 3], s[x]);
          m = fmaxf(m, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
        }
        // -inf (no score above it: the row keeps weight 0) or the maximum in log2 units
        const float ref = m == -INFINITY ? 0.f : m * sc;
        m = m == -INFINITY ? m : ref;
#pragma unroll
        for (int c0 = 0; c0 < BK; c0 += SH) {
          if (BK > SH) load_s(c0);
          // weights go to the matrix unit as pairs of the inputs' 16-bit type, so that
          // the result is rounded once (what rounding leaves of SH scores lies in the
          // columns behind their weights); their sum l is one of 32-bit weights
          float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < SH; c += 32) {
            uint32_t w[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              float &p0 = s[c + 2 * x], &p1 = s[c + 2 * x + 1];
              p0 = ba_exp2(fmaf(p0, sc, -ref));
              p1 = ba_exp2(fmaf(p1, sc, -ref));
              l4[x & 3] += p0 + p1;
              w[x] = MmaTraits<T>::pack(p0, p1);
              const float2 h = ba_unpack<T>(w[x]);
              p0 -= h.x;
              p1 -= h.y;
            }
            ba_tmem_st16(s_tm + lanes + c0 + c / 2, w);
#pragma unroll
            for (int x = 0; x < 16; ++x) w[x] = MmaTraits<T>::pack(s[c + 2 * x], s[c + 2 * x + 1]);
            ba_tmem_st16(s_tm + lanes + c0 + (SH + c) / 2, w);
          }
          l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncthreads();
        if (tid == 0) {
          tc_fence_after();
          constexpr uint32_t id = mma_idesc(DP, BF) | kIdescBMn;
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) {
            const uint32_t w = s_tm + kk * 16 / SH * SH + kk * 16 % SH / 2;
            tc_mma_f16_ts(o_tm, w + SH / 2, ba_mn_desc(vs + kk * 2048, BK * 128), id, kk > 0);
            tc_mma_f16_ts(o_tm, w, ba_mn_desc(vs + kk * 2048, BK * 128), id, 1);
          }
          tc_commit(bar_o);
        }
        // where this row's part goes (a window's parts number less than 2^31)
        const int row = t * ROWS + tid;
        int at = -1;
        if (row < rows) {
          const int li = ba_div_group(a, row);
          const uint32_t e = list[li];
          at = ((lbh * a.wq + ((int)(e >> 6) - a.w0)) * G + (row - li * G)) * a.topk + (int)(e & 63);
          // a wait that gave up leaves no number behind
          a.ml[at] = ok ? make_float2(m, l) : make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
        }
        dst[tid] = at;
        ok = ok && mbar_wait(bar_o, phase);
        phase ^= 1;
        tc_fence_after();
        // O to its parts: a warp's 32 rows through the Q tile's bytes (S is done with them)
        const uint32_t stage = qt + warp * 32 * 128;
#pragma unroll
        for (int c0 = 0; c0 < DP; c0 += OW) {
          float o[OW];
          ba_tmem_ld<OW>(o_tm + lanes + c0, o);
          __syncwarp();
#pragma unroll
          for (int x = 0; x < OW; x += 4)
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(stage + lane * 128 + (((x / 4) ^ (lane & 7)) << 4)),
                         "f"(o[x]), "f"(o[x + 1]), "f"(o[x + 2]), "f"(o[x + 3])
                         : "memory");
          __syncwarp();
          constexpr int LR = OW / 4;  // lanes of a row
#pragma unroll
          for (int x = 0; x < LR; ++x) {
            const int r = x * (32 / LR) + lane / LR, c = lane % LR;
            const uint4 v = lds128(stage + r * 128 + ((c ^ (r & 7)) << 4));
            const int to = dst[warp * 32 + r];
            if (to >= 0 && c0 + c * 4 < a.dim)
              *reinterpret_cast<uint4*>(a.part + (long long)to * a.dim + c0 + c * 4) = v;
          }
        }
      }
    }
    cp_async_wait_all();  // keys of an item that nobody chose
    __syncthreads();
    u = next_item;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, ba_fwd_tmem<DP, BK>());
}

// A row's place in the window, for the kernels that join parts: 2^cl lanes of
// eight channels each, times strands of lanes that take up to four parts each
// (where a warp has them); a warp holds as many rows as fit.
__host__ __device__ inline int ba_join_log2(int x) {
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}
__host__ __device__ inline int ba_join_lanes(int dim, int topk) {  // log2 of a row's lanes
  const int l = ba_join_log2(dim / 8) + ba_join_log2((topk + 3) / 4);
  return l < 5 ? l : 5;
}
struct BaRow {
  long long row;  // of the window
  int lbh, i, g, c, strand, strands, chunks;
  __device__ __forceinline__ BaRow(const BaArgs& a) {
    const int cl = ba_join_log2(a.dim / 8), rl = ba_join_lanes(a.dim, a.topk);
    const int lane = threadIdx.x & ((1 << rl) - 1);
    row = (long long)blockIdx.x * (kBaJoinThreads >> rl) + (threadIdx.x >> rl);
    c = (lane & ((1 << cl) - 1)) * 8;
    strand = lane >> cl;
    strands = 1 << (rl - cl);
    chunks = 1 << cl;
    const int iq = (int)(row / a.group);
    g = (int)(row - (long long)iq * a.group);
    lbh = iq / a.wq;
    i = a.w0 + iq - lbh * a.wq;
  }
};
// Sum over a row's strands.
__device__ __forceinline__ void ba_strand_sum(float (&acc)[8], const BaRow& r) {
  for (int m = r.chunks; m < r.chunks * r.strands; m <<= 1)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], m);
}

// Joins the parts of each row, four parts a lane in flight.
template <typename T>
__global__ __launch_bounds__(kBaJoinThreads) void block_attn_join_kernel(const BaArgs a) {
  const BaRow r(a);
  const bool there = r.row < (long long)a.nbh * a.wq * a.group;  // the others stay for the shuffles
  const int bh = there ? a.bh0 + r.lbh : 0, b = bh / a.kv_heads, h = (bh - b * a.kv_heads) * a.group + r.g;
  const unsigned long long slots = there ? a.slots[(long long)bh * a.q_rows + r.i] : 0ull;
  const float2* ml = a.ml + r.row * a.topk;
  const float* part = a.part + r.row * a.topk * a.dim + r.c;
  const bool on = r.c < a.dim;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f;
  for (int s0 = r.strand; s0 < a.topk; s0 += 4 * r.strands) {
    float2 p[4];
    float4 u[4], v[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int s = s0 + y * r.strands;
      const bool in = s < a.topk && (slots >> s & 1);
      p[y] = in ? ml[s] : make_float2(-INFINITY, 0.f);
      const float4* src = reinterpret_cast<const float4*>(part + (long long)s * a.dim);
      u[y] = in && on ? src[0] : make_float4(0.f, 0.f, 0.f, 0.f);
      v[y] = in && on ? src[1] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const float t = fmaxf(fmaxf(fmaxf(p[0].x, p[1].x), fmaxf(p[2].x, p[3].x)), top);
    const float ref = t == -INFINITY ? 0.f : t;
    const float w0 = ba_exp2(top - ref);
    top = t;
    sum *= w0;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= w0;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const float w = ba_exp2(p[y].x - ref);
      sum += w * p[y].y;
      acc[0] += w * u[y].x; acc[1] += w * u[y].y; acc[2] += w * u[y].z; acc[3] += w * u[y].w;
      acc[4] += w * v[y].x; acc[5] += w * v[y].y; acc[6] += w * v[y].z; acc[7] += w * v[y].w;
    }
  }
  float all = top;
  for (int m = r.chunks; m < r.chunks * r.strands; m <<= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, m));
  const float ref = all == -INFINITY ? 0.f : all;
  const float w = ba_exp2(top - ref);
  sum *= w;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= w;
  for (int m = r.chunks; m < r.chunks * r.strands; m <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  ba_strand_sum(acc, r);
  if (r.strand != 0 || !there) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  RotVec<T, 8> y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y.v[e] = rot_cast<T>(acc[e] * inv);
  if (on) *reinterpret_cast<RotVec<T, 8>*>((T*)a.o.p + b * a.o.b + h * a.o.h + r.i * a.o.s + r.c) = y;
  if (r.c == 0) a.lse[((long long)b * a.kv_heads * a.group + h) * a.q_rows + r.i] = (ref + log2f(sum)) * kLn2;
}

// ---- forward, few queries --------------------------------------------------------
// A cluster of CTAs per (batch, kv head, query): their warps take the row's blocks
// in turn, each with a key block of its own in shared memory, and keep running
// maxima, sums and output rows; the results are joined over a CTA's warps in
// shared memory, then over the cluster's CTAs in distributed shared memory, each
// CTA a share of the channels. The group's heads are the rows of the 16-row tile.
// Bound by the read of the chosen keys and values (8 x 8 rows, 4 heads of 128, 32
// blocks of 64: 30 us with one CTA a row, whose warps took 8 blocks one after
// another).
constexpr int kBaFewCluster = 8;
template <int DP, int BK>
constexpr int ba_few_warps() {
  return DP * BK >= 16384 ? 2 : DP * BK >= 8192 ? 4 : 8;
}
template <int DP, int BK>
constexpr int ba_few_smem() {
  return ba_few_warps<DP, BK>() * (2 * BK * DP * 2) + 16 * DP * 2 + 16 * DP * 4;
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
  __shared__ float2 cml[16];  // the CTA's maxima and sums
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int G = a.group, gt = (G + 15) / 16;
  const long long u = blockIdx.x / C;
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
  // the next block's keys load while this one's values are used, its values
  // while the next scores are computed
  const T* kp = (const T*)a.k.p + b * a.k.b + h * a.k.h;
  const T* vp = (const T*)a.v.p + b * a.v.b + h * a.v.h;
  auto load = [&](uint32_t to, const T* src, long long stride, int c) {
    if (c < n) {
      const int j = chosen[c];
      ba_load_rows<T, DP>(to, src + (long long)j * BK * stride, stride, BK, min(BK, kv - j * BK), a.dim, lane, 32);
    }
    cp_async_commit();
  };
  load(ks, kp, a.k.s, rank * W + warp);
  load(vs, vp, a.v.s, rank * W + warp);
  for (int c = rank * W + warp; c < n; c += C * W) {
    const int have = min(BK, kv - chosen[c] * BK);
    BaTile<T, DP, BK> tile;
    cp_async_wait<1>();
    __syncwarp();
    tile.scores(qs, ks, have, a.scale_log2);
    __syncwarp();
    load(ks, kp, a.k.s, c + C * W);
    cp_async_wait<1>();
    __syncwarp();
    tile.output(vs);
    __syncwarp();
    load(vs, vp, a.v.s, c + C * W);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float t = fmaxf(top[r], tile.m[r]);
      const float ref = t == -INFINITY ? 0.f : t;
      const float wo = ba_exp2(top[r] - ref), wn = ba_exp2(tile.m[r] - ref);
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
  cp_async_wait_all();
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
  float* cta = reinterpret_cast<float*>(ba_smem + W * (2 * BK * DP * 2) + 16 * DP * 2);  // [16][dim], the CTA's rows
  for (int x = threadIdx.x; x < rows * a.dim; x += W * 32) {
    const int row = x / a.dim, d = x - row * a.dim;
    float t = -INFINITY;
    for (int w = 0; w < W; ++w) t = fmaxf(t, sml[w][row].x);
    const float ref = t == -INFINITY ? 0.f : t;
    float acc = 0.f, s = 0.f;
    for (int w = 0; w < W; ++w) {
      const float f = ba_exp2(sml[w][row].x - ref);
      s += f * sml[w][row].y;
      acc += f * all[w * (16 * DP) + row * DP + d];
    }
    cta[x] = acc;
    if (d == 0) cml[row] = make_float2(t, s);
  }
  cluster.sync();
  for (int x = rank * W * 32 + threadIdx.x; x < rows * a.dim; x += C * W * 32) {
    const int row = x / a.dim, d = x - row * a.dim;
    float2 p[kBaFewCluster];
    float o[kBaFewCluster], t = -INFINITY;
#pragma unroll
    for (int c = 0; c < kBaFewCluster; ++c)
      if (c < C) {
        p[c] = cluster.map_shared_rank(cml, c)[row];
        o[c] = cluster.map_shared_rank(cta, c)[x];
        t = fmaxf(t, p[c].x);
      }
    const float ref = t == -INFINITY ? 0.f : t;
    float acc = 0.f, s = 0.f;
#pragma unroll
    for (int c = 0; c < kBaFewCluster; ++c)
      if (c < C) {
        const float f = ba_exp2(p[c].x - ref);
        s += f * p[c].y;
        acc += f * o[c];
      }
    const int hq = h * G + gi * 16 + row;
    ((T*)a.o.p)[b * a.o.b + hq * a.o.h + i * a.o.s + d] = rot_cast<T>(s == 0.f ? 0.f : acc / s);
    if (d == 0) a.lse[((long long)b * a.kv_heads * G + hq) * a.q_rows + i] = (ref + log2f(s)) * kLn2;
  }
  cluster.sync();  // a CTA's shared memory stays until the others have read it
}

// ---- backward --------------------------------------------------------------------
// delta = do . out of every row and the norm of do, 8 channels a lane.
template <typename T>
__global__ __launch_bounds__(256) void block_attn_delta_kernel(const BaArgs a) {
  const int chunks = a.dim / 8;
  int lanes = 1;
  while (lanes < chunks) lanes <<= 1;
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = x / lanes;
  const int c = (int)(x - row * lanes);
  const long long rows = (long long)a.batch * a.kv_heads * a.q_rows * a.group;
  float s = 0.f, n = 0.f;
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
      for (int e = 0; e < 8; ++e) {
        s += rot_f32(u.v[e]) * rot_f32(v.v[e]);
        n += rot_f32(v.v[e]) * rot_f32(v.v[e]);
      }
    }
  }
  for (int m = 1; m < lanes; m <<= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, m);
    n += __shfl_xor_sync(0xffffffffu, n, m);
  }
  if (row < rows && c == 0) a.delta[row] = make_float2(s, sqrtf(n));
}

// Work items as in the forward: one key block and a segment of the queries that
// chose it, tiles of 128 listed rows, a row a thread. Five products a tile on the
// tensor cores, all from shared memory:
//   S = Q K^T, dP = dO V^T                     128 rows x BK keys, into TMEM
//   p = 2^(S - lse), ds = p (dP - delta)       by the row's thread, to pairs of 16 bits
//   [dV; .] += [P | dS]^T dO, [.; dK] += [P | dS]^T Q   over the item's tiles, in TMEM
//   dQ = dS K                                  128 rows, a part of each pair
// P and dS are written [row][key] and read as M-major operands; for blocks of up
// to 64 keys both go through one 128-row operand (half of each result is not
// used), for 128 keys each is one. Both are pairs (what rounding leaves of a
// 16-bit number is another one), so that each gradient is rounded once; with single
// ones dv and dk were off by 1.4 times that, dq by 1.5 to 1.7. There is no room in
// shared memory for the second halves: they wait in TMEM over dP, from where dQ takes
// them as its left operand, and take the first ones' place for dV and dK once those
// are done. dQ lies over S, which is done with.
//
// f16 keeps full precision over 2^-14 to 2^16 only. There P is taken times 2^14 (it
// is 1 at most), and ds times a power of two that brings its bound
//   |ds| <= |do| max |v| + |delta|
// over the tile's rows and the block's keys below 2^15. The power holds for a work
// item (with two octaves to spare at first); a tile that needs a smaller one
// has the dk summed so far scaled down. Values down to 2^-37 of the bound are not lost.
//
// 8192 rows, 8 heads of 64, 16 of 128 blocks: 330 us, 266 with single 16-bit p and ds;
// an mma.sync form, 64 rows a tile, took 310 with those.
constexpr int kBaBwdThreads = 128;

template <int DP, int BK>
constexpr int ba_bwd_tmem() {
  constexpr int n = BK + (BK > DP ? BK : DP) + 2 * DP;
  return n <= 128 ? 128 : n <= 256 ? 256 : 512;
}
template <int DP, int BK>
constexpr int ba_bwd_smem() {
  constexpr int keys = BK > 64 ? 2 : 1;  // 64-key panels of P and dS
  constexpr int need = 1024 + ba_panels(DP) * (2 * BK + 2 * kBaFwdRows) * 128 +
                       (2 * keys + 1) * kBaFwdRows * 128 + kBaChunk * 4 + kBaFwdRows * 20;
  constexpr int least = 232448 / (512 / ba_bwd_tmem<DP, BK>() + 1) + 1;
  return need > least ? need : least;
}
template <int DP, int BK>
constexpr int ba_bwd_ctas() {
  constexpr int t = 512 / ba_bwd_tmem<DP, BK>(), m = 233472 / (ba_bwd_smem<DP, BK>() + 2048);
  return t < m ? t : m;
}
constexpr uint32_t kIdescAMn = 1u << 15;  // left operand M-major
constexpr int kBaPUp = 14;                // f16: P is held times 2^14
__device__ __forceinline__ float ba_pow2(int e) { return __int_as_float((e + 127) << 23); }  // |e| <= 126

template <typename T, int DP, int BK>
__global__ __launch_bounds__(kBaBwdThreads, ba_bwd_ctas<DP, BK>()) void block_attn_bwd_kernel(const BaArgs a) {
  constexpr int PAN = ba_panels(DP), CH = DP / 8, ROWS = kBaFwdRows, PK = BK > 64 ? 2 : 1;
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t KB = PAN * BK * 128, QB = PAN * ROWS * 128, PB = PK * ROWS * 128;
  constexpr int OW = DP < 32 ? DP : 32;  // channels staged at a time
  extern __shared__ char ba_smem_raw[];
  char* ba_smem = ba_smem_raw + (1024 - (smem_u32(ba_smem_raw) & 1023)) % 1024;
  const uint32_t ks = smem_u32(ba_smem), vs = ks + KB, qs = vs + KB, gs = qs + QB, ps = gs + QB, dss = ps + PB,
                 stages = dss + PB;  // P, dS, and the rows of dq on their way out
  uint32_t* list = reinterpret_cast<uint32_t*>(ba_smem + 2 * KB + 2 * QB + 2 * PB + ROWS * 128);
  long long* qoff = reinterpret_cast<long long*>(list + kBaChunk);  // [128] rows of the tile being loaded: q
  long long* goff = qoff + ROWS;                                     // [128] and dout
  int* dst = reinterpret_cast<int*>(goff + ROWS);                    // [128]: parts of the tile being stored
  __shared__ __align__(8) uint64_t bars[3];
  __shared__ uint32_t tmem_slot, next_item;
  __shared__ float row_norm[kBaBwdThreads / 32], row_delta[kBaBwdThreads / 32];  // the warps' largest of a tile
  __shared__ uint32_t v_bits;  // the largest sum of squares over 8 channels of a value
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t items = (uint32_t)a.nbh * (uint32_t)a.nb * (uint32_t)a.nseg;
  const int G = a.group;
  const uint32_t bar_s = smem_u32(&bars[0]), bar_o = smem_u32(&bars[1]), bar_r = smem_u32(&bars[2]);
  if (warp == 0) {
    tmem_alloc(smem_u32(&tmem_slot), ba_bwd_tmem<DP, BK>());
    tmem_relinquish();
  }
  if (tid == 0) {
    mbar_init(bar_s, 1);
    mbar_init(bar_o, 1);
    mbar_init(bar_r, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot, lanes = (uint32_t)(warp * 32) << 16;
  // dP and, 32 keys a piece, the rests of P and of dS (16 columns each); S and dQ
  const uint32_t dp_tm = tmem, s_tm = tmem + BK, dq_tm = s_tm;
  const uint32_t dv_tm = s_tm + (BK > DP ? BK : DP), dk_tm = dv_tm + DP;
  bool ok = true;
  uint32_t phase = 0;
  for (uint32_t u = blockIdx.x; u < items;) {
    const int sg = (int)(u % (uint32_t)a.nseg);
    const int j = (int)(u / (uint32_t)a.nseg % (uint32_t)a.nb);
    const int lbh = (int)(u / (uint32_t)a.nseg / (uint32_t)a.nb), bh = a.bh0 + lbh;
    const int b = bh / a.kv_heads, h = bh - b * a.kv_heads;
    int g = sg * a.seg;
    const int end = min(g + a.seg, (a.wq + kBaMark - 1) / kBaMark);
    const int have = max(0, min(BK, ba_kv_len(a, b) - j * BK));
    tc_fence_before();
    __syncthreads();  // the item before is done with the keys and with dv, dk
    if (tid == 0) {
      next_item = gridDim.x + atomicAdd(a.ticket, 1u);
      v_bits = 0;
    }
    if (have == 0) g = end;
    const T* qp = (const T*)a.q.p + b * a.q.b + (long long)h * G * a.q.h;
    const T* gp = (const T*)a.go.p + b * a.go.b + (long long)h * G * a.go.h;
    if (have > 0) {  // on their way while the list is made
      ba_load_panels<T, DP, BK>(ks, (const T*)a.k.p + b * a.k.b + h * a.k.h + (long long)j * BK * a.k.s, a.k.s, have, a.dim);
      ba_load_panels<T, DP, BK>(vs, (const T*)a.v.p + b * a.v.b + h * a.v.h + (long long)j * BK * a.v.s, a.v.s, have, a.dim);
    }
    bool any = false;  // dv, dk hold something of this item
    int ex = 0;        // f16: ds and dk are held times 2^ex
    float v_norm = 0.f;
    while (g < end) {
      const int n = ba_fill<kBaBwdThreads>(a, lbh, j, g, end, list);
      if (n == 0) continue;
      const int rows = n * G, tiles = (rows + ROWS - 1) / ROWS;
      float lse = INFINITY;  // of this thread's row of the next tile, as loaded
      float2 delta = make_float2(0.f, 0.f);
      int at = -1;
      // a warp loads the 32 rows whose offsets its lanes worked out
      auto load_tile = [&](int tile) {
        const int row = tile * ROWS + tid;
        long long off = -1, og = 0;
        lse = INFINITY;  // rows that are not there: weight 0
        delta = make_float2(0.f, 0.f);
        at = -1;
        if (row < rows) {
          const int li = ba_div_group(a, row), gr = row - li * G;
          const uint32_t e = list[li];
          const int i = (int)(e >> 6);
          off = gr * a.q.h + (long long)i * a.q.s;
          og = gr * a.go.h + (long long)i * a.go.s;
          lse = a.lse[((long long)b * a.kv_heads * G + h * G + gr) * a.q_rows + i];
          delta = a.delta[((long long)bh * a.q_rows + i) * G + gr];
          // where its dq part goes (a window's parts number less than 2^31)
          at = ((lbh * a.wq + (i - a.w0)) * G + gr) * a.topk + (int)(e & 63);
        }
        qoff[tid] = off;
        goff[tid] = og;
        __syncwarp();
#pragma unroll
        for (int x0 = 0; x0 < 32 * CH; x0 += 32) {
          const int r = warp * 32 + (x0 + lane) / CH, c = (x0 + lane) % CH;
          const long long o = qoff[r];
          const bool in = o >= 0 && c * 8 < a.dim;
          cp_async16(ba_panel_at(qs, ROWS, r, c), in ? qp + o + c * 8 : qp, in ? 16 : 0);
          cp_async16(ba_panel_at(gs, ROWS, r, c), in ? gp + goff[r] + c * 8 : gp, in ? 16 : 0);
        }
        __syncwarp();
      };
      // [P | dS]: the panel after P's first is dS for up to 64 keys, P's second for 128
      auto products = [&](bool add) {
        constexpr uint32_t id = mma_idesc(DP, BF) | kIdescAMn | kIdescBMn;
#pragma unroll
        for (int kk = 0; kk < ROWS / 16; ++kk)
          tc_mma_f16(dv_tm, ba_mn_desc(ps + kk * 2048, ROWS * 128), ba_mn_desc(gs + kk * 2048, ROWS * 128), id, add || kk > 0);
#pragma unroll
        for (int kk = 0; kk < ROWS / 16; ++kk)
          tc_mma_f16(dk_tm, ba_mn_desc((BK > 64 ? dss : ps) + kk * 2048, ROWS * 128), ba_mn_desc(qs + kk * 2048, ROWS * 128),
                     id, add || kk > 0);
      };
      load_tile(0);
      for (int t = 0; t < tiles; ++t) {
        // a row all of whose scores are -inf has no weights
        const float lse_t = lse == -INFINITY ? INFINITY : lse * kLog2e, delta_t = delta.x;
        if (!BF) {  // rows that hold infinities or NaN pass them on; the others' scale ignores them
          const uint32_t n = __reduce_max_sync(0xffffffffu, delta.y < INFINITY ? __float_as_uint(delta.y) : 0u);
          const uint32_t d = __reduce_max_sync(0xffffffffu, fabsf(delta_t) < INFINITY ? __float_as_uint(fabsf(delta_t)) : 0u);
          if (lane == 0) {
            row_norm[warp] = __uint_as_float(n);
            row_delta[warp] = __uint_as_float(d);
          }
        }
        dst[tid] = at;
        cp_async_wait_all();
        fence_proxy_async_smem();
        tc_fence_before();
        __syncthreads();  // the tile is there; every thread has read the dq of the one before
        tc_fence_after();
        if (tid == 0) {
          constexpr uint32_t id = mma_idesc(BK, BF);
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk)
            tc_mma_f16(s_tm, sw128_desc(qs + kk / 4 * ROWS * 128 + kk % 4 * 32),
                       sw128_desc(ks + kk / 4 * BK * 128 + kk % 4 * 32), id, kk > 0);
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk)
            tc_mma_f16(dp_tm, sw128_desc(gs + kk / 4 * ROWS * 128 + kk % 4 * 32),
                       sw128_desc(vs + kk / 4 * BK * 128 + kk % 4 * 32), id, kk > 0);
          tc_commit(bar_s);
        }
        if (!BF) {
          if (!any) {
            uint32_t most = 0;
            for (int x = tid; x < BK * CH; x += kBaBwdThreads) {
              const uint4 w = lds128(ba_panel_at(vs, BK, x / CH, x % CH));
              const float2 f[4] = {ba_unpack<T>(w.x), ba_unpack<T>(w.y), ba_unpack<T>(w.z), ba_unpack<T>(w.w)};
              float n = 0.f;
#pragma unroll
              for (int y = 0; y < 4; ++y) n += f[y].x * f[y].x + f[y].y * f[y].y;
              if (n < INFINITY) most = max(most, __float_as_uint(n));
            }
            most = __reduce_max_sync(0xffffffffu, most);
            if (lane == 0) atomicMax(&v_bits, most);
            __syncthreads();
            v_norm = sqrtf((float)CH * __uint_as_float(v_bits));
          }
          float n = 0.f, d = 0.f;
#pragma unroll
          for (int w = 0; w < kBaBwdThreads / 32; ++w) {
            n = fmaxf(n, row_norm[w]);
            d = fmaxf(d, row_delta[w]);
          }
          // bound < 2^(b + 1): times 2^(14 - b) it stays below 2^15
          const int most = 14 - ((int)(__float_as_uint(fmaxf(fmaf(n, v_norm, d), 1e-24f)) >> 23) - 127);
          if (!any) {
            ex = most - 2;
          } else if (ex > most) {
            const float f = ba_pow2(most - 2 - ex);
            ex = most - 2;
#pragma unroll
            for (int c0 = 0; c0 < DP; c0 += 16) {
              float o[16];
              uint32_t w[16];
              ba_tmem_ld<16>(dk_tm + lanes + c0, o);
#pragma unroll
              for (int x = 0; x < 16; ++x) w[x] = __float_as_uint(o[x] * f);
              ba_tmem_st16(dk_tm + lanes + c0, w);
            }
          }
        }
        const float p_up = BF ? 0.f : kBaPUp, g = BF ? 1.f : ba_pow2(ex - kBaPUp), ds_down = BF ? 1.f : ba_pow2(-ex);
        ok = ok && mbar_wait(bar_s, phase);
        tc_fence_after();
#pragma unroll
        for (int c0 = 0; c0 < BK; c0 += 32) {
          float s[32], dp[32];
          ba_tmem_ld<32>(s_tm + lanes + c0, s);
          ba_tmem_ld<32>(dp_tm + lanes + c0, dp);
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            s[x] = ba_exp2(fmaf(s[x], a.scale_log2, p_up - lse_t));
            dp[x] = s[x] * (BF ? dp[x] - delta_t : fmaf(dp[x], g, -delta_t * g));
          }
          if (c0 + 32 > have) {
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (c0 + x >= have) s[x] = dp[x] = 0.f;
          }
          uint32_t rp[16], rd[16];
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            uint32_t wp[4], wd[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int i = x + 2 * y;
              wp[y] = MmaTraits<T>::pack(s[i], s[i + 1]);
              rp[x / 2 + y] = ba_rest<T>(s[i], s[i + 1], wp[y]);
              wd[y] = MmaTraits<T>::pack(dp[i], dp[i + 1]);
              // past the type's range wd is infinite, and the product says so
              const float2 h = ba_unpack<T>(wd[y]);
              rd[x / 2 + y] = MmaTraits<T>::pack(isinf(h.x) ? 0.f : dp[i] - h.x, isinf(h.y) ? 0.f : dp[i + 1] - h.y);
            }
            const uint32_t to = ba_panel_at(0, ROWS, tid, (c0 + x) / 8);
            sts128(ps + to, wp);
            sts128(dss + to, wd);
          }
          ba_tmem_st16(dp_tm + lanes + c0, rp);
          ba_tmem_st16(dp_tm + lanes + c0 + 16, rd);
        }
        tmem_wait_st();
        fence_proxy_async_smem();
        tc_fence_before();
        __syncthreads();
        if (tid == 0) {
          tc_fence_after();
          constexpr uint32_t id_q = mma_idesc(DP, BF) | kIdescBMn;
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) {
            tc_mma_f16(dq_tm, sw128_desc(dss + kk / 4 * ROWS * 128 + kk % 4 * 32), ba_mn_desc(ks + kk * 2048, BK * 128), id_q,
                       kk > 0);
            tc_mma_f16_ts(dq_tm, dp_tm + kk / 2 * 32 + 16 + kk % 2 * 8, ba_mn_desc(ks + kk * 2048, BK * 128), id_q, 1);
          }
          products(any);
          tc_commit(bar_o);
        }
        any = true;
        ok = ok && mbar_wait(bar_o, phase);
        tc_fence_after();
        // the rests take the place of P and dS
#pragma unroll
        for (int c0 = 0; c0 < BK; c0 += 32) {
          float r[32];
          ba_tmem_ld<32>(dp_tm + lanes + c0, r);
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            const uint32_t to = ba_panel_at(0, ROWS, tid, (c0 + x) / 8);
            uint32_t w[4];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
#pragma unroll
              for (int y = 0; y < 4; ++y) w[y] = __float_as_uint(r[16 * z + x / 2 + y]);
              sts128((z ? dss : ps) + to, w);
            }
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncthreads();
        if (tid == 0) {
          tc_fence_after();
          products(true);
          tc_commit(bar_r);
        }
        // dq to its parts, a warp's 32 rows at a time through its stage
        const uint32_t stage = stages + warp * 32 * 128;
#pragma unroll
        for (int c0 = 0; c0 < DP; c0 += OW) {
          float o[OW];
          ba_tmem_ld<OW>(dq_tm + lanes + c0, o);
          if (!BF) {
#pragma unroll
            for (int x = 0; x < OW; ++x) o[x] *= ds_down;
          }
          if (!ok) o[0] = __int_as_float(0x7fc00000);  // a wait that gave up leaves no number
          __syncwarp();
#pragma unroll
          for (int x = 0; x < OW; x += 4)
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(stage + lane * 128 + (((x / 4) ^ (lane & 7)) << 4)),
                         "f"(o[x]), "f"(o[x + 1]), "f"(o[x + 2]), "f"(o[x + 3])
                         : "memory");
          __syncwarp();
          constexpr int LR = OW / 4;  // lanes of a row
#pragma unroll
          for (int x = 0; x < LR; ++x) {
            const int r = x * (32 / LR) + lane / LR, c = lane % LR;
            const uint4 v = lds128(stage + r * 128 + ((c ^ (r & 7)) << 4));
            const int to = dst[warp * 32 + r];
            if (to >= 0 && c0 + c * 4 < a.dim)
              *reinterpret_cast<uint4*>(a.part + (long long)to * a.dim + c0 + c * 4) = v;
          }
          if (c0 == 0) {  // q and dout are done with: the next rows load under the other channels
            ok = ok && mbar_wait(bar_r, phase);
            tc_fence_after();
            if (t + 1 < tiles) load_tile(t + 1);
          }
        }
        phase ^= 1;
        __syncwarp();  // dst is written over by the next tile
      }
    }
    cp_async_wait_all();  // keys of an item that nobody chose
    // the item's keys: final rows, or this segment's part; a lane of TMEM a key
#pragma unroll
    for (int w = 0; w < (BK > 64 ? 2 : 1); ++w) {
      const bool is_v = BK > 64 ? w == 0 : tid < 64;  // this warp's half: dv or dk
      const int key = BK > 64 ? tid : tid & 63;
      const float down = BF ? 1.f : ba_pow2(is_v ? -kBaPUp : -ex);
      const float f = !ok ? __int_as_float(0x7fc00000) : is_v ? down : a.scale * down;  // a wait that gave up leaves no number
#pragma unroll
      for (int c0 = 0; c0 < DP; c0 += 16) {
        float o[16];
        ba_tmem_ld<16>((is_v ? dv_tm : dk_tm) + lanes + c0, o);
        if (!any || key >= have) {  // dead keys: zeros, whatever the rows hold
#pragma unroll
          for (int x = 0; x < 16; ++x) o[x] = 0.f;
        }
        if (key >= BK) continue;
#pragma unroll
        for (int x = 0; x < 16; x += 8) {
          if (c0 + x >= a.dim) continue;
          if (a.sums > 0) {
            float4* p = reinterpret_cast<float4*>(
                a.kv_part + ((((long long)lbh * a.nb + j) * a.sums + sg) * 2 * BK + (is_v ? BK : 0) + key) * a.dim + c0 + x);
            // the sum over the segments scales; windows after the first add to what the ones before left
            const float one = ok ? down : f;
            float4 u = make_float4(0.f, 0.f, 0.f, 0.f), v = u;
            if (a.w0 > 0) {
              u = p[0];
              v = p[1];
            }
            p[0] = make_float4(u.x + o[x] * one, u.y + o[x + 1] * one, u.z + o[x + 2] * one, u.w + o[x + 3] * one);
            p[1] = make_float4(v.x + o[x + 4] * one, v.y + o[x + 5] * one, v.z + o[x + 6] * one, v.w + o[x + 7] * one);
          } else if (j * BK + key < a.kv_rows) {
            const HeadsView& d = is_v ? a.dv : a.dk;
            T* p = (T*)d.p + b * d.b + h * d.h + (long long)(j * BK + key) * d.s + c0 + x;
            *reinterpret_cast<uint4*>(p) =
                make_uint4(MmaTraits<T>::pack(o[x] * f, o[x + 1] * f), MmaTraits<T>::pack(o[x + 2] * f, o[x + 3] * f),
                           MmaTraits<T>::pack(o[x + 4] * f, o[x + 5] * f), MmaTraits<T>::pack(o[x + 6] * f, o[x + 7] * f));
          }
        }
      }
    }
    __syncthreads();
    u = next_item;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, ba_bwd_tmem<DP, BK>());
}

// dq of the window: the sum of each row's parts.
template <typename T>
__global__ __launch_bounds__(kBaJoinThreads) void block_attn_dq_kernel(const BaArgs a) {
  const BaRow r(a);
  const bool there = r.row < (long long)a.nbh * a.wq * a.group;  // the others stay for the shuffles
  const int bh = there ? a.bh0 + r.lbh : 0, b = bh / a.kv_heads, h = (bh - b * a.kv_heads) * a.group + r.g;
  const unsigned long long slots = there ? a.slots[(long long)bh * a.q_rows + r.i] : 0ull;
  const float* part = a.part + r.row * a.topk * a.dim + r.c;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s0 = r.strand; s0 < a.topk; s0 += 4 * r.strands) {
    float4 u[4], v[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int s = s0 + y * r.strands;
      const bool in = s < a.topk && (slots >> s & 1) && r.c < a.dim;
      const float4* src = reinterpret_cast<const float4*>(part + (long long)s * a.dim);
      u[y] = in ? src[0] : make_float4(0.f, 0.f, 0.f, 0.f);
      v[y] = in ? src[1] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      acc[0] += u[y].x; acc[1] += u[y].y; acc[2] += u[y].z; acc[3] += u[y].w;
      acc[4] += v[y].x; acc[5] += v[y].y; acc[6] += v[y].z; acc[7] += v[y].w;
    }
  }
  ba_strand_sum(acc, r);
  if (r.strand != 0 || r.c >= a.dim || !there) return;
  RotVec<T, 8> y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y.v[e] = rot_cast<T>(acc[e] * a.scale);
  *reinterpret_cast<RotVec<T, 8>*>((T*)a.dq.p + b * a.dq.b + h * a.dq.h + r.i * a.dq.s + r.c) = y;
}

// dk, dv of a step's heads: the sum over the segments, in their order.
template <typename T>
__global__ __launch_bounds__(256) void block_attn_dkv_kernel(const BaArgs a) {
  const int chunks = a.dim / 8;
  const long long total = (long long)a.nbh * a.kv_rows * chunks;
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  if (x >= total) return;
  const long long row = x / chunks;
  const int c = (int)(x - row * chunks);
  const int lbh = (int)(row / a.kv_rows), t = (int)(row - (long long)lbh * a.kv_rows);
  const int bh = a.bh0 + lbh, b = bh / a.kv_heads, h = bh - b * a.kv_heads;
  const int j = t / a.block, key = t - j * a.block;
  const long long step = 2ll * a.block * a.dim;
  const float* p = a.kv_part + ((long long)lbh * a.nb + j) * a.sums * step + (long long)key * a.dim + c * 8;
  float acc[2][8] = {};
  for (int s = 0; s < a.sums; ++s, p += step)
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
