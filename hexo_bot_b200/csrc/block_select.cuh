// Block means of the keys, and the key blocks that each query keeps.
//
//   mean[j]  = sum of the block's live keys / their count
//   score    = (sum over the group's query heads of q) . mean[j]
//   kept     = forced blocks (leading ones, the query's own), then the best
//              scores; ties to the lowest index, NaN below everything
//
// The choice is the one 64-bit arithmetic on the given means makes. Scores are
// computed in 32 bits together with a bound on their error; a row whose last
// kept and first dropped score lie within that bound of one another (or that
// holds a score that is not finite) is done again in 64 bits, all others are
// settled by their 32-bit scores.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>

#include "rotary.cuh"

namespace sb {

constexpr int kSelMaxDim = 256;
constexpr int kSelMaxTopk = 64;
constexpr int kSelMaxBlocks = 16384;
constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelChunk = 64;  // blocks of a score chunk

struct HeadsView {
  const void* p;
  long long b, h, s;
};

// ---- block means ------------------------------------------------------------
// One CTA per (batch, head, block). Sums run in 64 bits, so 16-bit keys add up
// without error and the mean is rounded once.
constexpr int kMeansThreads = 128;

template <typename T, int VEC>
__global__ __launch_bounds__(kMeansThreads) void block_means_kernel(HeadsView k, const int* __restrict__ kv_lens,
                                                                    int heads, int rows, int dim, int block, int nb,
                                                                    float* __restrict__ out) {
  __shared__ double red[kMeansThreads * VEC];
  const long long u = blockIdx.x;
  const int j = (int)(u % nb);
  const long long bh = u / nb;
  const int b = (int)(bh / heads), h = (int)(bh - (long long)b * heads);
  int len = kv_lens ? kv_lens[b] : rows;
  len = len < 0 ? 0 : len > rows ? rows : len;
  const int n = len - j * block < block ? len - j * block : block;
  const int chunks = dim / VEC;
  using V = RotVec<T, VEC>;
  const T* base = (const T*)k.p + b * k.b + h * k.h + (long long)j * block * k.s;
  for (int c0 = 0; c0 < chunks; c0 += kMeansThreads) {
    const int nc = chunks - c0 < kMeansThreads ? chunks - c0 : kMeansThreads;
    const int strands = kMeansThreads / nc;
    const int c = threadIdx.x % nc, g = threadIdx.x / nc;
    double acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.0;
    if (g < strands)
      for (int r = g; r < n; r += strands) {
        const V v = *reinterpret_cast<const V*>(base + r * k.s + (c0 + c) * VEC);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += (double)rot_f32(v.v[e]);
      }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) red[e * kMeansThreads + threadIdx.x] = acc[e];
    __syncthreads();
    for (int i = threadIdx.x; i < nc * VEC; i += kMeansThreads) {
      const int cc = i / VEC, e = i - cc * VEC;
      double s = 0.0;
      for (int g2 = 0; g2 < strands; ++g2) s += red[e * kMeansThreads + g2 * nc + cc];
      out[(bh * nb + j) * dim + (c0 + cc) * VEC + e] = n > 0 ? (float)(s / n) : 0.f;
    }
  }
}

// ---- selection --------------------------------------------------------------
struct SelArgs {
  HeadsView q;
  const float* means;  // (B, Hkv, nb, D)
  const int* kv_lens;
  const int* q_lens;
  int* out;            // (B, Hkv, Sq, topk)
  int batch, kv_heads, group, q_rows, kv_rows, dim, nb, block, topk, keep_first, keep_own;
  int tile;            // queries of a CTA
  int tiles;           // tiles of a sequence
};

// Order-preserving image of a float (larger float -> larger integer).
__device__ __forceinline__ uint32_t sel_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sel_unkey(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ bool sel_forced(int j, int own, int keep_first) { return j < keep_first || j == own; }

// Writes the kept blocks of one row in ascending order, -1 behind them. `kept`
// tells for a block index whether it is kept; called by a whole warp.
template <typename F>
__device__ __forceinline__ void sel_write(int* out, int live, int topk, F kept) {
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (int j0 = 0; j0 < live; j0 += 32) {
    const int j = j0 + lane;
    const bool k = j < live && kept(j);
    const uint32_t m = __ballot_sync(0xffffffffu, k);
    const int at = n + __popc(m & ((1u << lane) - 1u));
    if (k && at < topk) out[at] = j;
    n += __popc(m);
  }
  for (int i = n + lane; i < topk; i += 32) out[i] = -1;
}

// One row settled by 32-bit scores s[0..live): returns false when the row is
// too close to call. `err` bounds the error of every score.
__device__ __forceinline__ bool sel_row_fast(const float* s, int live, int topk, int forced, int own, int keep_first,
                                             float err, int* out) {
  const int lane = threadIdx.x & 31;
  const int want = topk - forced;  // among the blocks that are not forced
  const int rest = live - forced;
  if (want >= rest) {
    sel_write(out, live, topk, [](int) { return true; });
    return true;
  }
  if (want <= 0) {
    sel_write(out, live, topk, [&](int j) { return sel_forced(j, own, keep_first); });
    return true;
  }
  bool odd = false;
  for (int j = lane; j < live; j += 32) odd |= !isfinite(s[j]) && !sel_forced(j, own, keep_first);
  if (__any_sync(0xffffffffu, odd) || !isfinite(err)) return false;
  // largest threshold that at least `want` scores reach, bit by bit; done as
  // soon as exactly `want` of them do
  uint32_t t = 0;
  bool exact = false;
  for (int bit = 31; bit >= 0 && !exact; --bit) {
    const uint32_t cand = t | (1u << bit);
    unsigned c = 0;
    for (int j = lane; j < live; j += 32) c += !sel_forced(j, own, keep_first) && sel_key(s[j]) >= cand;
    c = __reduce_add_sync(0xffffffffu, c);
    if (c >= (unsigned)want) t = cand;
    exact = c == (unsigned)want;
  }
  // the smallest kept and the largest dropped score
  uint32_t lo = 0xffffffffu, hi = 0;
  unsigned c = 0;
  for (int j = lane; j < live; j += 32) {
    if (sel_forced(j, own, keep_first)) continue;
    const uint32_t k = sel_key(s[j]);
    if (k >= t) {
      lo = k < lo ? k : lo;
      ++c;
    } else {
      hi = k > hi ? k : hi;
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  c = __reduce_add_sync(0xffffffffu, c);
  if (c != (unsigned)want) return false;  // equal scores at the border
  if (!(sel_unkey(lo) - sel_unkey(hi) > 2.f * err)) return false;
  sel_write(out, live, topk, [&](int j) { return sel_forced(j, own, keep_first) || sel_key(s[j]) >= t; });
  return true;
}

// One row in 64 bits: s holds the scores; a taken block is marked by NaN.
__device__ __forceinline__ void sel_row_exact(double* s, int live, int topk, int forced, int own, int keep_first,
                                              int* out) {
  const int lane = threadIdx.x & 31;
  const int want = min(topk, live) - forced;
  for (int r = 0; r < want; ++r) {
    double best = 0.0;
    int at = 0x7fffffff;
    for (int j = lane; j < live; j += 32)
      if (!sel_forced(j, own, keep_first) && !isnan(s[j]) && (at == 0x7fffffff || s[j] > best)) {
        best = s[j];
        at = j;
      }
    for (int m = 16; m; m >>= 1) {
      const double ob = __shfl_xor_sync(0xffffffffu, best, m);
      const int oa = __shfl_xor_sync(0xffffffffu, at, m);
      if (oa != 0x7fffffff && (at == 0x7fffffff || ob > best || (ob == best && oa < at))) {
        best = ob;
        at = oa;
      }
    }
    if (at != 0x7fffffff && lane == 0) s[at] = __longlong_as_double(0x7ff8000000000000ll);
    __syncwarp();
  }
  sel_write(out, live, topk, [&](int j) { return sel_forced(j, own, keep_first) || isnan(s[j]); });
}

// Shared memory: scores [tile][nb] fp32 (later reused as 64-bit scores, one
// row per warp), the tile's summed queries (rows padded to 16 bytes plus 16) fp32, their 1-norms,
// a mean chunk with the same rows, the redo list.
__host__ __device__ inline int sel_smem_bytes(int tile, int nb, int dim) {
  const int scores = tile * (nb + (nb & 1)) * 4;
  const int ds = (dim + 3) / 4 * 4 + 4;
  return scores + tile * ds * 4 + kSelChunk * ds * 4 + tile * 8;
}

template <typename T>
__global__ __launch_bounds__(kSelThreads) void block_select_kernel(const SelArgs a) {
  extern __shared__ __align__(16) char sel_smem[];
  const int D = a.dim, DS = (D + 3) / 4 * 4 + 4, NBS = a.nb + (a.nb & 1), TQ = a.tile;
  float* sc = reinterpret_cast<float*>(sel_smem);
  float* qs = sc + TQ * NBS;
  float* ms = qs + TQ * DS;
  float* q1 = ms + kSelChunk * DS;
  int* redo = reinterpret_cast<int*>(q1 + TQ);
  __shared__ int redo_n;
  __shared__ uint32_t mmax_bits;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long u = blockIdx.x;
  const int tile = (int)(u % a.tiles);
  const long long bh = u / a.tiles;
  const int b = (int)(bh / a.kv_heads), h = (int)(bh - (long long)b * a.kv_heads);
  const int i0 = tile * TQ;
  int kv = a.kv_lens ? a.kv_lens[b] : a.kv_rows, ql = a.q_lens ? a.q_lens[b] : a.q_rows;
  kv = kv < 0 ? 0 : kv > a.kv_rows ? a.kv_rows : kv;
  ql = ql < 0 ? 0 : ql > a.q_rows ? a.q_rows : ql;
  const int live = (kv + a.block - 1) / a.block;
  const int nq = a.q_rows - i0 < TQ ? a.q_rows - i0 : TQ;  // rows of the tile
  const int nl = ql - i0 < 0 ? 0 : ql - i0 < nq ? ql - i0 : nq;  // live ones
  int* out = a.out + (bh * a.q_rows + i0) * a.topk;
  const float* means = a.means + bh * a.nb * D;
  if (tid == 0) {
    redo_n = 0;
    mmax_bits = 0;
  }
  for (int i = tid; i < (nq - nl) * a.topk; i += kSelThreads) out[(long long)nl * a.topk + i] = -1;
  if (nl == 0) return;

  // the group's summed queries and the 1-norm over all of their terms
  const T* qb = (const T*)a.q.p + b * a.q.b + (long long)h * a.group * a.q.h + (long long)i0 * a.q.s;
  for (int r = warp; r < nl; r += kSelWarps) {
    float n1 = 0.f;
    for (int d = lane; d < D; d += 32) {
      float s = 0.f;
      for (int g = 0; g < a.group; ++g) {
        const float v = rot_f32(qb[g * a.q.h + r * a.q.s + d]);
        s += v;
        n1 += fabsf(v);
      }
      qs[r * DS + d] = s;
    }
    for (int m = 16; m; m >>= 1) n1 += __shfl_xor_sync(0xffffffffu, n1, m);
    if (lane == 0) q1[r] = n1;
  }
  float mm = 0.f;
  for (int j0 = 0; j0 < live; j0 += kSelChunk) {
    const int nj = live - j0 < kSelChunk ? live - j0 : kSelChunk;
    __syncthreads();
    for (int i = tid; i < nj * D; i += kSelThreads) {
      const int r = i / D, d = i - r * D;
      const float v = means[(long long)j0 * D + i];
      ms[r * DS + d] = v;
      mm = fmaxf(mm, fabsf(v));
    }
    __syncthreads();
    // 4 queries x 4 blocks a thread: queries ty, ty + 16, ..., blocks tx, tx + 16, ...
    const int tx = tid & 15, ty = tid >> 4;
    for (int q0 = 0; q0 < nl; q0 += 64) {
      float acc[4][4];
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = 0.f;
      int d = 0;
      for (; d + 4 <= D; d += 4) {
        float4 qv[4], mv[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int r = q0 + ty + 16 * x;
          qv[x] = *reinterpret_cast<const float4*>(qs + (r < nl ? r : 0) * DS + d);
          mv[x] = *reinterpret_cast<const float4*>(ms + (tx + 16 * x < nj ? tx + 16 * x : 0) * DS + d);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y)
            acc[x][y] += qv[x].x * mv[y].x + qv[x].y * mv[y].y + qv[x].z * mv[y].z + qv[x].w * mv[y].w;
      }
      for (; d < D; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int r = q0 + ty + 16 * x, c = tx + 16 * y;
            acc[x][y] += qs[(r < nl ? r : 0) * DS + d] * ms[(c < nj ? c : 0) * DS + d];
          }
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int r = q0 + ty + 16 * x, c = tx + 16 * y;
          if (r < nl && c < nj) sc[r * NBS + j0 + c] = acc[x][y];
        }
    }
  }
  for (int m = 16; m; m >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, m));
  if (lane == 0) atomicMax(&mmax_bits, __float_as_uint(mm));  // mm >= 0: bits order as values
  __syncthreads();
  // |fl(score) - score| <= (D + group + 2) 2^-24 (1 + small) sum |q| |mean|, and
  // under 1e-40 more where products underflow
  const float unit = (float)(D + a.group + 8) * 5.9604645e-8f * __uint_as_float(mmax_bits);
  for (int r = warp; r < nl; r += kSelWarps) {
    const int own = a.keep_own && (i0 + r) / a.block < live ? (i0 + r) / a.block : -1;
    const int first = a.keep_first < live ? a.keep_first : live;
    const int forced = first + (own >= first ? 1 : 0);
    if (!sel_row_fast(sc + r * NBS, live, a.topk, forced, own, first, unit * q1[r] + 1e-40f, out + (long long)r * a.topk) &&
        lane == 0)
      redo[atomicAdd(&redo_n, 1)] = r;
  }
  __syncthreads();
  // close rows: every score again in 64 bits, one row per warp in the scratch
  // that the 32-bit scores leave (a tile of two rows holds one 64-bit row)
  const int rn = redo_n;
  const int workers = TQ / 2 < kSelWarps ? TQ / 2 : kSelWarps;
  if (warp >= workers) return;
  double* s64 = reinterpret_cast<double*>(sc) + (long long)warp * NBS;
  for (int x = warp; x < rn; x += workers) {
    const int r = redo[x];
    for (int j = lane; j < live; j += 32) s64[j] = 0.0;
    for (int j0 = 0; j0 < live; j0 += 32) {
      const int j = j0 + lane;
      double acc = 0.0;
      for (int d = 0; d < D; ++d) {
        double qd = 0.0;
        for (int g = 0; g < a.group; ++g) qd += (double)rot_f32(qb[g * a.q.h + r * a.q.s + d]);
        if (j < live) acc += qd * (double)means[(long long)j * D + d];
      }
      if (j < live) s64[j] = isnan(acc) ? -INFINITY : acc;
    }
    __syncwarp();
    const int own = a.keep_own && (i0 + r) / a.block < live ? (i0 + r) / a.block : -1;
    const int first = a.keep_first < live ? a.keep_first : live;
    const int forced = first + (own >= first ? 1 : 0);
    sel_row_exact(s64, live, a.topk, forced, own, first, out + (long long)r * a.topk);
    __syncwarp();
  }
}

}  // namespace sb
