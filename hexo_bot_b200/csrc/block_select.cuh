// Block means of the keys, and the key blocks that each query keeps.
//
//   mean[j]  = sum of the block's live keys / their count
//   score    = (sum over the group's query heads of q) . mean[j]
//   kept     = forced blocks (leading ones, the query's own), then the best
//              scores; ties to the lowest index, NaN below everything
//
// The choice is the one 64-bit arithmetic on the given means makes. Scores are
// computed in 32 bits together with a bound on their error. Where the last
// kept and the first dropped score lie further apart than that, they settle the
// row; else the few scores near the border are computed again in 64 bits, and
// the whole row where many are near or one is not finite.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>

#include "ptx.cuh"
#include "rotary.cuh"

namespace sb {

constexpr int kSelMaxDim = 256;
constexpr int kSelMaxTopk = 64;
constexpr int kSelMaxBlocks = 16384;
constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelChunk = 64;  // blocks of a score chunk
constexpr float kSelTiny = 1e-40f;  // more than the squares of a row lose to underflow

struct HeadsView {
  const void* p;
  long long b, h, s;
};

// ---- block means ------------------------------------------------------------
// Sums run in 64 bits, so 16-bit keys add up without error and the mean is
// rounded once. WPU warps make a unit (one block of one head): a lane holds a
// VEC-wide channel chunk, the lanes of one chunk split the rows and are joined
// by shuffles, the warps of a unit through shared memory. Bound by HBM (the
// keys are read once); loads of a lane are issued four rows at a time.
constexpr int kMeansThreads = 128;

template <typename T, int VEC, int WPU>
__global__ __launch_bounds__(kMeansThreads) void block_means_kernel(HeadsView k, const int* __restrict__ kv_lens,
                                                                    int heads, int rows, int dim, int block, int nb,
                                                                    long long units, int chunk_lanes,
                                                                    float* __restrict__ out) {
  constexpr int UNITS = kMeansThreads / 32 / WPU;
  __shared__ double red[WPU > 1 ? WPU : 1][32 * VEC];
  using V = RotVec<T, VEC>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wu = warp % WPU;
  const long long u = (long long)blockIdx.x * UNITS + warp / WPU;
  if (u >= units) return;  // whole units: with WPU > 1 a CTA is one unit
  const int j = (int)(u % nb);
  const long long bh = u / nb;
  const int b = (int)(bh / heads), h = (int)(bh - (long long)b * heads);
  int len = kv_lens ? kv_lens[b] : rows;
  len = len < 0 ? 0 : len > rows ? rows : len;
  const int n = min(len - j * block, block);
  const int chunks = dim / VEC;
  const int strands = 32 / chunk_lanes;  // row strands of a warp
  const int cl = lane % chunk_lanes, step = strands * WPU;
  const T* base = (const T*)k.p + b * k.b + h * k.h + (long long)j * block * k.s;
  for (int c0 = 0; c0 < chunks; c0 += chunk_lanes) {
    const int c = c0 + cl;
    double acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.0;
    if (c < chunks) {
      for (int r0 = wu * strands + lane / chunk_lanes; r0 < n; r0 += 4 * step) {
        V v[4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
          v[x] = r0 + x * step < n ? *reinterpret_cast<const V*>(base + (r0 + x * step) * k.s + c * VEC) : V{};
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] += (double)rot_f32(v[x].v[e]);
      }
    }
    for (int m = chunk_lanes; m < 32; m <<= 1)
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], m);
    if (WPU > 1) {
      __syncthreads();
      if (lane < chunk_lanes)
#pragma unroll
        for (int e = 0; e < VEC; ++e) red[wu][lane * VEC + e] = acc[e];
      __syncthreads();
      if (wu == 0 && lane < chunk_lanes)
#pragma unroll
        for (int w = 1; w < WPU; ++w)
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] += red[w][lane * VEC + e];
    }
    if (wu == 0 && lane < chunk_lanes && c < chunks) {
      float* o = out + (bh * nb + j) * dim + c * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = n > 0 ? (float)(acc[e] / n) : 0.f;
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
  int q_vec;           // query rows may be read in 16-byte pieces
};

// One row's choice.
struct SelRow {
  int live, topk, own, first, forced;
  __device__ __forceinline__ SelRow(const SelArgs& a, int row, int live_blocks) {
    live = live_blocks;
    topk = a.topk;
    first = a.keep_first < live ? a.keep_first : live;
    own = a.keep_own && row / a.block < live ? row / a.block : -1;
    forced = first + (own >= first ? 1 : 0);
  }
  __device__ __forceinline__ bool is_forced(int j) const { return j < first || j == own; }
  __device__ __forceinline__ int want() const { return topk - forced; }  // among the others
};

// Order-preserving image of a float (larger float -> larger integer), NaN the
// lowest (1); 0 marks blocks that do not compete.
__device__ __forceinline__ uint32_t sel_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return isnan(f) ? 1u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sel_unkey(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Threads that settle a row together: a warp, or a whole CTA.
struct SelWarp {
  static constexpr int N = 32;
  __device__ __forceinline__ int id() const { return threadIdx.x & 31; }
  __device__ __forceinline__ unsigned add(unsigned v) const { return __reduce_add_sync(0xffffffffu, v); }
  __device__ __forceinline__ unsigned min(unsigned v) const { return __reduce_min_sync(0xffffffffu, v); }
  __device__ __forceinline__ unsigned max(unsigned v) const { return __reduce_max_sync(0xffffffffu, v); }
};
struct SelCta {
  static constexpr int N = kSelThreads;
  unsigned* s;  // shared [2][kSelWarps], used in turn: one barrier a join
  int turn = 0;
  __device__ __forceinline__ int id() const { return threadIdx.x; }
  template <typename F>
  __device__ __forceinline__ unsigned join(unsigned v, F f) {
    unsigned* p = s + turn * kSelWarps;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) p[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned r = p[0];
#pragma unroll
    for (int w = 1; w < kSelWarps; ++w) r = f(r, p[w]);
    return r;
  }
  __device__ __forceinline__ unsigned add(unsigned v) {
    return join(__reduce_add_sync(0xffffffffu, v), [](unsigned a, unsigned b) { return a + b; });
  }
  __device__ __forceinline__ unsigned min(unsigned v) {
    return join(__reduce_min_sync(0xffffffffu, v), [](unsigned a, unsigned b) { return a < b ? a : b; });
  }
  __device__ __forceinline__ unsigned max(unsigned v) {
    return join(__reduce_max_sync(0xffffffffu, v), [](unsigned a, unsigned b) { return a > b ? a : b; });
  }
};

// Keys of a row over its threads: PER in registers, or (PER = 0) images of the
// scores made anew at each visit. Thread t holds blocks t, t + N, ...
template <typename G, int PER>
struct SelKeys {
  uint32_t k[PER ? PER : 1];
  const float* s;
  const SelRow& r;
  int id;
  __device__ __forceinline__ uint32_t image(int j) const { return j < r.live && !r.is_forced(j) ? sel_key(s[j]) : 0u; }
  __device__ __forceinline__ SelKeys(const float* s_, const SelRow& r_, int id_) : s(s_), r(r_), id(id_) {
    if (PER)
#pragma unroll
      for (int x = 0; x < PER; ++x) k[x] = image(id + x * G::N);
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if (PER) {
#pragma unroll
      for (int x = 0; x < PER; ++x) f(k[x], id + x * G::N);
    } else {
      for (int j = id; j < r.live; j += G::N) f(image(j), j);
    }
  }
};

enum SelCase { SEL_DONE, SEL_BAND, SEL_ALL };

// Where a row stands by its 32-bit scores (each within `err` of its 64-bit
// value). SEL_DONE: kept are the forced blocks and keys >= lo. SEL_BAND: kept
// for certain are keys > hi, certainly dropped keys < lo; `sure` counts the
// former, `band` the keys between, from which the rest is chosen in 64 bits.
// SEL_ALL: a score is not finite or the band is long; everything in 64 bits.
template <typename G, int PER>
__device__ __forceinline__ SelCase sel_place(G& g, const SelKeys<G, PER>& keys, const SelRow& r, float err,
                                             uint32_t& lo, uint32_t& hi, int& sure, int& band) {
  const int want = r.want();
  lo = 1;
  hi = 0xffffffffu;
  if (want >= r.live - r.forced) return SEL_DONE;
  if (want <= 0) {
    lo = 0xffffffffu;
    return SEL_DONE;
  }
  uint32_t most = 0, least = 0xffffffffu;
  keys.each([&](uint32_t k, int) {
    if (k) {
      most = k > most ? k : most;
      least = k < least ? k : least;
    }
  });
  most = g.max(most);
  least = g.min(least);
  if (!(most < sel_key(INFINITY) && least > sel_key(-INFINITY)) || !isfinite(err)) return SEL_ALL;
  // a threshold that exactly `want` keys reach, by halving the range of the
  // scores; where that fails (scores that agree in most of their bits) the
  // largest one that at least `want` keys reach, bit by bit
  const int top = 31 - __clz(most ^ least);  // -1: all keys equal
  uint32_t t = top < 0 ? least : most & ~((2u << top) - 1u);
  bool exact = false;
  float f0 = sel_unkey(least), f1 = sel_unkey(most);
  for (int step = 0; step < 16 && !exact; ++step) {
    const float mid = 0.5f * f0 + 0.5f * f1;
    const uint32_t cand = sel_key(mid);
    unsigned c = 0;
    keys.each([&](uint32_t k, int) { c += k >= cand; });
    c = g.add(c);
    exact = c == (unsigned)want;
    if (exact) t = cand;
    if (c > (unsigned)want) f0 = mid;
    else f1 = mid;
  }
  for (int bit = top; bit >= 0 && !exact; --bit) {
    const uint32_t cand = t | (1u << bit);
    unsigned c = 0;
    keys.each([&](uint32_t k, int) { c += k >= cand; });
    c = g.add(c);
    if (c >= (unsigned)want) t = cand;
    exact = c == (unsigned)want;
  }
  // the smallest kept and the largest dropped key
  uint32_t kept = 0xffffffffu, dropped = 0;
  unsigned c = 0;
  keys.each([&](uint32_t k, int) {
    if (k >= t) {
      kept = k < kept ? k : kept;
      ++c;
    } else {
      dropped = k > dropped ? k : dropped;
    }
  });
  kept = g.min(kept);
  dropped = g.max(dropped);
  c = g.add(c);
  const float kf = sel_unkey(kept);
  if (c == (unsigned)want && kf - sel_unkey(dropped) > 2.f * err) {
    lo = kept;
    return SEL_DONE;
  }
  // the want-th largest 64-bit score lies within err of kf
  lo = sel_key(kf - 2.1f * err);
  hi = sel_key(kf + 2.1f * err);
  unsigned over = 0, in = 0;
  keys.each([&](uint32_t k, int) {
    over += k > hi;
    in += k >= lo && k <= hi;
  });
  sure = (int)g.add(over);
  band = (int)g.add(in);
  return band <= 32 ? SEL_BAND : SEL_ALL;
}

// 64-bit scores of up to four blocks, by a warp: lanes over the channels.
template <typename T>
__device__ __forceinline__ void sel_score64(const SelArgs& a, const T* q, const float* (&mean)[4], double (&s)[4]) {
#pragma unroll
  for (int y = 0; y < 4; ++y) s[y] = 0.0;
#pragma unroll 4
  for (int d = threadIdx.x & 31; d < a.dim; d += 32) {
    float m[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) m[y] = mean[y] ? mean[y][d] : 0.f;
    double x = 0.0;
#pragma unroll 4
    for (int g = 0; g < a.group; ++g) x += (double)rot_f32(q[g * a.q.h + d]);
#pragma unroll
    for (int y = 0; y < 4; ++y) s[y] += x * (double)m[y];
  }
  for (int m = 16; m; m >>= 1)
#pragma unroll
    for (int y = 0; y < 4; ++y) s[y] += __shfl_xor_sync(0xffffffffu, s[y], m);
#pragma unroll
  for (int y = 0; y < 4; ++y)
    if (isnan(s[y])) s[y] = -INFINITY;
}
// All of a row's 64-bit scores, blocks j0, j0 + 4 step, ... to s, by a warp.
template <typename T>
__device__ __forceinline__ void sel_scores64(const SelArgs& a, const T* q, const float* means, int j0, int step, int live,
                                             double* s) {
  for (; j0 < live; j0 += 4 * step) {
    const float* mean[4];
    double v[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) mean[y] = j0 + y * step < live ? means + (long long)(j0 + y * step) * a.dim : nullptr;
    sel_score64(a, q, mean, v);
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (mean[y] && (threadIdx.x & 31) == 0) s[j0 + y * step] = v[y];
  }
}

// SEL_BAND by a warp: `members` (shared, ascending, n of them) hold the band's
// blocks; returns the mask of those that are kept: the `need` largest 64-bit
// scores, ties to the lowest index.
template <typename T>
__device__ __forceinline__ uint32_t sel_band(const SelArgs& a, const T* q, const float* means, const int* members, int n,
                                             int need) {
  const int lane = threadIdx.x & 31;
  double mine = 0.0;
  for (int c = 0; c < n; c += 4) {
    const float* mean[4];
    double v[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) mean[y] = c + y < n ? means + (long long)members[c + y] * a.dim : nullptr;
    sel_score64(a, q, mean, v);
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (lane == c + y) mine = v[y];
  }
  int rank = 0;
  for (int c = 0; c < n; ++c) {
    const double o = __shfl_sync(0xffffffffu, mine, c);
    rank += o > mine || (o == mine && c < lane);
  }
  return __ballot_sync(0xffffffffu, lane < n && rank < need);
}

// Writes kept blocks among [j0, j1) in ascending order from place n on, by a
// warp; returns the next place.
template <typename F>
__device__ __forceinline__ int sel_write(int* out, int j0, int j1, int n, int topk, F kept) {
  const int lane = threadIdx.x & 31;
  for (; j0 < j1; j0 += 32) {
    const int j = j0 + lane;
    const bool k = j < j1 && kept(j);
    const uint32_t m = __ballot_sync(0xffffffffu, k);
    const int at = n + __popc(m & ((1u << lane) - 1u));
    if (out && k && at < topk) out[at] = j;
    n += __popc(m);
  }
  return n;
}
__device__ __forceinline__ void sel_fill(int* out, int n, int topk) {
  for (int i = n + (threadIdx.x & 31); i < topk; i += 32) out[i] = -1;
}

// A row of 64-bit scores s (a taken block is marked by NaN), by a warp.
__device__ __forceinline__ void sel_row_exact(double* s, const SelRow& r, int* out) {
  const int lane = threadIdx.x & 31;
  const int want = min(r.topk, r.live) - r.forced;
  for (int x = 0; x < want; ++x) {
    double best = 0.0;
    int at = 0x7fffffff;
    for (int j = lane; j < r.live; j += 32)
      if (!r.is_forced(j) && !isnan(s[j]) && (at == 0x7fffffff || s[j] > best)) {
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
  const int n = sel_write(out, 0, r.live, 0, r.topk, [&](int j) { return r.is_forced(j) || isnan(s[j]); });
  sel_fill(out, n, r.topk);
}

// One row by a warp from its 32-bit scores; false: all of it in 64 bits.
template <typename T, int PER>
__device__ __forceinline__ bool sel_row_fast(const SelArgs& a, const float* s, const SelRow& r, float err, const T* q,
                                             const float* means, int* members, int* out) {
  SelWarp g;
  SelKeys<SelWarp, PER> keys(s, r, g.id());
  uint32_t lo, hi;
  int sure = 0, band = 0;
  const SelCase c = sel_place(g, keys, r, err, lo, hi, sure, band);
  if (c == SEL_ALL) return false;
  uint32_t won = 0;
  if (c == SEL_BAND) {
    sel_write(members, 0, r.live, 0, 32, [&](int j) {
      const uint32_t k = keys.image(j);
      return k >= lo && k <= hi;
    });
    __syncwarp();
    won = sel_band(a, q, means, members, band, r.want() - sure);
    __syncwarp();
    if (g.id() < band && !(won >> g.id() & 1)) members[g.id()] = -1;
    __syncwarp();
  }
  int seen = 0;  // band members before this lane's chunk: they come in the same ascending order
  int n = 0;
  const int lane = g.id();
  for (int j0 = 0; j0 < r.live; j0 += 32) {
    const int j = j0 + lane;
    const uint32_t k = keys.image(j);
    bool kept = j < r.live && (r.is_forced(j) || (c == SEL_BAND ? k > hi : k >= lo));
    if (c == SEL_BAND) {
      const bool in = k >= lo && k <= hi;
      const uint32_t m = __ballot_sync(0xffffffffu, in);
      if (in) kept = members[seen + __popc(m & ((1u << lane) - 1u))] >= 0;
      seen += __popc(m);
    }
    const uint32_t m = __ballot_sync(0xffffffffu, kept);
    const int at = n + __popc(m & ((1u << lane) - 1u));
    if (kept && at < r.topk) out[at] = j;
    n += __popc(m);
  }
  sel_fill(out, n, r.topk);
  __syncwarp();
  return true;
}

// 32 / LPR rows by a warp, LPR lanes a row, scores in registers (live <= LPR PER).
// Lanes of a row whose 32-bit scores settle it write it; returns whether this
// lane's row is settled. `on`: this lane's row exists. The border is looked for
// by halving the range of the scores until as many as wanted lie above.
template <int PER, int LPR>
__device__ __forceinline__ bool sel_rows(const float* s, const SelRow& r, float err, bool on, int* out) {
  const int lane = threadIdx.x & 31, id = lane & (LPR - 1), shift = lane & ~(LPR - 1);
  constexpr uint32_t kRow = (1u << LPR) - 1u;  // a row's lanes in a ballot
  const int want = r.want();
  float v[PER];
  float most = -INFINITY, least = INFINITY;
  bool odd = !(err < INFINITY);
#pragma unroll
  for (int x = 0; x < PER; ++x) {
    const int j = id + LPR * x;
    v[x] = -INFINITY;  // blocks that do not compete are never above the border
    if (j < r.live && !r.is_forced(j)) {
      v[x] = s[j];
      odd |= !(fabsf(v[x]) < INFINITY);
      most = fmaxf(most, v[x]);
      least = fminf(least, v[x]);
    }
  }
  odd = (__ballot_sync(0xffffffffu, odd) >> shift & kRow) != 0;
#pragma unroll
  for (int m = 1; m < LPR; m <<= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, m));
    least = fminf(least, __shfl_xor_sync(0xffffffffu, least, m));
  }
  const bool all = want >= r.live - r.forced, search = on && !all && want > 0;
  bool busy = search && !odd;
  float t = 0.f;
  bool exact = false;
#pragma unroll 1
  for (int step = 0; step < 26 && __any_sync(0xffffffffu, busy); ++step) {
    const float mid = 0.5f * least + 0.5f * most;
    int c = 0;
#pragma unroll
    for (int x = 0; x < PER; ++x) c += v[x] >= mid;
#pragma unroll
    for (int m = 1; m < LPR; m <<= 1) c += __shfl_xor_sync(0xffffffffu, c, m);
    if (busy) {
      if (c == want) {
        exact = true;
        busy = false;
        t = mid;
      }
      if (c > want) least = mid;
      else most = mid;
    }
  }
  // the smallest kept and the largest dropped score
  float kept = INFINITY, dropped = -INFINITY;
#pragma unroll
  for (int x = 0; x < PER; ++x) {
    const bool in = v[x] >= t;
    kept = in ? fminf(kept, v[x]) : kept;
    dropped = in ? dropped : fmaxf(dropped, v[x]);
  }
#pragma unroll
  for (int m = 1; m < LPR; m <<= 1) {
    kept = fminf(kept, __shfl_xor_sync(0xffffffffu, kept, m));
    dropped = fmaxf(dropped, __shfl_xor_sync(0xffffffffu, dropped, m));
  }
  const bool settled = !search || (exact && kept - dropped > 2.f * err);
  const bool write = on && settled;
  int n = 0;
#pragma unroll
  for (int x = 0; x < PER; ++x) {
    const int j = id + LPR * x;
    const bool in = j < r.live && (all || r.is_forced(j) || (search && v[x] >= t));
    const uint32_t m = __ballot_sync(0xffffffffu, in) >> shift & kRow;
    const int at = n + __popc(m & ((1u << id) - 1u));
    if (write && in && at < r.topk) out[at] = j;
    n += __popc(m);
  }
  if (write)
    for (int x = n + id; x < r.topk; x += LPR) out[x] = -1;
  return settled;
}

// Shared memory of a CTA:
//   scores [tile][stride] fp32, later 64-bit scores, one row a warp
//   summed queries [2][tile][dp + 8] and a chunk of means [2][64][dp + 8] as
//   bf16 pairs (x = hi + mid + rest, |rest| <= 2^-18 |x|), the rows' squares
//   two lists of rows left to do
// stride: an odd multiple of 8 (neighbouring rows meet distinct banks); rows of
// dp + 8: an odd number of 16-byte chunks, so ldmatrix meets every bank once.
__host__ __device__ inline int sel_stride(int nb) { return ((nb + 7) / 8 | 1) * 8; }
__host__ __device__ inline int sel_dp(int dim) { return (dim + 15) / 16 * 16; }
__host__ __device__ inline int sel_smem_bytes(int tile, int nb, int dim) {
  return tile * sel_stride(nb) * 4 + 2 * (max(tile, 16) + kSelChunk) * (sel_dp(dim) + 8) * 2 + tile * 12;
}

// Error of a 32-bit score, relative to ||q|| ||mean|| (||q||: of the sums of the
// heads' magnitudes). Matrix form: three products of bf16 pairs lose mid mid and
// both rests, 3 2^-18 with the rounding of the parts, and the sums of 3 dp / 16
// steps 2^-22 each. Plain form (few queries): products are added four at a time
// and the groups in turn, D / 4 + group + 6 roundings. Both with some to spare.
__device__ __forceinline__ float sel_unit_mma(const SelArgs& a) {
  return 3.5f * 3.8146973e-6f + (float)(3 * a.dim / 16 + a.group + 16) * 2.3841858e-7f;
}
__device__ __forceinline__ float sel_unit(const SelArgs& a) {
  return (float)(a.dim / 4 + a.group + 12) * 5.9604645e-8f;
}

// x as bf16 hi + mid, eight channels to 16 bytes each.
__device__ __forceinline__ void sel_split8(const float (&x)[8], __nv_bfloat16* hi, __nv_bfloat16* mid) {
  RotVec<__nv_bfloat16, 8> h, m;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    h.v[e] = __float2bfloat16_rn(x[e]);
    m.v[e] = __float2bfloat16_rn(x[e] - __bfloat162float(h.v[e]));
  }
  *reinterpret_cast<RotVec<__nv_bfloat16, 8>*>(hi) = h;
  *reinterpret_cast<RotVec<__nv_bfloat16, 8>*>(mid) = m;
}

// PER > 0: rows of up to LPR PER blocks, LPR lanes a row (the fewer, the fewer
// instructions a row); 0: a warp a row.
template <typename T, int PER, int LPR>
__global__ __launch_bounds__(kSelThreads, 3) void block_select_kernel(const SelArgs a) {
  extern __shared__ __align__(16) char sel_smem[];
  const int D = a.dim, DP = sel_dp(D), RS = DP + 8, NBS = sel_stride(a.nb), TQ = a.tile, TQ16 = max(TQ, 16);
  float* sc = reinterpret_cast<float*>(sel_smem);
  __nv_bfloat16* qhi = reinterpret_cast<__nv_bfloat16*>(sc + TQ * NBS);
  __nv_bfloat16 *qmid = qhi + TQ16 * RS, *mhi = qmid + TQ16 * RS, *mmid = mhi + kSelChunk * RS;
  float* qn = reinterpret_cast<float*>(mmid + kSelChunk * RS);
  int* todo = reinterpret_cast<int*>(qn + TQ);
  int* redo = todo + TQ;
  __shared__ int todo_n, redo_n;
  __shared__ uint32_t mmax_bits;
  __shared__ int members[kSelWarps][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bh32 = blockIdx.x / a.tiles, tile = blockIdx.x - bh32 * a.tiles;
  const long long bh = bh32;
  const int b = bh32 / a.kv_heads, h = bh32 - b * a.kv_heads;
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
    todo_n = redo_n = 0;
    mmax_bits = 0;
  }
  for (int i = tid; i < (nq - nl) * a.topk; i += kSelThreads) out[(long long)nl * a.topk + i] = -1;
  if (nl == 0) return;

  // the group's summed queries as bf16 pairs, and the squares of the sums of
  // magnitudes; items of eight channels, two a thread and step so that several
  // loads are in flight; 2^cl lanes a row, joined by shuffles
  const T* qb = (const T*)a.q.p + b * a.q.b + (long long)h * a.group * a.q.h + (long long)i0 * a.q.s;
  const bool q_wide = a.q_vec != 0;
  const int cl = 32 - __clz(DP / 8 - 1);
  for (int it0 = tid; it0 < TQ16 << cl; it0 += 2 * kSelThreads) {
    float x[2][8], m[2][8];
    int rr[2], cc[2];
    bool on[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int it = it0 + y * kSelThreads;
      rr[y] = it >> cl;
      cc[y] = (it - (rr[y] << cl)) * 8;
      on[y] = rr[y] < nl;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[y][e] = m[y][e] = 0.f;
    }
    if (q_wide) {  // D is a multiple of 8, rows are 16-byte aligned
      constexpr int V = 16 / sizeof(T), NV = 8 / V;
#pragma unroll 4
      for (int g = 0; g < a.group; ++g) {
        RotVec<T, V> w[2][NV];
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int z = 0; z < NV; ++z)
            w[y][z] = on[y] && cc[y] < D
                          ? *reinterpret_cast<const RotVec<T, V>*>(qb + g * a.q.h + rr[y] * a.q.s + cc[y] + z * V)
                          : RotVec<T, V>{};
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = rot_f32(w[y][e / V].v[e % V]);
            x[y][e] += v;
            m[y][e] += fabsf(v);
          }
      }
    } else {
      for (int g = 0; g < a.group; ++g)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = on[y] && cc[y] + e < D ? rot_f32(qb[g * a.q.h + rr[y] * a.q.s + cc[y] + e]) : 0.f;
            x[y][e] += v;
            m[y][e] += fabsf(v);
          }
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      float n2 = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) n2 += m[y][e] * m[y][e];
      for (int z = 1; z < 1 << cl; z <<= 1) n2 += __shfl_xor_sync(0xffffffffu, n2, z);
      if (cc[y] == 0 && rr[y] < TQ) qn[rr[y]] = n2 + kSelTiny;
      if (rr[y] < TQ16 && cc[y] < DP) sel_split8(x[y], qhi + rr[y] * RS + cc[y], qmid + rr[y] * RS + cc[y]);
    }
  }
  const bool m_wide = D % 4 == 0 && ((uintptr_t)means & 15) == 0;
  for (int j0 = 0; j0 < live; j0 += kSelChunk) {
    const int nj = live - j0 < kSelChunk ? live - j0 : kSelChunk;
    __syncthreads();
    float most = 0.f;
    for (int it0 = tid; it0 < kSelChunk << cl; it0 += 2 * kSelThreads) {
      float x[2][8];
      int rr[2], cc[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int it = it0 + y * kSelThreads;
        rr[y] = it >> cl;
        cc[y] = (it - (rr[y] << cl)) * 8;
        const bool on = rr[y] < nj;
        const float* src = means + (long long)(j0 + rr[y]) * D + cc[y];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          if (m_wide) {
            const float4 v = on && cc[y] + 4 * z < D ? *reinterpret_cast<const float4*>(src + 4 * z) : make_float4(0.f, 0.f, 0.f, 0.f);
            x[y][4 * z] = v.x; x[y][4 * z + 1] = v.y; x[y][4 * z + 2] = v.z; x[y][4 * z + 3] = v.w;
          } else {
#pragma unroll
            for (int e = 4 * z; e < 4 * z + 4; ++e) x[y][e] = on && cc[y] + e < D ? src[e] : 0.f;
          }
        }
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float n2 = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) n2 += x[y][e] * x[y][e];
        for (int z = 1; z < 1 << cl; z <<= 1) n2 += __shfl_xor_sync(0xffffffffu, n2, z);
        most = fmaxf(most, n2 >= 0.f ? n2 + kSelTiny : INFINITY);
        if (rr[y] < kSelChunk && cc[y] < DP) sel_split8(x[y], mhi + rr[y] * RS + cc[y], mmid + rr[y] * RS + cc[y]);
      }
    }
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    if (lane == 0) atomicMax(&mmax_bits, bits);  // values >= 0: bits order as they do
    __syncthreads();
    // units of 16 queries x 32 blocks: hi hi + hi mid + mid hi
    for (int unit = warp; unit < TQ16 / 16 * 2; unit += kSelWarps) {
      const int r0 = unit / 2 * 16, c0 = unit % 2 * 32;
      if (r0 >= nl || c0 >= nj) continue;
      float acc[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
      for (int kk = 0; kk < DP; kk += 16) {
        uint32_t ah[4], am[4];
        const int qa = (r0 + (lane & 15)) * RS + kk + (lane >> 4) * 8;
        ldmatrix_x4(ah, smem_u32(qhi + qa));
        ldmatrix_x4(am, smem_u32(qmid + qa));
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          uint32_t bh4[4], bm4[4];
          const int ma = (c0 + 16 * n + (lane & 7) + ((lane >> 4) << 3)) * RS + kk + ((lane >> 3) & 1) * 8;
          ldmatrix_x4(bh4, smem_u32(mhi + ma));
          ldmatrix_x4(bm4, smem_u32(mmid + ma));
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t bh2[2] = {bh4[2 * y], bh4[2 * y + 1]}, bm2[2] = {bm4[2 * y], bm4[2 * y + 1]};
            MmaTraits<__nv_bfloat16>::mma(acc[2 * n + y], am, bh2);
            MmaTraits<__nv_bfloat16>::mma(acc[2 * n + y], ah, bm2);
            MmaTraits<__nv_bfloat16>::mma(acc[2 * n + y], ah, bh2);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = r0 + (lane >> 2) + 8 * (e >> 1), c = c0 + 8 * n + 2 * (lane & 3) + (e & 1);
          if (r < nl && c < nj) sc[r * NBS + j0 + c] = acc[n][e];
        }
    }
  }
  __syncthreads();
  const float mmax = sqrtf(__uint_as_float(mmax_bits)), unit = sel_unit_mma(a) * mmax;
  // parts below the smallest normal number may be lost: 1e-34 of the norms covers them
  auto err_of = [&](int r) {
    const float q = sqrtf(qn[r]);
    return unit * q + 1e-34f * (mmax + q) + 1e-40f;
  };
  if constexpr (PER > 0) {
    for (int r0 = warp * (32 / LPR); r0 < nl; r0 += kSelThreads / LPR) {
      const int r = r0 + lane / LPR;
      const bool on = r < nl;
      const int rr = on ? r : 0;
      const SelRow row(a, i0 + rr, live);
      const bool done = sel_rows<PER, LPR>(sc + rr * NBS, row, err_of(rr), on, out + (long long)rr * a.topk);
      if (on && !done && lane % LPR == 0) todo[atomicAdd(&todo_n, 1)] = r;
    }
    __syncthreads();
  }
  const int rows = PER > 0 ? todo_n : nl;
  for (int x = warp; x < rows; x += kSelWarps) {
    const int r = PER > 0 ? todo[x] : x;
    const SelRow row(a, i0 + r, live);
    if (!sel_row_fast<T, 0>(a, sc + r * NBS, row, err_of(r), qb + r * a.q.s, means, members[warp],
                            out + (long long)r * a.topk) &&
        lane == 0)
      redo[atomicAdd(&redo_n, 1)] = r;
  }
  __syncthreads();
  // the remaining rows: every score in 64 bits, one row per warp in the scratch
  // that the 32-bit scores leave (a tile of two rows holds one 64-bit row)
  const int rn = redo_n;
  const int workers = TQ / 2 < kSelWarps ? TQ / 2 : kSelWarps;
  if (warp >= workers) return;
  double* s64 = reinterpret_cast<double*>(sc) + (long long)warp * NBS;
  for (int x = warp; x < rn; x += workers) {
    const int r = redo[x];
    sel_scores64(a, qb + r * a.q.s, means, 0, 1, live, s64);
    __syncwarp();
    sel_row_exact(s64, SelRow(a, i0 + r, live), out + (long long)r * a.topk);
    __syncwarp();
  }
}

// ---- selection, few queries ---------------------------------------------------
// A cluster of CTAs per row: every CTA scores its share of the blocks straight
// from global memory (a warp reads whole mean rows, eight in flight) into the
// shared memory of the cluster's first CTA, which settles the row with all of
// its threads. Bound by the read of the means.
constexpr int kSelFewCluster = 8;

__host__ __device__ inline int sel_few_smem_bytes(int nb) { return (nb + (nb & 1)) * 12; }

template <typename T, int PER>
__global__ __launch_bounds__(kSelThreads) void block_select_few_kernel(const SelArgs a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) char sel_smem[];
  float* sc = reinterpret_cast<float*>(sel_smem);                                        // [nb], CTA 0's
  double* s64 = reinterpret_cast<double*>(sel_smem + (size_t)(a.nb + (a.nb & 1)) * 4);  // [nb], CTA 0's
  __shared__ __align__(16) float qs[kSelMaxDim];
  __shared__ unsigned red[2 * kSelWarps];
  __shared__ uint32_t mmax_bits;  // CTA 0's
  __shared__ int members[32], counts[kSelWarps];
  __shared__ uint32_t won_sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const long long u = blockIdx.x / C;
  const int i = (int)(u % a.q_rows);
  const long long bh = u / a.q_rows;
  const int b = (int)(bh / a.kv_heads), h = (int)(bh - (long long)b * a.kv_heads);
  int kv = a.kv_lens ? a.kv_lens[b] : a.kv_rows;
  kv = kv < 0 ? 0 : kv > a.kv_rows ? a.kv_rows : kv;
  const bool on = !a.q_lens || i < a.q_lens[b];
  const int D = a.dim, live = on ? (kv + a.block - 1) / a.block : 0;
  const T* q = (const T*)a.q.p + b * a.q.b + (long long)h * a.group * a.q.h + (long long)i * a.q.s;
  const float* means = a.means + bh * a.nb * D;
  if (tid == 0) mmax_bits = 0;
  float n2 = 0.f;
  for (int d = tid; d < D; d += kSelThreads) {
    float s = 0.f, m = 0.f;
    for (int g = 0; g < a.group; ++g) {
      const float v = rot_f32(q[g * a.q.h + d]);
      s += v;
      m += fabsf(v);
    }
    qs[d] = s;
    n2 += m * m;
  }
  cluster.sync();  // CTA 0's maximum is set to zero
  float* sc0 = cluster.map_shared_rank(sc, 0);
  uint32_t* mm0 = cluster.map_shared_rank(&mmax_bits, 0);
  float mx = 0.f;
  if (D % 4 == 0 && ((uintptr_t)means & 15) == 0) {
    // LB lanes a mean row (16 bytes a lane and step), 32 / LB rows a warp and step
    int LB = 1;
    while (LB < 32 && LB * 4 < D) LB <<= 1;
    const int per = 32 / LB, sub = lane / LB, l = lane % LB;
    const int stride = C * kSelWarps * per;
    for (int j0 = (rank * kSelWarps + warp) * per; j0 < live; j0 += 8 * stride) {
      float dot[8], nn[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) dot[x] = nn[x] = 0.f;
      for (int d = l * 4; d < D; d += LB * 4) {
        float4 m[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int j = j0 + sub + x * stride;
          m[x] = j < live ? *reinterpret_cast<const float4*>(means + (long long)j * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const float4 v = *reinterpret_cast<const float4*>(qs + d);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          dot[x] += fmaf(v.w, m[x].w, fmaf(v.z, m[x].z, fmaf(v.y, m[x].y, v.x * m[x].x)));
          nn[x] += fmaf(m[x].w, m[x].w, fmaf(m[x].z, m[x].z, fmaf(m[x].y, m[x].y, m[x].x * m[x].x)));
        }
      }
      for (int m = 1; m < LB; m <<= 1) {
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          dot[x] += __shfl_xor_sync(0xffffffffu, dot[x], m);
          nn[x] += __shfl_xor_sync(0xffffffffu, nn[x], m);
        }
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int j = j0 + sub + x * stride;
        if (l == 0 && j < live) sc0[j] = dot[x];
        mx = fmaxf(mx, nn[x] >= 0.f ? nn[x] + kSelTiny : INFINITY);
      }
    }
  } else {
    for (int j = rank * kSelWarps + warp; j < live; j += C * kSelWarps) {
      float dot = 0.f, nn = 0.f;
      for (int d = lane; d < D; d += 32) {
        const float m = means[(long long)j * D + d];
        dot += qs[d] * m;
        nn += m * m;
      }
      for (int m = 16; m; m >>= 1) {
        dot += __shfl_xor_sync(0xffffffffu, dot, m);
        nn += __shfl_xor_sync(0xffffffffu, nn, m);
      }
      if (lane == 0) sc0[j] = dot;
      mx = fmaxf(mx, nn >= 0.f ? nn + kSelTiny : INFINITY);
    }
  }
  for (int m = 16; m; m >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, m));
  if (lane == 0) atomicMax(mm0, __float_as_uint(mx));
  cluster.sync();
  if (rank != 0) return;

  SelCta g{red};
  for (int m = 16; m; m >>= 1) n2 += __shfl_xor_sync(0xffffffffu, n2, m);
  n2 = __uint_as_float(g.join(__float_as_uint(n2), [](unsigned x, unsigned y) {
    return __float_as_uint(__uint_as_float(x) + __uint_as_float(y));
  }));
  const float err = sel_unit(a) * sqrtf(__uint_as_float(mmax_bits)) * sqrtf(n2 + kSelTiny) + 1e-40f;
  const SelRow row(a, i, live);
  int* out = a.out + (bh * a.q_rows + i) * a.topk;
  SelKeys<SelCta, PER> keys(sc, row, tid);
  uint32_t lo, hi;
  int sure = 0, band = 0;
  const SelCase c = sel_place(g, keys, row, err, lo, hi, sure, band);
  if (c == SEL_ALL) {
    sel_scores64(a, q, means, warp, kSelWarps, live, s64);
    __syncthreads();
    if (warp == 0) sel_row_exact(s64, row, out);
    return;
  }
  // each warp writes a range of blocks; the warps' counts give the places
  const int span = ((live + kSelWarps - 1) / kSelWarps + 31) / 32 * 32;
  const int j0 = min(live, warp * span), j1 = min(live, j0 + span);
  if (c == SEL_BAND) {
    if (warp == 0) {
      sel_write(members, 0, live, 0, 32, [&](int j) {
        const uint32_t k = keys.image(j);
        return k >= lo && k <= hi;
      });
      __syncwarp();
      const uint32_t won = sel_band(a, q, means, members, band, row.want() - sure);
      if (lane == 0) won_sh = won;
    }
    __syncthreads();
  }
  auto kept = [&](int j) {
    if (row.is_forced(j)) return true;
    const uint32_t k = keys.image(j);
    if (c != SEL_BAND) return k >= lo;
    if (k > hi) return true;
    if (k < lo) return false;
    for (int x = 0; x < band; ++x)
      if (members[x] == j) return (won_sh >> x & 1) != 0;
    return false;
  };
  const int mine = sel_write(nullptr, j0, j1, 0, a.topk, kept);
  if (lane == 0) counts[warp] = mine;
  __syncthreads();
  int n = 0;
  for (int w = 0; w < warp; ++w) n += counts[w];
  n = sel_write(out, j0, j1, n, a.topk, kept);
  if (warp == kSelWarps - 1) sel_fill(out, n, a.topk);
}

}  // namespace sb
