// Rotary positions with several axes, alone or behind an RMS norm of every
// query and key head, and the gradients of the latter.
//
//   pair p of axis a(p):  angle = coord[a(p)] * freq[p],
//   (y1, y2) = (x1 cos - x2 sin, x2 cos + x1 sin)          (inverse: -sin)
//   norm:      x^ = x rstd, rstd = (mean(x^2) + eps)^-1/2,  y = R (w x^)
//   backward:  g = R^T dy, dw = sum g x^, dx = rstd (w g - x^ mean(w g x^))
//
// A CTA owns a tile of tokens. It first fills a shared table with the cos and
// sin of every (token, pair) once, which all heads of the token then use; the
// angle is reduced in 64 bits as turns (coord * freq / 2 pi minus its nearest
// integer), so positions of any size keep fp32 accuracy, and only the
// remainder goes through the 32-bit sincospi. Then its threads run over
// (token, head, lane) items: a lane holds VEC pairs of one head (both members
// of a pair in the same thread), L lanes make a head and sum its squares by
// shuffles. Rows are read once and written once, in 16-byte accesses where
// shapes and strides allow (VEC below), so the kernels are bound by HBM.
//
// Channels: half pairing (p, P + p), adjacent pairing (2p, 2p + 1), P pairs in
// all; channels from 2P on are not turned. Leading `prefix` rows of each
// sequence have no coordinates and are not turned either.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/shrimp_b200.h"

namespace sb {

constexpr int kRotThreads = 256;
constexpr int kRotMaxDim = 256;
constexpr int kRotMaxAxes = 4;
constexpr int kRotMaxTile = 64;         // tokens of a tile
constexpr int kRotTableBytes = 16384;   // cos / sin pairs of a tile
constexpr int kRotMaxGrid = 148 * 4;    // CTAs of the gradient kernel (one partial weight gradient each)

enum RotOp { ROT_TURN = 0, ROT_NORM = 1, ROT_NORM_BWD = 2 };

// One strided (batch, head, row) tensor set: queries and keys.
struct RotArgs {
  const void* x[2];
  const void* dy[2];           // backward only
  void* y[2];                  // outputs (backward: dx)
  long long xs[2][3], gs[2][3], ys[2][3];
  int heads[2];
  const void* w[2];            // norm weights or null (= 1)
  int w_dtype;
  float* dw_part;              // backward: [grid][2][D]
  const void* coords;
  int coord_dtype, axes;
  long long cs[3];             // batch, row, axis
  const double* freqs;
  int axis_end[kRotMaxAxes];   // exclusive end of each axis' pairs
  int pairs, prefix, batch, rows, dim, items, lanes_log2;
  float sign, eps, inv_dim;
  int tile, num_tiles;
};

template <typename T>
__device__ __forceinline__ float rot_f32(T v) { return static_cast<float>(v); }
template <typename T>
__device__ __forceinline__ T rot_cast(float v) { return static_cast<T>(v); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) RotVec {
  T v[VEC];
};

__device__ __forceinline__ double rot_coord(const void* p, int dtype, long long i) {
  switch (dtype) {
    case SB_I64: return (double)((const long long*)p)[i];
    case SB_I32: return (double)((const int*)p)[i];
    case SB_I16: return (double)((const short*)p)[i];
    default: return (double)((const float*)p)[i];
  }
}
__device__ __forceinline__ float rot_weight(const void* p, int dtype, int i) {
  if (!p) return 1.f;
  switch (dtype) {
    case SB_F32: return ((const float*)p)[i];
    case SB_F16: return __half2float(((const __half*)p)[i]);
    default: return __bfloat162float(((const __nv_bfloat16*)p)[i]);
  }
}

// Slots of one lane: NI items of two VEC-wide chunks. Item i of a head:
//   half pairing:  i < P / VEC: chunks at i * VEC and P + i * VEC (turned);
//                  else two chunks of the unturned rest (the second may be missing)
//   adjacent:      channels [2 VEC i, 2 VEC (i + 1)), every pair inside.
template <typename T, int VEC, int NI, bool ADJ, int OP>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(const RotArgs a) {
  extern __shared__ __align__(16) char rot_smem[];
  float2* table = reinterpret_cast<float2*>(rot_smem);                       // [tile][pairs]
  long long* off = reinterpret_cast<long long*>(rot_smem + kRotTableBytes);  // [tile][2][3]
  float* wsm = reinterpret_cast<float*>(off + kRotMaxTile * 6);              // [2][dim]
  using V = RotVec<T, VEC>;
  const int tid = threadIdx.x;
  const int L = 1 << a.lanes_log2, lane = tid & (L - 1);
  const int P = a.pairs, D = a.dim;
  if (OP != ROT_TURN)
    for (int i = tid; i < 2 * D; i += kRotThreads)
      wsm[i] = rot_weight(a.w[i >= D], a.w_dtype, i >= D ? i - D : i);

  // this lane's channels and its place in the table (pair < 0: not turned)
  int ca[NI], cb[NI], pr[NI];
#pragma unroll
  for (int k = 0; k < NI; ++k) {
    const int i = lane + k * L;
    if (i >= a.items) {
      ca[k] = cb[k] = pr[k] = -1;
    } else if (ADJ) {
      ca[k] = 2 * VEC * i;
      cb[k] = ca[k] + VEC < D ? ca[k] + VEC : -1;
      pr[k] = VEC * i;
    } else if (i * VEC < P) {
      ca[k] = i * VEC;
      cb[k] = P + i * VEC;
      pr[k] = i * VEC;
    } else {
      const int j = i - P / VEC;
      ca[k] = 2 * P + 2 * VEC * j;
      cb[k] = ca[k] + VEC < D ? ca[k] + VEC : -1;
      pr[k] = -1;
    }
  }
  float dwa[2][NI][2 * VEC];
  if (OP == ROT_NORM_BWD) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < NI; ++k)
#pragma unroll
        for (int e = 0; e < 2 * VEC; ++e) dwa[h][k][e] = 0.f;
  }

  const long long tokens = (long long)a.batch * a.rows;
  for (long long tile = blockIdx.x; tile < a.num_tiles; tile += gridDim.x) {
    const long long t0 = tile * a.tile;
    const int nt = (int)(tokens - t0 < a.tile ? tokens - t0 : a.tile);
    if (tile != blockIdx.x) __syncthreads();  // the table of the tile before is still being read
    for (int i = tid; i < nt * P; i += kRotThreads) {
      const int tk = i / P, p = i - tk * P;
      const long long t = t0 + tk;
      const int b = (int)(t / a.rows), s = (int)(t - (long long)b * a.rows);
      float2 cs = make_float2(1.f, 0.f);
      if (s >= a.prefix) {
        int ax = 0;
        while (p >= a.axis_end[ax]) ++ax;
        const double c = rot_coord(a.coords, a.coord_dtype, b * a.cs[0] + (s - a.prefix) * a.cs[1] + ax * a.cs[2]);
        const double turns = c * (a.freqs[p] * 0.15915494309189533577);  // 1 / (2 pi)
        const float r = (float)(2.0 * (turns - rint(turns)));
        float sn, co;
        sincospif(r, &sn, &co);
        cs = make_float2(co, a.sign * sn);
      }
      table[i] = cs;
    }
    for (int i = tid; i < nt * 2; i += kRotThreads) {
      const int h = i & 1;
      const long long t = t0 + (i >> 1);
      const long long b = t / a.rows, s = t - b * a.rows;
      off[i * 3] = b * a.xs[h][0] + s * a.xs[h][2];
      off[i * 3 + 1] = b * a.ys[h][0] + s * a.ys[h][2];
      off[i * 3 + 2] = b * a.gs[h][0] + s * a.gs[h][2];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int H = a.heads[h];
      if (H == 0) continue;
      const T* __restrict__ xp = (const T*)a.x[h];
      const T* __restrict__ gp = (const T*)a.dy[h];
      T* yp = (T*)a.y[h];
      const int total = nt * H << a.lanes_log2;
      // whole warps stay in the loop together: the shuffles need every lane
      for (int base = 0; base < total; base += kRotThreads) {
        const int row = (base + tid) >> a.lanes_log2;
        const bool live = base + tid < total;
        const int tk = live ? row / H : 0, hd = live ? row - tk * H : 0;
        const long long* o = off + (tk * 2 + h) * 3;
        float u[NI][VEC], v[NI][VEC], gu[NI][VEC], gv[NI][VEC];
#pragma unroll
        for (int k = 0; k < NI; ++k) {
          V xa{}, xb{}, ga{}, gb{};
          const long long xo = o[0] + hd * a.xs[h][1], go = o[2] + hd * a.gs[h][1];
          if (live && ca[k] >= 0) {
            xa = *reinterpret_cast<const V*>(xp + xo + ca[k]);
            if (OP == ROT_NORM_BWD) ga = *reinterpret_cast<const V*>(gp + go + ca[k]);
          }
          if (live && cb[k] >= 0) {
            xb = *reinterpret_cast<const V*>(xp + xo + cb[k]);
            if (OP == ROT_NORM_BWD) gb = *reinterpret_cast<const V*>(gp + go + cb[k]);
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            u[k][e] = rot_f32(xa.v[e]);
            v[k][e] = rot_f32(xb.v[e]);
            if (OP == ROT_NORM_BWD) {
              gu[k][e] = rot_f32(ga.v[e]);
              gv[k][e] = rot_f32(gb.v[e]);
            }
          }
        }
        float rstd = 1.f;
        if (OP != ROT_TURN) {
          float ss = 0.f;
#pragma unroll
          for (int k = 0; k < NI; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) ss += u[k][e] * u[k][e] + v[k][e] * v[k][e];
          for (int m = 1; m < L; m <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
          rstd = rsqrtf(ss * a.inv_dim + a.eps);
        }
        float c1 = 0.f;  // backward: sum of w g x^ over the head
#pragma unroll
        for (int k = 0; k < NI; ++k) {
          if (ca[k] < 0) continue;
          float cs[VEC], sn[VEC];
          bool turn[VEC];  // an unturned channel never meets its neighbour's infinities
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            turn[e] = pr[k] >= 0 && pr[k] + e < P;
            const float2 t = turn[e] ? table[tk * P + pr[k] + e] : make_float2(1.f, 0.f);
            cs[e] = t.x;
            sn[e] = t.y;
          }
          // the two members of pair e: (u[e], v[e]) in the half pairing,
          // neighbours of the 2 VEC contiguous channels in the adjacent one
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const int i0 = ADJ ? 2 * e : e, i1 = ADJ ? 2 * e + 1 : VEC + e;
            float& x0 = i0 < VEC ? u[k][i0 % VEC] : v[k][i0 % VEC];
            float& x1 = i1 < VEC ? u[k][i1 % VEC] : v[k][i1 % VEC];
            const int c0 = i0 < VEC ? ca[k] + i0 : cb[k] + i0 - VEC;
            const int c1i = i1 < VEC ? ca[k] + i1 : cb[k] + i1 - VEC;
            const bool two = cb[k] >= 0;
            if (OP == ROT_TURN) {
              const float p0 = x0, p1 = x1;
              if (turn[e]) {
                x0 = p0 * cs[e] - p1 * sn[e];
                x1 = p1 * cs[e] + p0 * sn[e];
              }
            } else if (OP == ROT_NORM) {
              const float p0 = x0 * rstd * wsm[h * D + c0], p1 = two ? x1 * rstd * wsm[h * D + c1i] : 0.f;
              x0 = turn[e] ? p0 * cs[e] - p1 * sn[e] : p0;
              x1 = turn[e] ? p1 * cs[e] + p0 * sn[e] : p1;
            } else {
              float& g0 = i0 < VEC ? gu[k][i0 % VEC] : gv[k][i0 % VEC];
              float& g1 = i1 < VEC ? gu[k][i1 % VEC] : gv[k][i1 % VEC];
              // turned back: the transpose of the rotation
              const float q0 = turn[e] ? g0 * cs[e] + g1 * sn[e] : g0, q1 = turn[e] ? g1 * cs[e] - g0 * sn[e] : g1;
              x0 *= rstd;
              x1 *= rstd;
              dwa[h][k][i0] += q0 * x0;
              dwa[h][k][i1] += q1 * x1;
              g0 = q0 * wsm[h * D + c0];
              g1 = two ? q1 * wsm[h * D + c1i] : 0.f;
              c1 += g0 * x0 + g1 * x1;
            }
          }
        }
        if (OP == ROT_NORM_BWD) {
          for (int m = 1; m < L; m <<= 1) c1 += __shfl_xor_sync(0xffffffffu, c1, m);
          c1 *= a.inv_dim;
        }
#pragma unroll
        for (int k = 0; k < NI; ++k) {
          V ya, yb;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            if (OP == ROT_NORM_BWD) {
              ya.v[e] = rot_cast<T>(rstd * (gu[k][e] - u[k][e] * c1));
              yb.v[e] = rot_cast<T>(rstd * (gv[k][e] - v[k][e] * c1));
            } else {
              ya.v[e] = rot_cast<T>(u[k][e]);
              yb.v[e] = rot_cast<T>(v[k][e]);
            }
          }
          const long long yo = o[1] + hd * a.ys[h][1];
          if (live && ca[k] >= 0) *reinterpret_cast<V*>(yp + yo + ca[k]) = ya;
          if (live && cb[k] >= 0) *reinterpret_cast<V*>(yp + yo + cb[k]) = yb;
        }
      }
    }
  }

  if (OP == ROT_NORM_BWD) {
    // CTA sum of the weight gradients in a fixed order: threads with the same
    // lane hold the same channels; each adds in turn of its group
    float* red = reinterpret_cast<float*>(rot_smem);  // [groups][dim], over the table
    for (int h = 0; h < 2; ++h) {
      if (a.heads[h] == 0) continue;
      // groups of a warp first (shuffles), then the warps through shared memory
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NI; ++k)
#pragma unroll
        for (int e = 0; e < 2 * VEC; ++e) {
          float s = dwa[h][k][e];
          for (int m = L; m < 32; m <<= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
          const int c = e < VEC ? ca[k] + e : cb[k] + e - VEC;
          const bool have = e < VEC ? ca[k] >= 0 : cb[k] >= 0;
          if (have && (tid & 31) < L) red[(tid >> 5) * D + c] = s;
        }
      __syncthreads();
      for (int c = tid; c < D; c += kRotThreads) {
        float s = 0.f;
        for (int g = 0; g < kRotThreads / 32; ++g) s += red[g * D + c];
        a.dw_part[((long long)blockIdx.x * 2 + h) * D + c] = s;
      }
    }
  }
}

// Weight gradients: the sum of every CTA's part, in 64 bits and in CTA order
// within each of 32 strands, then over the strands.
__global__ __launch_bounds__(1024) void rotary_dw_kernel(const float* __restrict__ part, int grid, int dim, void* dw0,
                                                         void* dw1, int w_dtype, int heads0, int heads1) {
  __shared__ double red[32][33];
  const int h = blockIdx.y, c = blockIdx.x * 32 + threadIdx.x;
  void* dw = h ? dw1 : dw0;
  double s = 0.0;
  if (c < dim && (h ? heads1 : heads0) > 0)
    for (int g = threadIdx.y; g < grid; g += 32) s += (double)part[((long long)g * 2 + h) * dim + c];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < dim && dw) {
    double t = 0.0;
    for (int i = 0; i < 32; ++i) t += red[i][threadIdx.x];
    const float f = (float)t;
    if (w_dtype == SB_F32) ((float*)dw)[c] = f;
    else if (w_dtype == SB_F16) ((__half*)dw)[c] = __float2half_rn(f);
    else ((__nv_bfloat16*)dw)[c] = __float2bfloat16_rn(f);
  }
}

}  // namespace sb
