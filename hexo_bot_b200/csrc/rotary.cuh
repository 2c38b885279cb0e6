// Rotary positions with several axes, alone or behind an RMS norm of every
// query and key head, and the gradients of the latter.
//
//   pair p of axis a(p):  angle = coord[a(p)] * freq[p],
//   (y1, y2) = (x1 cos - x2 sin, x2 cos + x1 sin)          (inverse: -sin)
//   norm:      x^ = x rstd, rstd = (mean(x^2) + eps)^-1/2,  y = R (w x^)
//   backward:  g = R^T dy, dw = sum g x^, dx = rstd (w g - x^ mean(w g x^))
//
// A warp owns a few tokens and all (or a share) of their heads. A lane holds VEC
// pairs of one head (both members of a pair in the same thread), L lanes make a
// head and sum its squares by shuffles, HL heads lie side by side in the warp, so
// that a load covers whole lines of a token's heads. The warp works out the cos
// and sin of its tokens' pairs once, each lane its share, passes them through its
// own piece of shared memory into registers and uses them for every head; the
// rows of the first heads are on their way meanwhile, and no warp waits for
// another. The angle is reduced in pairs of 64-bit numbers, so positions and angles
// up to 2^53 keep fp32 accuracy. Rows are read once and written once, in 16-byte
// accesses where shapes and strides allow. Bound by HBM.
//
// Channels: half pairing (p, P + p), adjacent pairing (2p, 2p + 1), P pairs in
// all; channels from 2P on are not turned. Leading `prefix` rows of each
// sequence have no coordinates and are not turned either.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/shrimp_b200.h"

namespace sb {

constexpr int kRotThreads = 256;
constexpr int kRotMaxDim = 256;
constexpr int kRotMaxAxes = 4;
constexpr int kRotWarps = kRotThreads / 32;
constexpr int kRotAdds = 32;            // weight gradients of so many heads are summed in 32 bits before 64
constexpr int kRotMaxGrid = 148 * 2;    // CTAs of the gradient kernel (one partial weight gradient each)

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
  double* dw_part;             // backward: [grid][2][D]
  const void* coords;
  int coord_dtype, axes;
  long long cs[3];             // batch, row, axis
  const double* freqs;
  int axis_end[kRotMaxAxes];   // exclusive end of each axis' pairs
  int pairs, prefix, batch, rows, dim, items;
  int lanes_log2, side_log2;   // L, HL
  float sign, eps, inv_dim;
  int groups, split;           // token groups of a warp's size, shares of a token's heads
  uint32_t rows_inv, pairs_inv;  // floor(2^32 / rows), floor(2^32 / pairs); 2^32 - 1 for 1
};

template <typename T>
__device__ __forceinline__ float rot_f32(T v) { return static_cast<float>(v); }
template <typename T>
__device__ __forceinline__ T rot_cast(float v) { return static_cast<T>(v); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) RotVec {
  T v[VEC];
};

// VEC values to and from 32 bits, 16-bit types in pairs.
template <typename T, int VEC>
__device__ __forceinline__ void rot_unpack(const RotVec<T, VEC>& x, float (&f)[VEC]) {
  if constexpr (sizeof(T) == 2 && VEC >= 2) {
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      float2 p;
      if constexpr (std::is_same<T, __half>::value) p = __half22float2(__halves2half2(x.v[e], x.v[e + 1]));
      else p = __bfloat1622float2(__halves2bfloat162(x.v[e], x.v[e + 1]));
      f[e] = p.x;
      f[e + 1] = p.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = rot_f32(x.v[e]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ RotVec<T, VEC> rot_pack(const float (&f)[VEC]) {
  RotVec<T, VEC> x;
  if constexpr (sizeof(T) == 2 && VEC >= 2) {
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 p = __floats2half2_rn(f[e], f[e + 1]);
        x.v[e] = p.x;
        x.v[e + 1] = p.y;
      } else {
        const __nv_bfloat162 p = __floats2bfloat162_rn(f[e], f[e + 1]);
        x.v[e] = p.x;
        x.v[e + 1] = p.y;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) x.v[e] = rot_cast<T>(f[e]);
  }
  return x;
}

// x / d and the remainder by m = floor(2^32 / d), for 0 <= x < 2^31: the product
// falls short of the quotient by one at most.
__device__ __forceinline__ int rot_div(int x, int d, uint32_t m, int& rest) {
  int q = (int)__umulhi((uint32_t)x, m);
  rest = x - q * d;
  if (rest >= d) {
    rest -= d;
    ++q;
  }
  return q;
}

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

// 2 / pi as a sum of two 64-bit numbers.
constexpr double kRotTwoPi = 0.6366197723675814, kRotTwoPiRest = -3.935735335036497e-17;

// cos and sin of coord (f.x + f.y) quarter turns (f.y: what f.x's rounding left),
// reduced to the nearest one (at most half a quarter off): the product as a pair of
// 64-bit numbers, whose second part counts as soon as the first one's last bit does;
// past 2^50 quarters it is itself as large as one. Then the Taylor series of both on
// [-pi/4, pi/4] (to x^9 and x^8: off by under 3e-8).
__device__ __forceinline__ float2 rot_cos_sin(double2 f, double coord) {
  const double p = f.x * coord, r = fma(f.x, coord, -p) + f.y * coord;
  const double q0 = rint(p), t = (p - q0) + r, q1 = rint(t), q = q0 + q1;
  const float x = (float)(t - q1) * 1.5707963267948966f, x2 = x * x;
  const float sn = x + x * x2 * (-1.f / 6.f + x2 * (1.f / 120.f + x2 * (-1.f / 5040.f + x2 * (1.f / 362880.f))));
  const float co = 1.f + x2 * (-0.5f + x2 * (1.f / 24.f + x2 * (-1.f / 720.f + x2 * (1.f / 40320.f))));
  const int n = (int)(long long)q;
  const float c = n & 1 ? sn : co, v = n & 1 ? co : sn;
  return make_float2((n + 1) & 2 ? -c : c, n & 2 ? -v : v);
}

// Slots of one lane: NI items of two VEC-wide chunks. Item i of a head:
//   half pairing:  i < P / VEC: chunks at i * VEC and P + i * VEC (turned);
//                  else two chunks of the unturned rest (the second may be missing)
//   adjacent:      channels [2 VEC i, 2 VEC (i + 1)), every pair inside.
// The gradient kernel runs queries and keys in CTAs of their own (blockIdx.y), so
// that a thread adds up one set of weight gradients.
template <typename T, int VEC, int NI, bool ADJ, int OP>
__global__ __launch_bounds__(kRotThreads, OP == ROT_NORM_BWD ? 2 : 3) void rotary_kernel(const RotArgs a) {
  constexpr int U = OP == ROT_NORM_BWD || NI > 1 ? 1 : 2;  // heads whose rows a lane has in flight
  constexpr bool BWD = OP == ROT_NORM_BWD;
  __shared__ __align__(16) float2 tables[kRotWarps][32 * VEC * NI];
  __shared__ double2 freqs[kRotMaxDim / 2];        // quarter turns per coordinate step
  __shared__ unsigned char axis[kRotMaxDim / 2];
  __shared__ float weights[2][OP == ROT_TURN ? 1 : kRotMaxDim];
  using V = RotVec<T, VEC>;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int L = 1 << a.lanes_log2, HL = 1 << a.side_log2, ll = lane & (L - 1);
  const int side = lane >> a.lanes_log2 & (HL - 1), sub = lane >> (a.lanes_log2 + a.side_log2);
  const int TW = 32 >> (a.lanes_log2 + a.side_log2);  // tokens of a unit
  const int P = a.pairs, D = a.dim;
  float2* table = tables[warp];  // [TW][P]

  // this lane's channels and its place in the table (pair < 0: not turned)
  int ca[NI], cb[NI], pr[NI];
#pragma unroll
  for (int k = 0; k < NI; ++k) {
    const int i = ll + k * L;
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
  // weight gradients: a thread's own sum of a few heads, and the warp's, in 64 bits
  // (a channel's by one lane), so that long sums lose no more than short ones
  __shared__ double dw_sum[BWD ? kRotWarps : 1][BWD ? kRotMaxDim : 1];
  float dwa[NI][2 * VEC];
  int adds = 0;
  auto flush = [&] {
    adds = 0;
#pragma unroll
    for (int k = 0; k < NI; ++k)
#pragma unroll
      for (int e = 0; e < 2 * VEC; ++e) {
        float s = dwa[k][e];
        dwa[k][e] = 0.f;
        for (int m = L; m < 32; m <<= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        const int c = e < VEC ? ca[k] + e : cb[k] + e - VEC;
        if ((e < VEC ? ca[k] : cb[k]) >= 0 && lane < L) dw_sum[warp][c] += (double)s;
      }
  };
  if (BWD) {
    for (int c = tid; c < kRotWarps * kRotMaxDim; c += kRotThreads) dw_sum[c / kRotMaxDim][c % kRotMaxDim] = 0.0;
#pragma unroll
    for (int k = 0; k < NI; ++k)
#pragma unroll
      for (int e = 0; e < 2 * VEC; ++e) dwa[k][e] = 0.f;
  }
  for (int p = tid; p < P; p += kRotThreads) {
    int ax = 0;
    while (p >= a.axis_end[ax]) ++ax;
    axis[p] = (unsigned char)ax;
    const double f = a.freqs[p], q = f * kRotTwoPi;
    freqs[p] = make_double2(q, fma(f, kRotTwoPi, -q) + f * kRotTwoPiRest);
  }
  if (OP != ROT_TURN)
    for (int i = tid; i < 2 * D; i += kRotThreads)
      weights[i >= D][i >= D ? i - D : i] = rot_weight(a.w[i >= D], a.w_dtype, i >= D ? i - D : i);
  __syncthreads();
  float w0[NI][2 * VEC];  // this lane's weights
  auto load_weights = [&](int h) {
#pragma unroll
    for (int k = 0; k < NI; ++k)
#pragma unroll
      for (int e = 0; e < 2 * VEC; ++e) {
        const int c = e < VEC ? ca[k] + e : cb[k] + e - VEC;
        w0[k][e] = (e < VEC ? ca[k] : cb[k]) >= 0 ? weights[h][c] : 0.f;
      }
  };
  if (BWD) load_weights(blockIdx.y);
  const int tokens = a.batch * a.rows;  // below 2^31
  const int units = a.groups * a.split, stride = gridDim.x * kRotWarps;
  for (int unit = blockIdx.x * kRotWarps + warp; unit < units; unit += stride) {
    const int group = a.split == 1 ? unit : unit / a.split;
    const int share = unit - group * a.split, t = group * TW + sub;
    int s;
    const int b = rot_div(t, a.rows, a.rows_inv, s);
    float cs[NI][VEC], sn[NI][VEC];
    bool made = false;
    const bool placed = s >= a.prefix;
#pragma unroll
    for (int hh = 0; hh < (BWD ? 1 : 2); ++hh) {
      const int h = BWD ? blockIdx.y : hh;
      const int H = a.heads[h];
      if (H == 0) continue;
      // this share's heads, and the rows of this lane's first one
      const int per = a.split == 1 ? H : ((H + a.split - 1) / a.split + HL - 1) & ~(HL - 1);
      const int end = t < tokens ? min(H, (share + 1) * per) : 0;
      int hd = share * per + side;
      const long long xh = a.xs[h][1] << a.side_log2, yh = a.ys[h][1] << a.side_log2, gh = BWD ? a.gs[h][1] << a.side_log2 : 0;
      const T* x = (const T*)a.x[h] + b * a.xs[h][0] + hd * a.xs[h][1] + s * a.xs[h][2];
      const T* g = BWD ? (const T*)a.dy[h] + b * a.gs[h][0] + hd * a.gs[h][1] + s * a.gs[h][2] : nullptr;
      T* y = (T*)a.y[h] + b * a.ys[h][0] + hd * a.ys[h][1] + s * a.ys[h][2];
      if (OP == ROT_NORM) load_weights(h);
      // whole warps stay in the loop together: the shuffles need every lane
      for (int h0 = share * per; h0 < min(H, (share + 1) * per); h0 += U * HL) {
        V xa[U][NI], xb[U][NI], ga[U][NI], gb[U][NI];
#pragma unroll
        for (int w = 0; w < U; ++w) {
          const bool live = hd + w * HL < end;
#pragma unroll
          for (int k = 0; k < NI; ++k) {
            xa[w][k] = live && ca[k] >= 0 ? *reinterpret_cast<const V*>(x + w * xh + ca[k]) : V{};
            xb[w][k] = live && cb[k] >= 0 ? *reinterpret_cast<const V*>(x + w * xh + cb[k]) : V{};
            if (BWD) {
              ga[w][k] = live && ca[k] >= 0 ? *reinterpret_cast<const V*>(g + w * gh + ca[k]) : V{};
              gb[w][k] = live && cb[k] >= 0 ? *reinterpret_cast<const V*>(g + w * gh + cb[k]) : V{};
            }
          }
        }
        if (!made) {
          made = true;
          __syncwarp();
          for (int i = lane; i < TW * P; i += 32) {
            int p, sr;
            const int ti = rot_div(i, P, a.pairs_inv, p);
            const int tt = t - sub + ti, tb = rot_div(tt, a.rows, a.rows_inv, sr);
            float2 c = make_float2(1.f, 0.f);
            if (tt < tokens && sr >= a.prefix) {
              c = rot_cos_sin(freqs[p], rot_coord(a.coords, a.coord_dtype,
                                                  tb * a.cs[0] + (sr - a.prefix) * a.cs[1] + axis[p] * a.cs[2]));
              c.y *= a.sign;
            }
            table[i] = c;
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < NI; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const float2 c = pr[k] >= 0 && (!ADJ || pr[k] + e < P) ? table[sub * P + pr[k] + e] : make_float2(1.f, 0.f);
              cs[k][e] = c.x;
              sn[k][e] = BWD ? -c.y : c.y;  // gradients turn back
            }
        }
#pragma unroll
        for (int w = 0; w < U; ++w) {
          if (w > 0 && h0 + w * HL >= min(H, (share + 1) * per)) break;  // the whole warp
          const bool live = hd + w * HL < end;
          float u[NI][VEC], v[NI][VEC], gu[NI][VEC], gv[NI][VEC];
#pragma unroll
          for (int k = 0; k < NI; ++k) {
            rot_unpack(xa[w][k], u[k]);
            rot_unpack(xb[w][k], v[k]);
            if (BWD) {
              rot_unpack(ga[w][k], gu[k]);
              rot_unpack(gb[w][k], gv[k]);
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
            // a head that is not there has no norm: with eps = 0 its 0 / 0 would reach the weight gradients
            rstd = live ? rsqrtf(ss * a.inv_dim + a.eps) : 0.f;
#pragma unroll
            for (int k = 0; k < NI; ++k)
#pragma unroll
              for (int e = 0; e < VEC; ++e) {
                u[k][e] *= BWD ? rstd : rstd * w0[k][e];
                v[k][e] *= BWD ? rstd : rstd * w0[k][VEC + e];
              }
          }
#pragma unroll
          for (int k = 0; k < NI; ++k) {
            // unturned channels and rows never meet their neighbours' infinities. Rows
            // without a place have cos 1 and sin 0: the rotation alone drops the other
            // member (2 x 13824 rows, 16 heads of 128: 46 us, 51 with the result selected),
            // behind the norm the result is selected (8 x 2440 rows with gradients: 95 us, 99)
            if (OP == ROT_TURN && pr[k] < 0) continue;
            const bool turn = pr[k] >= 0 && placed;
            float(&m0)[VEC] = BWD ? gu[k] : u[k];
            float(&m1)[VEC] = BWD ? gv[k] : v[k];
            // the two members of pair e: (m0[e], m1[e]) in the half pairing,
            // neighbours of the 2 VEC contiguous channels in the adjacent one
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const int i0 = ADJ ? 2 * e : e, i1 = ADJ ? 2 * e + 1 : VEC + e;
              float& x0 = i0 < VEC ? m0[i0 % VEC] : m1[i0 % VEC];
              float& x1 = i1 < VEC ? m0[i1 % VEC] : m1[i1 % VEC];
              if (OP == ROT_TURN && ADJ && pr[k] + e >= P) continue;
              const float p0 = x0, p1 = x1;
              if (OP == ROT_TURN) {
                x0 = p0 * cs[k][e] - (placed ? p1 : 0.f) * sn[k][e];
                x1 = p1 * cs[k][e] + (placed ? p0 : 0.f) * sn[k][e];
              } else {
                const bool on = turn && !(ADJ && pr[k] + e >= P);
                x0 = on ? p0 * cs[k][e] - p1 * sn[k][e] : p0;
                x1 = on ? p1 * cs[k][e] + p0 * sn[k][e] : p1;
              }
            }
          }
          if (BWD) {
            ++adds;
            float c1 = 0.f;  // sum of w g x^ over the head
#pragma unroll
            for (int k = 0; k < NI; ++k)
#pragma unroll
              for (int e = 0; e < VEC; ++e) {
                dwa[k][e] += gu[k][e] * u[k][e];
                dwa[k][VEC + e] += gv[k][e] * v[k][e];
                gu[k][e] *= w0[k][e];
                gv[k][e] *= w0[k][VEC + e];
                c1 += gu[k][e] * u[k][e] + gv[k][e] * v[k][e];
              }
            for (int m = 1; m < L; m <<= 1) c1 += __shfl_xor_sync(0xffffffffu, c1, m);
            c1 *= a.inv_dim;
#pragma unroll
            for (int k = 0; k < NI; ++k)
#pragma unroll
              for (int e = 0; e < VEC; ++e) {
                u[k][e] = rstd * (gu[k][e] - u[k][e] * c1);
                v[k][e] = rstd * (gv[k][e] - v[k][e] * c1);
              }
          }
#pragma unroll
          for (int k = 0; k < NI; ++k) {
            if (live && ca[k] >= 0) *reinterpret_cast<V*>(y + w * yh + ca[k]) = rot_pack<T, VEC>(u[k]);
            if (live && cb[k] >= 0) *reinterpret_cast<V*>(y + w * yh + cb[k]) = rot_pack<T, VEC>(v[k]);
          }
        }
        hd += U * HL;
        x += U * xh;
        y += U * yh;
        if (BWD) g += U * gh;
      }
    }
    if (BWD && adds >= kRotAdds) flush();
  }

  if (BWD) {
    // CTA sum of the weight gradients, warp after warp
    flush();
    __syncthreads();
    for (int c = tid; c < D; c += kRotThreads) {
      double s = 0.0;
      for (int g = 0; g < kRotWarps; ++g) s += dw_sum[g][c];
      a.dw_part[((long long)blockIdx.x * 2 + blockIdx.y) * D + c] = s;
    }
  }
}

// Weight gradients: the sum of every CTA's part, in 64 bits and in CTA order
// within each of 32 strands, then over the strands.
__global__ __launch_bounds__(1024) void rotary_dw_kernel(const double* __restrict__ part, int grid, int dim, void* dw0,
                                                         void* dw1, int w_dtype, int heads0, int heads1) {
  __shared__ double red[32][33];
  const int h = blockIdx.y, c = blockIdx.x * 32 + threadIdx.x;
  void* dw = h ? dw1 : dw0;
  double s = 0.0;
  if (c < dim && (h ? heads1 : heads0) > 0)
#pragma unroll 8
    for (int g = threadIdx.y; g < grid; g += 32) s += part[((long long)g * 2 + h) * dim + c];
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
