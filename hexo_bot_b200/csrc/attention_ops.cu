// C ABI of the long-support attention operators (declared in
// include/shrimp_b200.h): rotary positions with several axes, the query / key
// norm with the rotation, block means and selection, block-sparse attention
// and their gradients. Argument checks, launch shapes and workspace layout.
#include <cuda_runtime.h>

#include <cmath>

#include "block_attention.cuh"
#include "block_select.cuh"
#include "host.cuh"
#include "rotary.cuh"

namespace sb {
namespace {

int elem_size(int dtype) { return dtype == SB_F32 ? 4 : 2; }
bool float_dtype(int d) { return d == SB_F32 || d == SB_F16 || d == SB_BF16; }
bool half_dtype(int d) { return d == SB_F16 || d == SB_BF16; }
size_t align256(size_t n) { return (n + 255) / 256 * 256; }
int pow2_log2(int n) {
  int l = 0;
  while ((1 << l) < n) ++l;
  return l;
}
HeadsView view(const sb_heads* t) {
  return HeadsView{t->data, t->batch_stride, t->head_stride, t->row_stride};
}
// Largest power of two up to `most` that divides n (0 counts as divisible).
int common_vec(long long n, int most) {
  while (most > 1 && n % most) most >>= 1;
  return most;
}
int heads_vec(const sb_heads* t, int esize, int most) {
  int v = common_vec(t->batch_stride, most);
  v = common_vec(t->head_stride, v);
  v = common_vec(t->row_stride, v);
  while (v > 1 && (uintptr_t)t->data % (v * esize)) v >>= 1;
  return v;
}
int check_heads(const char* what, const char* name, const sb_heads* t, int esize) {
  if (!t || !t->data) return fail(SB_ERR_INVALID_ARG, "%s: %s is NULL", what, name);
  if ((uintptr_t)t->data % esize) return fail(SB_ERR_INVALID_ARG, "%s: %s is not aligned to its element", what, name);
  return SB_OK;
}
// 16-bit operands that are read in 16-byte pieces.
int check_heads16(const char* what, const char* name, const sb_heads* t) {
  if (int s = check_heads(what, name, t, 2)) return s;
  if (heads_vec(t, 2, 8) != 8)
    return fail(SB_ERR_INVALID_ARG, "%s: %s needs a 16-byte aligned base and strides that are multiples of 8", what, name);
  return SB_OK;
}

// ---- rotary -------------------------------------------------------------------
int fill_rotary(const char* what, const sb_rotary* r, int rows, RotArgs* a) {
  if (!r) return SB_OK;
  if (r->axes < 1 || r->axes > kRotMaxAxes) return fail(SB_ERR_INVALID_ARG, "%s: %d axes (1 to %d)", what, r->axes, kRotMaxAxes);
  int pairs = 0;
  for (int i = 0; i < r->axes; ++i) {
    if (r->sections[i] < 1 || r->sections[i] > kRotMaxDim)
      return fail(SB_ERR_INVALID_ARG, "%s: axis %d has %d pairs", what, i, r->sections[i]);
    pairs += r->sections[i];
    a->axis_end[i] = pairs;
  }
  if (2 * pairs > a->dim) return fail(SB_ERR_INVALID_ARG, "%s: %d pairs do not fit head_dim %d", what, pairs, a->dim);
  if (r->prefix < 0 || r->prefix > rows) return fail(SB_ERR_INVALID_ARG, "%s: prefix %d of %d rows", what, r->prefix, rows);
  if (!r->freqs || (uintptr_t)r->freqs % 8) return fail(SB_ERR_INVALID_ARG, "%s: freqs is NULL or misaligned", what);
  if (r->coords_dtype != SB_I64 && r->coords_dtype != SB_I32 && r->coords_dtype != SB_I16 && r->coords_dtype != SB_F32)
    return fail(SB_ERR_UNSUPPORTED, "%s: coords dtype %d", what, r->coords_dtype);
  const int csize = r->coords_dtype == SB_I64 ? 8 : r->coords_dtype == SB_I16 ? 2 : 4;
  if (r->prefix < rows && (!r->coords || (uintptr_t)r->coords % csize))
    return fail(SB_ERR_INVALID_ARG, "%s: coords is NULL or misaligned", what);
  a->pairs = pairs;
  a->prefix = r->prefix;
  a->axes = r->axes;
  a->coords = r->coords;
  a->coord_dtype = r->coords_dtype;
  a->cs[0] = r->batch_stride;
  a->cs[1] = r->row_stride;
  a->cs[2] = r->axis_stride;
  a->freqs = r->freqs;
  return SB_OK;
}

template <typename T, int VEC, int NI, bool ADJ, int OP>
int launch_rotary_as(const RotArgs& a, int grid, cudaStream_t st) {
  // gradients: queries and keys in CTAs of their own
  const dim3 ctas((unsigned)grid, OP == ROT_NORM_BWD && a.heads[1] > 0 ? 2 : 1);
  rotary_kernel<T, VEC, NI, ADJ, OP><<<ctas, kRotThreads, 0, st>>>(a);
  return check_launch("rotary_kernel");
}
template <typename T, bool ADJ, int OP>
int launch_rotary_vec(const RotArgs& a, int vec, int grid, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return launch_rotary_as<T, 8, 1, ADJ, OP>(a, grid, st);
  if (vec == 4) return launch_rotary_as<T, 4, 1, ADJ, OP>(a, grid, st);
  if (vec == 2) return launch_rotary_as<T, 2, 2, ADJ, OP>(a, grid, st);
  return launch_rotary_as<T, 1, 4, ADJ, OP>(a, grid, st);
}
template <int OP>
int launch_rotary_op(const RotArgs& a, int dtype, bool adjacent, int vec, int grid, cudaStream_t st) {
  if (dtype == SB_F32)
    return adjacent ? launch_rotary_vec<float, true, OP>(a, vec, grid, st) : launch_rotary_vec<float, false, OP>(a, vec, grid, st);
  if (dtype == SB_F16)
    return adjacent ? launch_rotary_vec<__half, true, OP>(a, vec, grid, st)
                    : launch_rotary_vec<__half, false, OP>(a, vec, grid, st);
  return adjacent ? launch_rotary_vec<__nv_bfloat16, true, OP>(a, vec, grid, st)
                  : launch_rotary_vec<__nv_bfloat16, false, OP>(a, vec, grid, st);
}

// Vector width, lanes and grid of a call whose operands are filled in.
// `vec` comes in as the widest that bases and strides allow.
int launch_rotary(RotArgs& a, int op, int dtype, bool adjacent, int vec, cudaStream_t st, int* grid_out) {
  const int D = a.dim, P = a.pairs;
  while (vec > 1 && (adjacent ? D % (2 * vec) : (D % vec || P % vec))) vec >>= 1;
  a.items = adjacent ? (D + 2 * vec - 1) / (2 * vec) : P / vec + ((D - 2 * P) / vec + 1) / 2;
  a.lanes_log2 = pow2_log2(a.items < 32 ? a.items : 32);
  a.inv_dim = 1.f / (float)D;
  // heads side by side: no more than share the work of the angles, and half of
  // them at most, so that a lane's angles serve two heads or more (4096 x 69 rows,
  // 8 heads of 16: 49 us with all side by side, 37 with half, 37 with a quarter,
  // 54 with an eighth, where loads touch too many lines)
  const int least = a.heads[1] > 0 && a.heads[1] < a.heads[0] ? a.heads[1] : a.heads[0];
  int side = 0;
  while (side + a.lanes_log2 < 5 && (2 << side) <= vec && 2 * (2 << side) <= a.heads[0] && (2 << side) <= least) ++side;
  a.side_log2 = side;
  const long long tokens = (long long)a.batch * a.rows;
  a.groups = (int)cdiv(tokens, 32 >> (a.lanes_log2 + side));
  // few tokens: their heads split over warps until every SM has some (never for
  // the gradients, whose warps go over many units)
  a.split = 1;
  while (op != ROT_NORM_BWD && (long long)a.groups * a.split < 8 * num_sms() && (2 << side) * a.split <= a.heads[0]) a.split *= 2;
  a.rows_inv = a.rows > 1 ? (uint32_t)(0x100000000ull / a.rows) : 0xffffffffu;
  a.pairs_inv = P > 1 ? (uint32_t)(0x100000000ull / P) : 0xffffffffu;
  int grid = (int)cdiv((long long)a.groups * a.split, kRotWarps);
  const int most = op == ROT_NORM_BWD ? kRotMaxGrid : 3 * num_sms();  // the CTAs that run at once
  if (grid > most) grid = most;
  if (grid_out) *grid_out = grid;
  if (op == ROT_TURN) return launch_rotary_op<ROT_TURN>(a, dtype, adjacent, vec, grid, st);
  if (op == ROT_NORM) return launch_rotary_op<ROT_NORM>(a, dtype, adjacent, vec, grid, st);
  return launch_rotary_op<ROT_NORM_BWD>(a, dtype, adjacent, vec, grid, st);
}

int check_rotary_shape(const char* what, int dtype, int batch, int heads, int rows, int dim) {
  if (!float_dtype(dtype)) return fail(SB_ERR_UNSUPPORTED, "%s: dtype %d (f32, f16, bf16)", what, dtype);
  if (batch < 0 || rows < 0 || heads < 1 || heads > 65535) return fail(SB_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (dim < 1 || dim > kRotMaxDim) return fail(SB_ERR_UNSUPPORTED, "%s: head_dim %d (1 to %d)", what, dim, kRotMaxDim);
  // row numbers, rounded up to a warp's or a launch's next, stay below 2^31
  if ((long long)batch * rows > 0x7fff0000ll) return fail(SB_ERR_UNSUPPORTED, "%s: more than 2^31 - 2^16 rows", what);
  return SB_OK;
}

void put(RotArgs* a, int slot, const sb_heads* x, const sb_heads* dy, const sb_heads* y) {
  a->x[slot] = x->data;
  a->y[slot] = y->data;
  a->xs[slot][0] = x->batch_stride;
  a->xs[slot][1] = x->head_stride;
  a->xs[slot][2] = x->row_stride;
  a->ys[slot][0] = y->batch_stride;
  a->ys[slot][1] = y->head_stride;
  a->ys[slot][2] = y->row_stride;
  if (dy) {
    a->dy[slot] = dy->data;
    a->gs[slot][0] = dy->batch_stride;
    a->gs[slot][1] = dy->head_stride;
    a->gs[slot][2] = dy->row_stride;
  }
}

// ---- block selection ----------------------------------------------------------
// Up to so many queries of a sequence take the few-query kernel (few / many, us,
// 8 heads of 64 over 128 blocks: 6 / 13 at 2 rows, 7 / 14 at 8, 11 / 14 at 16,
// 14 / 23 at 32; 8 x 8 heads of 128: 14 / 26, 17 / 34, 32 / 35, 47 / 37).
constexpr int kSelFewRows = 16;

template <typename T, int PER, int LPR>
int launch_select_per(const SelArgs& a, unsigned grid, cudaStream_t st) {
  const int smem = sel_smem_bytes(a.tile, a.nb, a.dim);
  if (int s = ensure_smem(reinterpret_cast<const void*>(block_select_kernel<T, PER, LPR>), smem)) return s;
  block_select_kernel<T, PER, LPR><<<grid, kSelThreads, smem, st>>>(a);
  return check_launch("block_select_kernel");
}
// The form with the fewest scores and lanes a row that holds the blocks (2 lanes of
// 20 / 2 of 32 / 4 of 32 / a warp a row, us, 16 x 2440 rows, 8 heads of 16: 110 / 151 /
// 237 / 383 at 39 blocks, - / 157 / 243 / 385 at 64, - / - / 302 / 577 at 128; 8192 rows,
// 4 heads of 128: 44 / 50 / 54 / 79, - / 57 / 62 / 86, - / - / 78 / 125).
template <typename T>
int launch_select(const SelArgs& a, unsigned grid, cudaStream_t st) {
  if (a.nb <= 40) return launch_select_per<T, 20, 2>(a, grid, st);
  if (a.nb <= 64) return launch_select_per<T, 32, 2>(a, grid, st);
  if (a.nb <= 128) return launch_select_per<T, 32, 4>(a, grid, st);
  return launch_select_per<T, 0, 8>(a, grid, st);
}
template <typename T, int PER>
int launch_select_few_per(const SelArgs& a, unsigned rows, int cluster, cudaStream_t st) {
  const int smem = sel_few_smem_bytes(a.nb);
  if (int s = ensure_smem(reinterpret_cast<const void*>(block_select_few_kernel<T, PER>), smem)) return s;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = rows * cluster;
  cfg.blockDim = kSelThreads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, block_select_few_kernel<T, PER>, a);  // errors surface in check_launch
  return check_launch("block_select_few_kernel");
}
template <typename T>
int launch_select_few(const SelArgs& a, unsigned rows, int cluster, cudaStream_t st) {
  if (a.nb <= 2 * kSelThreads) return launch_select_few_per<T, 2>(a, rows, cluster, st);
  if (a.nb <= 8 * kSelThreads) return launch_select_few_per<T, 8>(a, rows, cluster, st);
  return launch_select_few_per<T, 0>(a, rows, cluster, st);
}

// ---- block-sparse attention ------------------------------------------------------
// Bytes of parts that a window of rows may hold. Windows that fit the 126 MB L2
// keep the parts off HBM but leave the SMs short of work at every launch's end:
// 8192 rows, 8 heads of 64, 16 of 128 blocks, forward / backward: 402 / 598 us with
// windows of 64 MB, 276 / 557 with 100, 254 / 510 with 200, 210 / 412 with one; 16 x
// 2440 rows, 8 heads of 16: 278 / 577, 258 / 537, 228 / 494 with 200 MB or more.
constexpr long long kBaWindowBytes = 1ll << 30;
// Up to so many queries take the few-query kernel (few / many, us, 8 heads of 64, 16
// of 128 blocks: 8 / 21 at 2 rows, 11 / 22 at 16, 21 / 22 at 32, 40 / 22 at 64; 8 x 8
// groups of 4 heads of 128, 32 of 512: 30 / 302, 205 / 435, 408 / 488, 812 / 544).
constexpr int kBaFewRows = 16;
// Work items an SM and window, and the listed rows that an item may hold: fewer
// items leave SMs idle behind popular blocks (8192 rows, 8 heads of 64, 16 of 128
// blocks, forward: 212 us with 8 an SM, 200 with 16 to 32; backward, where every
// segment of a block leaves a part of dk and dv: 431 / 429 / 397 / 402 / 403 us
// with 4 / 6 / 8 / 12 / 16), smaller ones repeat the listing and the key loads.
constexpr int kBaItems = 16, kBaBwdItems = 8, kBaMinTarget = 256, kBaMaxTarget = 1024;

struct BaPlan {
  int marks, bh_step, wq, seg, sums;
  size_t ticket, entries, spans, slots, part, ml, delta, kv_part, total;
};

BaPlan ba_plan(long long bh, int q_rows, int group, int dim, int nb, int block, int topk, bool backward) {
  BaPlan p{};
  const long long row_bytes = (long long)group * topk * (dim * 4 + (backward ? 0 : 8));
  const long long per_bh = row_bytes * q_rows;
  if (per_bh <= kBaWindowBytes) {
    const long long n = per_bh ? kBaWindowBytes / per_bh : bh;
    p.bh_step = (int)(n < bh ? n : bh);
    p.wq = q_rows;
  } else {
    p.bh_step = 1;
    const long long w = kBaWindowBytes / row_bytes / kBaMark * kBaMark;
    p.wq = (int)(w < kBaMark ? kBaMark : w);
  }
  // a segment: as many groups as give a work item its target of listed rows on
  // average (several items a CTA, to even out popular blocks), evenly split
  const long long pairs = (long long)p.bh_step * p.wq * topk * group;
  long long target = pairs / ((backward ? kBaBwdItems : kBaItems) * num_sms());
  const int most = backward ? 2 * kBaMaxTarget : kBaMaxTarget;
  target = target < kBaMinTarget ? kBaMinTarget : target > most ? most : target;
  const long long groups = cdiv(p.wq, kBaMark);
  p.marks = (int)groups;
  long long seg = cdiv(target * nb, (long long)topk * group * kBaMark);
  seg = seg < 1 ? 1 : seg > groups ? groups : seg;
  p.seg = (int)cdiv(groups, cdiv(groups, seg));
  // backward: sums of dk and dv that a block has, one a segment of its window; the
  // windows of a head add to the same ones, and all heads of a step share them
  const int nseg = (int)cdiv(groups, p.seg);
  p.sums = backward && (nseg > 1 || p.wq < q_rows) ? nseg : 0;
  const long long rows = (long long)p.bh_step * p.wq * group;
  size_t at = 0;
  p.ticket = at;
  at += 256;
  p.entries = at;
  at += align256((size_t)p.bh_step * p.marks * kBaMark * topk * 2);
  p.spans = at;
  at += align256((size_t)p.bh_step * nb * p.marks * 4);
  p.slots = at;
  at += align256((size_t)bh * q_rows * 8);
  p.part = at;
  at += align256((size_t)rows * topk * dim * 4);
  p.ml = at;
  if (!backward) at += align256((size_t)rows * topk * 8);
  p.delta = at;
  if (backward) at += align256((size_t)bh * q_rows * group * 8);
  p.kv_part = at;
  at += align256((size_t)p.bh_step * nb * p.sums * 2 * block * dim * 4);
  p.total = at;
  return p;
}

int check_ba(const char* what, int dtype, int batch, int q_heads, int kv_heads, int q_rows, int kv_rows, int dim, int block,
             int topk) {
  if (!half_dtype(dtype)) return fail(SB_ERR_UNSUPPORTED, "%s: dtype %d (f16, bf16)", what, dtype);
  if (batch < 0 || q_rows < 0 || kv_rows < 0 || q_heads < 1 || kv_heads < 1)
    return fail(SB_ERR_INVALID_ARG, "%s: bad sizes", what);
  if (q_heads % kv_heads) return fail(SB_ERR_INVALID_ARG, "%s: %d query heads over %d key heads", what, q_heads, kv_heads);
  if (kv_rows > 0x7fff0000) return fail(SB_ERR_UNSUPPORTED, "%s: %d key rows (at most 2^31 - 2^16)", what, kv_rows);
  if (q_rows > 1 << 26) return fail(SB_ERR_UNSUPPORTED, "%s: %d rows (at most 2^26)", what, q_rows);
  if (q_heads > 65535 || q_heads / kv_heads > 1024 || (long long)batch * kv_heads > 0x7fffffffll)
    return fail(SB_ERR_UNSUPPORTED, "%s: too many heads", what);
  if (dim < 8 || dim > kBaMaxDim || dim % 8)
    return fail(SB_ERR_UNSUPPORTED, "%s: head_dim %d (a multiple of 8 up to %d)", what, dim, kBaMaxDim);
  if (block != 32 && block != 64 && block != 128) return fail(SB_ERR_UNSUPPORTED, "%s: block %d (32, 64, 128)", what, block);
  if (topk < 1 || topk > kBaMaxTopk) return fail(SB_ERR_UNSUPPORTED, "%s: topk %d (1 to %d)", what, topk, kBaMaxTopk);
  return SB_OK;
}

// Calls f.template operator()<T, DP, BK>() for the call's type and sizes.
template <typename F>
int ba_dispatch(int dtype, int dim, int block, F f) {
  auto by_block = [&](auto t, auto dp) {
    using T = typename decltype(t)::type;
    constexpr int DP = decltype(dp)::value;
    if (block == 32) return f.template operator()<T, DP, 32>();
    if (block == 64) return f.template operator()<T, DP, 64>();
    return f.template operator()<T, DP, 128>();
  };
  auto by_dim = [&](auto t) {
    if (dim <= 16) return by_block(t, std::integral_constant<int, 16>{});
    if (dim <= 32) return by_block(t, std::integral_constant<int, 32>{});
    if (dim <= 64) return by_block(t, std::integral_constant<int, 64>{});
    return by_block(t, std::integral_constant<int, 128>{});
  };
  struct H { using type = __half; };
  struct B { using type = __nv_bfloat16; };
  return dtype == SB_F16 ? by_dim(H{}) : by_dim(B{});
}

template <typename K>
int launch_ba(K kern, const char* name, long long grid, int threads, int smem, const BaArgs& a, cudaStream_t st) {
  if (grid > 0x7fffffffll) return fail(SB_ERR_UNSUPPORTED, "%s: too many blocks for one launch", name);
  if (grid == 0) return SB_OK;
  if (int s = ensure_smem(reinterpret_cast<const void*>(kern), smem)) return s;
  kern<<<(unsigned)grid, threads, smem, st>>>(a);
  return check_launch(name);
}

int launch_list(const BaArgs& a, cudaStream_t st) {
  const long long grid = a.nbh * cdiv(a.wq, kBaMark);
  const int smem = ba_list_smem(a.nb, a.topk);
  if (a.topk <= 8) return launch_ba(block_list_kernel<8>, "block_list_kernel", grid, kBaMark, smem, a, st);
  if (a.topk <= 16) return launch_ba(block_list_kernel<16>, "block_list_kernel", grid, kBaMark, smem, a, st);
  return launch_ba(block_list_kernel<kBaMaxTopk>, "block_list_kernel", grid, kBaMark, smem, a, st);
}
struct LaunchFew {
  const BaArgs& a;
  cudaStream_t st;
  template <typename T, int DP, int BK>
  int operator()() const {
    constexpr int W = ba_few_warps<DP, BK>();
    const long long rows = (long long)a.batch * a.kv_heads * a.q_rows * ((a.group + 15) / 16);
    // CTAs of a row: as many as have a block for every warp and run at once (64
    // rows of 32 blocks, D = 128: 30 us with one CTA a row, 19 with two, 23 with
    // four, 39 with eight, which take turns)
    int cluster = 1;
    while (cluster < kBaFewCluster && cluster * W < a.topk && 2 * rows * cluster <= num_sms()) cluster *= 2;
    if (rows * cluster > 0x7fffffffll) return fail(SB_ERR_UNSUPPORTED, "block_attention: too many rows for one launch");
    auto kern = block_attn_few_kernel<T, DP, BK>;
    if (int s = ensure_smem(reinterpret_cast<const void*>(kern), ba_few_smem<DP, BK>())) return s;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = (unsigned)(rows * cluster);
    cfg.blockDim = W * 32;
    cfg.dynamicSmemBytes = ba_few_smem<DP, BK>();
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kern, a);  // errors surface in check_launch
    return check_launch("block_attn_few_kernel");
  }
};
struct LaunchFwd {
  const BaArgs& a;
  cudaStream_t st;
  template <typename T, int DP, int BK>
  int operator()() const {
    const long long items = (long long)a.nbh * a.nb * a.nseg, most = (long long)num_sms() * ba_fwd_ctas<DP, BK>();
    if (items > 0x7fffffffll) return fail(SB_ERR_UNSUPPORTED, "block_attention: too many blocks for one launch");
    if (int s = launch_ba(block_attn_kernel<T, DP, BK>, "block_attn_kernel", items < most ? items : most, kBaFwdThreads,
                          ba_fwd_smem<DP, BK>(), a, st))
      return s;
    return launch_ba(block_attn_join_kernel<T>, "block_attn_join_kernel",
                     cdiv((long long)a.nbh * a.wq * a.group, kBaJoinThreads >> ba_join_lanes(a.dim, a.topk)),
                     kBaJoinThreads, 0, a, st);
  }
};
struct LaunchBwd {
  const BaArgs& a;
  cudaStream_t st;
  template <typename T, int DP, int BK>
  int operator()() const {
    const long long items = (long long)a.nbh * a.nb * a.nseg, most = (long long)num_sms() * ba_bwd_ctas<DP, BK>();
    if (items > 0x7fffffffll) return fail(SB_ERR_UNSUPPORTED, "block_attention_backward: too many blocks for one launch");
    if (int s = launch_ba(block_attn_bwd_kernel<T, DP, BK>, "block_attn_bwd_kernel", items < most ? items : most,
                          kBaBwdThreads, ba_bwd_smem<DP, BK>(), a, st))
      return s;
    return launch_ba(block_attn_dq_kernel<T>, "block_attn_dq_kernel",
                     cdiv((long long)a.nbh * a.wq * a.group, kBaJoinThreads >> ba_join_lanes(a.dim, a.topk)),
                     kBaJoinThreads, 0, a, st);
  }
};

uint32_t magic(int d) { return d <= 1 ? 0u : (uint32_t)((0x100000000ull + d - 1) / d); }

void ba_fill(BaArgs* a, const int32_t* index, const int32_t* kv_lens, const int32_t* q_lens, int batch, int q_heads,
             int kv_heads, int q_rows, int kv_rows, int dim, int block, int topk, float scale) {
  a->idx = index;
  a->kv_lens = kv_lens;
  a->q_lens = q_lens;
  a->batch = batch;
  a->kv_heads = kv_heads;
  a->group = q_heads / kv_heads;
  a->q_rows = q_rows;
  a->kv_rows = kv_rows;
  a->dim = dim;
  a->block = block;
  a->nb = (int)cdiv(kv_rows, block);
  a->topk = topk;
  a->scale = scale;
  a->scale_log2 = scale * kLog2e;
  a->group_magic = magic(a->group);
}

// Lists every window of the plan and runs f() for it, and done() behind the last one of each step of heads.
template <typename F, typename G>
int ba_windows(BaArgs& a, const BaPlan& p, cudaStream_t st, F f, G done) {
  const int bh = a.batch * a.kv_heads;
  for (a.bh0 = 0; a.bh0 < bh; a.bh0 += p.bh_step) {
    a.nbh = bh - a.bh0 < p.bh_step ? bh - a.bh0 : p.bh_step;
    for (a.w0 = 0; a.w0 < a.q_rows; a.w0 += p.wq) {
      a.wq = a.q_rows - a.w0 < p.wq ? a.q_rows - a.w0 : p.wq;
      a.seg = p.seg;
      a.nseg = (int)cdiv(cdiv(a.wq, kBaMark), p.seg);
      if (int s = launch_list(a, st)) return s;
      if (int s = f()) return s;
    }
    if (int s = done()) return s;
  }
  return SB_OK;
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" {

int sb_axes_rotary(const sb_heads* x, int dtype, const sb_rotary* rotary, int inverse, int batch, int heads, int rows,
                   int head_dim, const sb_heads* out, void* stream) {
  const char* what = "axes_rotary";
  if (int s = check_rotary_shape(what, dtype, batch, heads, rows, head_dim)) return s;
  if (!rotary) return fail(SB_ERR_INVALID_ARG, "%s: rotary is NULL", what);
  RotArgs a{};
  a.dim = head_dim;
  if (int s = fill_rotary(what, rotary, rows, &a)) return s;
  if (batch == 0 || rows == 0) return SB_OK;
  const int e = elem_size(dtype);
  if (int s = check_heads(what, "x", x, e)) return s;
  if (int s = check_heads(what, "out", out, e)) return s;
  put(&a, 0, x, nullptr, out);
  a.heads[0] = heads;
  a.batch = batch;
  a.rows = rows;
  a.sign = inverse ? -1.f : 1.f;
  const int vec = heads_vec(out, e, heads_vec(x, e, 16 / e));
  return launch_rotary(a, ROT_TURN, dtype, rotary->adjacent != 0, vec, (cudaStream_t)stream, nullptr);
}

static int qk_norm(const char* what, const sb_heads* q, const sb_heads* k, const sb_heads* dq_out, const sb_heads* dk_out,
                   int dtype, const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                   const sb_rotary* rotary, int batch, int q_heads, int k_heads, int rows, int head_dim, const sb_heads* y0,
                   const sb_heads* y1, void* dqw, void* dkw, void* workspace, size_t workspace_bytes, bool backward,
                   cudaStream_t st) {
  if (int s = check_rotary_shape(what, dtype, batch, q_heads, rows, head_dim)) return s;
  if (k_heads < 0 || k_heads > 65535) return fail(SB_ERR_INVALID_ARG, "%s: %d key heads", what, k_heads);
  if (!float_dtype(weight_dtype)) return fail(SB_ERR_UNSUPPORTED, "%s: weight dtype %d", what, weight_dtype);
  if (!(eps >= 0.f)) return fail(SB_ERR_INVALID_ARG, "%s: eps %g", what, (double)eps);
  const int we = elem_size(weight_dtype);
  if ((uintptr_t)q_weight % we || (uintptr_t)k_weight % we || (uintptr_t)dqw % we || (uintptr_t)dkw % we)
    return fail(SB_ERR_INVALID_ARG, "%s: a weight is not aligned to its element", what);
  RotArgs a{};
  a.dim = head_dim;
  if (int s = fill_rotary(what, rotary, rows, &a)) return s;
  const int e = elem_size(dtype);
  const bool work = batch > 0 && rows > 0;
  int vec = 16 / e;
  const sb_heads* xs[2] = {q, k};
  const sb_heads* gs[2] = {dq_out, dk_out};
  const sb_heads* ys[2] = {y0, y1};
  const char* xn[2] = {"q", "k"};
  const char* gn[2] = {"dq_out", "dk_out"};
  const char* yn[2] = {backward ? "dq" : "q_out", backward ? "dk" : "k_out"};
  a.heads[0] = q_heads;
  a.heads[1] = k_heads;
  for (int h = 0; h < 2 && work; ++h) {
    if (a.heads[h] == 0) continue;
    if (int s = check_heads(what, xn[h], xs[h], e)) return s;
    if (int s = check_heads(what, yn[h], ys[h], e)) return s;
    vec = heads_vec(ys[h], e, heads_vec(xs[h], e, vec));
    if (backward) {
      if (int s = check_heads(what, gn[h], gs[h], e)) return s;
      vec = heads_vec(gs[h], e, vec);
    }
    put(&a, h, xs[h], backward ? gs[h] : nullptr, ys[h]);
  }
  a.w[0] = q_weight;
  a.w[1] = k_weight;
  a.w_dtype = weight_dtype;
  a.batch = batch;
  a.rows = rows;
  a.sign = 1.f;
  a.eps = eps;
  const bool adjacent = rotary && rotary->adjacent != 0;
  int grid = 0;
  if (backward) {
    const size_t need = (size_t)kRotMaxGrid * 2 * head_dim * 8;
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need)
      return fail(SB_ERR_WORKSPACE, "%s: workspace of %zu bytes, 16-byte aligned, needed", what, need);
    a.dw_part = (double*)workspace;
    if (work)
      if (int s = launch_rotary(a, ROT_NORM_BWD, dtype, adjacent, vec, st, &grid)) return s;
    if (!dqw && !dkw) return SB_OK;
    // no rows: grid is 0 and the gradients are written as zeros
    rotary_dw_kernel<<<dim3((unsigned)cdiv(head_dim, 32), 2), dim3(32, 32), 0, st>>>(a.dw_part, grid, head_dim, dqw, dkw,
                                                                                   weight_dtype, q_heads, k_heads);
    return check_launch("rotary_dw_kernel");
  }
  if (!work) return SB_OK;
  return launch_rotary(a, ROT_NORM, dtype, adjacent, vec, st, nullptr);
}

int sb_qk_norm_rotary(const sb_heads* q, const sb_heads* k, int dtype, const void* q_weight, const void* k_weight,
                      int weight_dtype, float eps, const sb_rotary* rotary, int batch, int q_heads, int k_heads, int rows,
                      int head_dim, const sb_heads* q_out, const sb_heads* k_out, void* stream) {
  return qk_norm("qk_norm_rotary", q, k, nullptr, nullptr, dtype, q_weight, k_weight, weight_dtype, eps, rotary, batch,
                 q_heads, k_heads, rows, head_dim, q_out, k_out, nullptr, nullptr, nullptr, 0, false, (cudaStream_t)stream);
}

int sb_qk_norm_rotary_backward_workspace_bytes(int head_dim, size_t* bytes) {
  if (!bytes || head_dim < 1 || head_dim > kRotMaxDim) return fail(SB_ERR_INVALID_ARG, "qk_norm_rotary_backward: bad args");
  *bytes = (size_t)kRotMaxGrid * 2 * head_dim * 8;
  return SB_OK;
}

int sb_qk_norm_rotary_backward(const sb_heads* dq_out, const sb_heads* dk_out, const sb_heads* q, const sb_heads* k, int dtype,
                               const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                               const sb_rotary* rotary, int batch, int q_heads, int k_heads, int rows, int head_dim,
                               const sb_heads* dq, const sb_heads* dk, void* dq_weight, void* dk_weight, void* workspace,
                               size_t workspace_bytes, void* stream) {
  return qk_norm("qk_norm_rotary_backward", q, k, dq_out, dk_out, dtype, q_weight, k_weight, weight_dtype, eps, rotary, batch,
                 q_heads, k_heads, rows, head_dim, dq, dk, dq_weight, dk_weight, workspace, workspace_bytes, true,
                 (cudaStream_t)stream);
}

int sb_block_means(const sb_heads* k, int dtype, const int32_t* kv_lens, int batch, int kv_heads, int kv_rows, int head_dim,
                   int block, float* means, void* stream) {
  const char* what = "block_means";
  if (!float_dtype(dtype)) return fail(SB_ERR_UNSUPPORTED, "%s: dtype %d (f32, f16, bf16)", what, dtype);
  if (batch < 0 || kv_heads < 1 || kv_rows < 0 || block < 1) return fail(SB_ERR_INVALID_ARG, "%s: bad sizes", what);
  if ((long long)kv_rows + block > 0x7fffffffll) return fail(SB_ERR_UNSUPPORTED, "%s: rows and block exceed 2^31", what);
  if (head_dim < 1 || head_dim > kSelMaxDim)
    return fail(SB_ERR_UNSUPPORTED, "%s: head_dim %d (1 to %d)", what, head_dim, kSelMaxDim);
  if (batch == 0 || kv_rows == 0) return SB_OK;
  const int e = elem_size(dtype);
  if (int s = check_heads(what, "k", k, e)) return s;
  if (!means || (uintptr_t)means % 4 || (uintptr_t)kv_lens % 4)
    return fail(SB_ERR_INVALID_ARG, "%s: means is NULL or an operand is misaligned", what);
  const int nb = (int)cdiv(kv_rows, block);
  const long long grid = (long long)batch * kv_heads * nb;
  if (grid > 0x7fffffffll) return fail(SB_ERR_UNSUPPORTED, "%s: too many blocks for one launch", what);
  const bool wide = heads_vec(k, e, 16 / e) == 16 / e && head_dim % (16 / e) == 0;
  cudaStream_t st = (cudaStream_t)stream;
  const HeadsView kv = view(k);
  // a warp a block, or a CTA of four where that leaves SMs without work
  const bool split = grid < 8ll * num_sms();
  const int vec = wide ? 16 / e : 1;
  const int chunk_lanes = 1 << pow2_log2(head_dim / vec < 32 ? head_dim / vec : 32);
  const unsigned ctas = (unsigned)(split ? grid : cdiv(grid, kMeansThreads / 32));
#define SB_MEANS_AS(T, V, W)                                                                                      \
  block_means_kernel<T, V, W><<<ctas, kMeansThreads, 0, st>>>(kv, kv_lens, kv_heads, kv_rows, head_dim, block, nb, grid, \
                                                              chunk_lanes, means)
#define SB_MEANS(T, V) \
  if (split) SB_MEANS_AS(T, V, 4); else SB_MEANS_AS(T, V, 1)
  if (dtype == SB_F32) {
    if (wide) { SB_MEANS(float, 4); } else { SB_MEANS(float, 1); }
  } else if (dtype == SB_F16) {
    if (wide) { SB_MEANS(__half, 8); } else { SB_MEANS(__half, 1); }
  } else {
    if (wide) { SB_MEANS(__nv_bfloat16, 8); } else { SB_MEANS(__nv_bfloat16, 1); }
  }
#undef SB_MEANS_AS
#undef SB_MEANS
  return check_launch("block_means_kernel");
}

int sb_block_select(const sb_heads* q, int dtype, const float* means, const int32_t* kv_lens, const int32_t* q_lens, int batch,
                    int q_heads, int kv_heads, int q_rows, int kv_rows, int head_dim, int block, int topk, int keep_first,
                    int keep_own, int32_t* index, void* stream) {
  const char* what = "block_select";
  if (!float_dtype(dtype)) return fail(SB_ERR_UNSUPPORTED, "%s: dtype %d (f32, f16, bf16)", what, dtype);
  if (batch < 0 || q_heads < 1 || kv_heads < 1 || q_rows < 0 || kv_rows < 0 || block < 1)
    return fail(SB_ERR_INVALID_ARG, "%s: bad sizes", what);
  if ((long long)kv_rows + block > 0x7fffffffll) return fail(SB_ERR_UNSUPPORTED, "%s: rows and block exceed 2^31", what);
  if (q_heads % kv_heads) return fail(SB_ERR_INVALID_ARG, "%s: %d query heads over %d key heads", what, q_heads, kv_heads);
  if (head_dim < 1 || head_dim > kSelMaxDim)
    return fail(SB_ERR_UNSUPPORTED, "%s: head_dim %d (1 to %d)", what, head_dim, kSelMaxDim);
  if (topk < 1 || topk > kSelMaxTopk) return fail(SB_ERR_UNSUPPORTED, "%s: topk %d (1 to %d)", what, topk, kSelMaxTopk);
  if (keep_first < 0 || keep_first + (keep_own ? 1 : 0) > topk)
    return fail(SB_ERR_INVALID_ARG, "%s: %d forced blocks exceed topk %d", what, keep_first + (keep_own ? 1 : 0), topk);
  const long long nb = cdiv(kv_rows, block);
  if (nb > kSelMaxBlocks) return fail(SB_ERR_UNSUPPORTED, "%s: %lld blocks (at most %d)", what, nb, kSelMaxBlocks);
  if (batch == 0 || q_rows == 0) return SB_OK;
  const int e = elem_size(dtype);
  if (int s = check_heads(what, "q", q, e)) return s;
  if ((nb > 0 && !means) || !index) return fail(SB_ERR_INVALID_ARG, "%s: means or index is NULL", what);
  if ((uintptr_t)means % 4 || (uintptr_t)index % 4 || (uintptr_t)kv_lens % 4 || (uintptr_t)q_lens % 4)
    return fail(SB_ERR_INVALID_ARG, "%s: an operand is misaligned", what);
  SelArgs a{};
  a.q = view(q);
  a.means = means;
  a.kv_lens = kv_lens;
  a.q_lens = q_lens;
  a.out = index;
  a.batch = batch;
  a.kv_heads = kv_heads;
  a.group = q_heads / kv_heads;
  a.q_rows = q_rows;
  a.kv_rows = kv_rows;
  a.dim = head_dim;
  a.nb = (int)nb;
  a.block = block;
  a.topk = topk;
  a.keep_first = keep_first;
  a.keep_own = keep_own != 0;
  a.q_vec = head_dim % 8 == 0 && heads_vec(q, e, 16 / e) == 16 / e;
  cudaStream_t st = (cudaStream_t)stream;
  if (q_rows <= kSelFewRows) {
    const long long rows = (long long)batch * kv_heads * q_rows;
    // CTAs of a row: enough that the means are read by every SM, each with some rows to read
    int cluster = 1;
    while (cluster < kSelFewCluster && rows * cluster < 2 * num_sms() && nb >= 64 * cluster) cluster *= 2;
    if (rows * cluster > 0x7fffffffll) return fail(SB_ERR_UNSUPPORTED, "%s: too many rows for one launch", what);
    if (dtype == SB_F32) return launch_select_few<float>(a, (unsigned)rows, cluster, st);
    if (dtype == SB_F16) return launch_select_few<__half>(a, (unsigned)rows, cluster, st);
    return launch_select_few<__nv_bfloat16>(a, (unsigned)rows, cluster, st);
  }
  // the widest tile that leaves the three CTAs an SM which registers allow their
  // shared memory (16 x 2440 rows, 8 heads of 16, limits of 40 / 56 / 72 KB: 191 / 155 /
  // 155 us at 41 blocks, 293 / 292 / 270 at 96, the same at others), or two of them
  // where 64 rows are too many for that (112 KB, or 72: 1248 and 1039 us at 256 blocks,
  // 3976 and 4940 at 1024), no wider than the rows
  int tile = 128;
  while (tile > 64 && (sel_smem_bytes(tile, a.nb, head_dim) > 56 * 1024 || tile / 2 >= q_rows)) tile >>= 1;
  while (tile > 2 && (sel_smem_bytes(tile, a.nb, head_dim) > 112 * 1024 || tile / 2 >= q_rows)) tile >>= 1;
  a.tile = tile;
  a.tiles = (int)cdiv(q_rows, tile);
  const long long grid = (long long)batch * kv_heads * a.tiles;
  if (grid > 0x7fffffffll) return fail(SB_ERR_UNSUPPORTED, "%s: too many rows for one launch", what);
  if (dtype == SB_F32) return launch_select<float>(a, (unsigned)grid, st);
  if (dtype == SB_F16) return launch_select<__half>(a, (unsigned)grid, st);
  return launch_select<__nv_bfloat16>(a, (unsigned)grid, st);
}

int sb_block_attention_workspace_bytes(int batch, int q_heads, int kv_heads, int q_rows, int kv_rows, int head_dim, int block,
                                       int topk, int backward, size_t* bytes) {
  if (!bytes) return fail(SB_ERR_INVALID_ARG, "block_attention: bytes is NULL");
  if (int s = check_ba("block_attention", SB_F16, batch, q_heads, kv_heads, q_rows, kv_rows, head_dim, block, topk)) return s;
  *bytes = 0;
  if (batch == 0 || q_rows == 0 || (!backward && q_rows <= kBaFewRows)) return SB_OK;
  *bytes = ba_plan((long long)batch * kv_heads, q_rows, q_heads / kv_heads, head_dim, (int)cdiv(kv_rows, block), block, topk,
                   backward != 0)
               .total;
  return SB_OK;
}

int sb_block_attention(const sb_heads* q, const sb_heads* k, const sb_heads* v, int dtype, const int32_t* index,
                       const int32_t* kv_lens, const int32_t* q_lens, int batch, int q_heads, int kv_heads, int q_rows,
                       int kv_rows, int head_dim, int block, int topk, float scale, const sb_heads* out, float* lse,
                       void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "block_attention";
  if (int s = check_ba(what, dtype, batch, q_heads, kv_heads, q_rows, kv_rows, head_dim, block, topk)) return s;
  if (!std::isfinite(scale)) return fail(SB_ERR_INVALID_ARG, "%s: scale is not finite", what);
  if (batch == 0 || q_rows == 0) return SB_OK;
  if (int s = check_heads16(what, "q", q)) return s;
  if (int s = check_heads16(what, "out", out)) return s;
  if (kv_rows > 0) {
    if (int s = check_heads16(what, "k", k)) return s;
    if (int s = check_heads16(what, "v", v)) return s;
  }
  if (!index || !lse) return fail(SB_ERR_INVALID_ARG, "%s: index or lse is NULL", what);
  if ((uintptr_t)index % 4 || (uintptr_t)lse % 4 || (uintptr_t)kv_lens % 4 || (uintptr_t)q_lens % 4)
    return fail(SB_ERR_INVALID_ARG, "%s: an operand is misaligned", what);
  BaArgs a{};
  ba_fill(&a, index, kv_lens, q_lens, batch, q_heads, kv_heads, q_rows, kv_rows, head_dim, block, topk, scale);
  a.q = view(q);
  if (kv_rows > 0) {
    a.k = view(k);
    a.v = view(v);
  }
  a.o = view(out);
  a.lse = lse;
  cudaStream_t st = (cudaStream_t)stream;
  if (q_rows <= kBaFewRows) return ba_dispatch(dtype, head_dim, block, LaunchFew{a, st});
  const BaPlan p = ba_plan((long long)batch * kv_heads, q_rows, a.group, head_dim, a.nb, block, topk, false);
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < p.total)
    return fail(SB_ERR_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed", what, p.total);
  char* ws = (char*)workspace;
  a.marks = p.marks;
  a.entries = (uint16_t*)(ws + p.entries);
  a.spans = (uint32_t*)(ws + p.spans);
  a.slots = (unsigned long long*)(ws + p.slots);
  a.part = (float*)(ws + p.part);
  a.ml = (float2*)(ws + p.ml);
  a.ticket = (uint32_t*)(ws + p.ticket);
  return ba_windows(a, p, st, [&] { return ba_dispatch(dtype, head_dim, block, LaunchFwd{a, st}); }, [] { return SB_OK; });
}

int sb_block_attention_backward(const sb_heads* dout, const sb_heads* q, const sb_heads* k, const sb_heads* v,
                                const sb_heads* out, const float* lse, int dtype, const int32_t* index,
                                const int32_t* kv_lens, const int32_t* q_lens, int batch, int q_heads, int kv_heads,
                                int q_rows, int kv_rows, int head_dim, int block, int topk, float scale, const sb_heads* dq,
                                const sb_heads* dk, const sb_heads* dv, void* workspace, size_t workspace_bytes,
                                void* stream) {
  const char* what = "block_attention_backward";
  if (int s = check_ba(what, dtype, batch, q_heads, kv_heads, q_rows, kv_rows, head_dim, block, topk)) return s;
  if (!std::isfinite(scale)) return fail(SB_ERR_INVALID_ARG, "%s: scale is not finite", what);
  if (batch == 0) return SB_OK;
  if (q_rows == 0) return fail(SB_ERR_UNSUPPORTED, "%s: no query rows", what);
  const sb_heads* ts[4] = {dout, q, out, dq};
  const char* tn[4] = {"dout", "q", "out", "dq"};
  for (int i = 0; i < 4; ++i)
    if (int s = check_heads16(what, tn[i], ts[i])) return s;
  const sb_heads* ks[4] = {k, v, dk, dv};
  const char* kn[4] = {"k", "v", "dk", "dv"};
  for (int i = 0; i < 4 && kv_rows > 0; ++i)
    if (int s = check_heads16(what, kn[i], ks[i])) return s;
  if (!index || !lse) return fail(SB_ERR_INVALID_ARG, "%s: index or lse is NULL", what);
  if ((uintptr_t)index % 4 || (uintptr_t)lse % 4 || (uintptr_t)kv_lens % 4 || (uintptr_t)q_lens % 4)
    return fail(SB_ERR_INVALID_ARG, "%s: an operand is misaligned", what);
  BaArgs a{};
  ba_fill(&a, index, kv_lens, q_lens, batch, q_heads, kv_heads, q_rows, kv_rows, head_dim, block, topk, scale);
  a.q = view(q);
  a.o = view(out);
  a.go = view(dout);
  a.dq = view(dq);
  if (kv_rows > 0) {
    a.k = view(k);
    a.v = view(v);
    a.dk = view(dk);
    a.dv = view(dv);
  }
  a.lse = const_cast<float*>(lse);
  const long long bh = (long long)batch * kv_heads;
  const BaPlan p = ba_plan(bh, q_rows, a.group, head_dim, a.nb, block, topk, true);
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < p.total)
    return fail(SB_ERR_WORKSPACE, "%s: workspace of %zu bytes, 256-byte aligned, needed", what, p.total);
  char* ws = (char*)workspace;
  a.marks = p.marks;
  a.entries = (uint16_t*)(ws + p.entries);
  a.spans = (uint32_t*)(ws + p.spans);
  a.slots = (unsigned long long*)(ws + p.slots);
  a.part = (float*)(ws + p.part);
  a.delta = (float2*)(ws + p.delta);
  a.kv_part = (float*)(ws + p.kv_part);
  a.ticket = (uint32_t*)(ws + p.ticket);
  a.sums = p.sums;
  cudaStream_t st = (cudaStream_t)stream;
  const int chunks = 1 << pow2_log2(head_dim / 8);
  const long long dgrid = cdiv(bh * q_rows * a.group * chunks, 256);
  const bool f16 = dtype == SB_F16;
  if (int s = f16 ? launch_ba(block_attn_delta_kernel<__half>, "block_attn_delta_kernel", dgrid, 256, 0, a, st)
                  : launch_ba(block_attn_delta_kernel<__nv_bfloat16>, "block_attn_delta_kernel", dgrid, 256, 0, a, st))
    return s;
  return ba_windows(
      a, p, st, [&] { return ba_dispatch(dtype, head_dim, block, LaunchBwd{a, st}); },
      [&] {
        if (a.sums == 0) return (int)SB_OK;
        const long long kgrid = cdiv((long long)a.nbh * kv_rows * (head_dim / 8), 256);
        return f16 ? launch_ba(block_attn_dkv_kernel<__half>, "block_attn_dkv_kernel", kgrid, 256, 0, a, st)
                   : launch_ba(block_attn_dkv_kernel<__nv_bfloat16>, "block_attn_dkv_kernel", kgrid, 256, 0, a, st);
      });
}

}  // extern "C"
