// layer_kernels.hip -- the kernels on the way into the experts and beside them (kernels_norm.h,
// kernels_route.h, kernels_adapters.h) and their launches.
#include "layer_kernels.h"

#include "../../include/moe_block.h"
#include "kernels_adapters.h"
#include "kernels_norm.h"
#include "kernels_route.h"
#include "launch_common.h"

#include <type_traits>

// Outputs of more than this go past the caches: a kernel ends only when the caches have written back what it left
// there, and the next one reads it from the memory's cache as fast.  us, through them / past them, norm and then
// moe_quantize_i8 of its y, H = 7168 bf16 with residual:  64 rows (1.8 MB) 7.5 / 7.6, 512 (14.7 MB) 15.8 / 13.0, 1500
// 31.0 / 29.5, 4096 62.0 / 60.4; 2000 of 2048 (16.4 MB) 16.1 / 14.2, 8191 36.6 / 36.3.  The gradient alone, with dres: 509 rows of 5120
// f32 17.8 / 15.7, 4096 of 7168 bf16 54.4 / 54.1, 2048 of 7168 f32 52.1 / 52.3; adapters, 4096 rows of 7168 x 64 x 7168 bf16 60.5 / 56.3.
static constexpr size_t MOE_LAYER_STREAM_BYTES = (size_t)4 << 20;

// f(integral_constant) for the bytes of an element of type t.
template <typename F>
static void with_size(int t, F f) {
  if (t == MOE_GGML_F32) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 2>{});
}

template <int SX, int SR, int LANES, int VPT>
static bool launch_norm(const norm_call &a, hipStream_t st) {
  constexpr int NT = LANES < 256 ? 256 : LANES;
  const int n = ceil_div(a.T, NT / LANES);
  if (!fits(n, NT)) return false;
  hipLaunchKernelGGL((k_rms_norm<SX, SR, LANES, VPT>), dim3(n), dim3(NT), 0, st, a);
  return true;
}

// Threads a row and vectors a thread.  A row of 4097 to 8192 in one vector a thread where the rows are too few to fill
// the chip.  us, bf16 with residual, output in values / in 8 bits (* the rule's):
//   threads x vectors:      1024 x 1         512 x 2          256 x 4          (128 x 8: 4096 rows 80 / 90)
//   4096 rows of 7168       47.6  / 54.6     45.7* / 48.1*    49.9  / 45.4
//   600 of 7168             8.4   / 13.0     9.6*  / 12.0*    9.0   / 11.0
//   500 of 7168             6.9*  / 9.7*     7.1   / 8.9      8.0   / 9.4
//   509 of 5120             7.4*  / 9.9*     7.7   / 8.9      8.1   / 8.9
//   one of 7168             3.6*             4.0              5.2
//                           256 x 1          128 x 2          64 x 4
//   8191 of 2048            26.8* / 26.4*    27.9  / 22.8     28.9  / 24.0
//                           128 x 1          64 x 2
//   8191 of 1024            14.7* / 15.1*    15.4  / 13.6
// The rule is the one for values at both ends, one row and thousands.  In 8 bits, bound by instructions, half the threads would
// take up to a seventh off; the rule does not look at the output.
template <int SX, int SR>
static bool launch_norm(const norm_call &a, int n_cu, hipStream_t st) {
  const int H = a.H;
  if (H <= 128) return launch_norm<SX, SR, 16, 1>(a, st);
  if (H <= 512) return launch_norm<SX, SR, 64, 1>(a, st);
  if (H <= 1024) return launch_norm<SX, SR, 128, 1>(a, st);
  if (H <= 2048) return launch_norm<SX, SR, 256, 1>(a, st);
  if (H <= 4096) return launch_norm<SX, SR, 256, 2>(a, st);
  if (H <= 8192 && a.T < 2 * n_cu) return launch_norm<SX, SR, 1024, 1>(a, st);
  if (H <= 8192) return launch_norm<SX, SR, 512, 2>(a, st);
  if (H <= 16384) return launch_norm<SX, SR, 1024, 2>(a, st);
  return launch_norm<SX, SR, 1024, 4>(a, st);
}

bool launch_rms_norm(const norm_call &args, int n_cu, hipStream_t st) {
  norm_call a = args;
  if (a.H > 32768) {
    if (!fits(a.T, 256)) return false;
    hipLaunchKernelGGL(k_rms_norm_long, dim3(a.T), dim3(256), 0, st, a);
    return true;
  }
  auto size = [](const void *p, int type) { return p ? type == MOE_GGML_F32 ? 4 : 2 : 0; };
  a.nt = (size_t)a.T * a.H * (size(a.total, a.res_type) + size(a.y, a.y_type) + (a.q ? 1 : 0)) > MOE_LAYER_STREAM_BYTES;
  bool fine = false;
  with_size(a.x_type, [&](auto sx) {
    if (!a.res) fine = launch_norm<sx, 0>(a, n_cu, st);
    else with_size(a.res_type, [&](auto sr) { fine = launch_norm<sx, sr>(a, n_cu, st); });
  });
  return fine;
}

// The gradient's workgroups walk rows, G of them at once, one workgroup a CU: each has a share of dw.
static int grad_groups(int H) { return H <= 128 ? 64 : H <= 512 ? 16 : H <= 1024 ? 8 : H <= 2048 ? 4 : H <= 4096 ? 2 : 1; }
static int grad_blocks(int T, int H, int n_cu) {
  const int most = ceil_div(T, grad_groups(H));
  return most < n_cu ? most : n_cu;
}

size_t norm_grad_need(int T, int H, int n_cu) { return H > 16384 ? 1 : (size_t)grad_blocks(T, H, n_cu) * H; }

// Grows with T and H: a workspace for the largest call serves every smaller one.  (Longer rows have no shares, and the
// workspace of rows of 16384.)
size_t norm_grad_scratch(int T, int H, int n_cu) { return norm_grad_need(T, H < 16384 ? H : 16384, n_cu); }

template <int SD, int SH, int SX, int LANES, int VPT, int G>
static void launch_grad(const norm_grad_call &a, int n, hipStream_t st) {
  hipLaunchKernelGGL((k_rms_norm_grad<SD, SH, SX, LANES, VPT, G>), dim3(n), dim3(LANES * G), 0, st, a);
}

template <int SD, int SH, int SX>
static void launch_grad(const norm_grad_call &a, int n, hipStream_t st) {
  const int H = a.H;
  if (H <= 128) launch_grad<SD, SH, SX, 16, 1, 64>(a, n, st);
  else if (H <= 512) launch_grad<SD, SH, SX, 64, 1, 16>(a, n, st);
  else if (H <= 1024) launch_grad<SD, SH, SX, 128, 1, 8>(a, n, st);
  else if (H <= 2048) launch_grad<SD, SH, SX, 256, 1, 4>(a, n, st);
  else if (H <= 4096) launch_grad<SD, SH, SX, 512, 1, 2>(a, n, st);
  else if (H <= 8192) launch_grad<SD, SH, SX, 1024, 1, 1>(a, n, st);
  else launch_grad<SD, SH, SX, 512, 4, 1>(a, n, st);
}

bool launch_rms_norm_grad(const norm_grad_call &args, int n_cu, hipStream_t st) {
  norm_grad_call a = args;
  a.nt = (size_t)a.T * a.H * (a.dx_type == MOE_GGML_F32 ? 4 : 2) > MOE_LAYER_STREAM_BYTES;
  if (a.H > 16384) {
    if (!fits(a.T, 256)) return false;
    hipLaunchKernelGGL(k_rms_norm_dx_long, dim3(a.T), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_rms_norm_dw_long, dim3(ceil_div(a.H, 64)), dim3(256), 0, st, a);
    return true;
  }
  const int n = grad_blocks(a.T, a.H, n_cu);
  with_size(a.dy_type, [&](auto sd) {
    with_size(a.h_type, [&](auto sh) { with_size(a.dx_type, [&](auto sx) { launch_grad<sd, sh, sx>(a, n, st); }); });
  });
  if (n > 1) hipLaunchKernelGGL(k_rms_norm_dw, dim3(ceil_div(a.H, 64)), dim3(1024), 0, st, a.part, n, a.H, a.dw);
  return true;
}

template <int NJ>
static void launch_route(route_call a, hipStream_t st) {
  const int n = a.per / NJ;
  if (a.per % NJ == 0 && n <= 16 && (n & (n - 1)) == 0) a.lanes = n;
  if (a.T >= 1024) hipLaunchKernelGGL((k_route_groups<NJ, 4>), dim3(ceil_div(a.T, 4)), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_route_groups<NJ, 1>), dim3(a.T), dim3(64), 0, st, a);
}

bool launch_route_groups(const route_call &args, hipStream_t st) {
  if (!fits(args.T, 64)) return false;
  route_call a = args;
  a.per = a.E / a.n_group;
  for (a.width = 16; a.width * a.n_group > 64;) a.width >>= 1;
  if (a.E <= 64) launch_route<1>(a, st);
  else if (a.E <= 128) launch_route<2>(a, st);
  else if (a.E <= 256) launch_route<4>(a, st);
  else if (a.E <= 512) launch_route<8>(a, st);
  else launch_route<16>(a, st);
  return true;
}

template <int NJ>
static void launch_grad(const route_grad_call &a, hipStream_t st) {
  if (a.T >= 1024) hipLaunchKernelGGL((k_route_grad<NJ, 4>), dim3(ceil_div(a.T, 4)), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_route_grad<NJ, 1>), dim3(a.T), dim3(64), 0, st, a);
}

bool launch_route_grad(const route_grad_call &a, hipStream_t st) {
  if (!fits(a.T, 64)) return false;
  if (a.E <= 64) launch_grad<1>(a, st);
  else if (a.E <= 128) launch_grad<2>(a, st);
  else if (a.E <= 256) launch_grad<4>(a, st);
  else if (a.E <= 512) launch_grad<8>(a, st);
  else launch_grad<16>(a, st);
  return true;
}

// Rows of an adapter a workgroup, and the waves of one that multiplies with A: 64 KB of results meet in LDS.
static int adapters_tile(int M) { return M <= 64 ? 16 : 32; }
static constexpr int shrink_waves(int MT, int RT) { return MT * RT <= 2 ? 16 : 8; }

static int split_waves(int M, int R) { return shrink_waves(adapters_tile(M) / 16, R <= 16 ? 1 : R <= 32 ? 2 : 4); }
// Pieces of K that the product with A is cut into: 16 waves a CU where every tile is full, two steps a wave at least.
static int most_splits(int M, int K, int R) { return ceil_div(K, 64 * split_waves(M, R)); }
static int adapters_splits(int M, int K, int R, int n_cu) {
  const int most = most_splits(M, K, R), want = ceil_div(16L * n_cu, (long)ceil_div(M, adapters_tile(M)) * split_waves(M, R));
  return most < want ? most : want;
}

size_t adapters_need(int M, int K, int R, int n_cu) { return (size_t)adapters_splits(M, K, R, n_cu) * M * R; }

// The pieces get fewer as the tiles get more, so what a call needs goes up and down with M.  This is a bound that grows
// with M, K and R, so that a workspace for the largest call serves every smaller one: of M rows in t tiles of h, the
// ceil(16 n_cu / (t w)) pieces have fewer than 16 n_cu h / w + M rows.  (h / w grows with M and R, from 1 to 4, and so does
// the most pieces of K, as w falls.)
size_t adapters_scratch(int M, int K, int R, int n_cu) {
  const size_t some = (size_t)16 * n_cu * adapters_tile(M) / split_waves(M, R) + M, all = (size_t)most_splits(M, K, R) * M;
  return (some < all ? some : all) * R;
}

template <typename T, int MT, int RT>
static void launch_shrink(const adapters_call &a, long tiles, hipStream_t st) {
  constexpr int W = shrink_waves(MT, RT);
  hipLaunchKernelGGL((k_adapters_shrink<T, MT, RT, W>), dim3((unsigned)(tiles * a.splits), ceil_div(a.R, 16 * RT)), dim3(64 * W), 0,
                     st, a);
}
template <typename T, int MT>
static void launch_shrink(const adapters_call &a, long tiles, hipStream_t st) {
  if (a.R <= 16) launch_shrink<T, MT, 1>(a, tiles, st);
  else if (a.R <= 32) launch_shrink<T, MT, 2>(a, tiles, st);
  else launch_shrink<T, MT, 4>(a, tiles, st);
}

template <typename T, typename TO, int MT>
static void launch_expand(const adapters_call &a, long tiles, hipStream_t st) {
  hipLaunchKernelGGL((k_adapters_expand<T, TO, MT>), dim3((unsigned)(tiles * a.col_blocks)), dim3(256), 0, st, a);
}

bool launch_adapters(const adapters_call &args, int n_cu, hipStream_t st) {
  adapters_call a = args;
  const int matrices = a.M < a.n ? a.M : a.n, each = a.M / matrices;  // adapters that can have rows; rows of each
  const size_t size = a.type == MOE_GGML_F32 ? 4 : 2;
  // Staged where adapters have rows for its tiles: the product with A from rank 33 on, the one with B where there are
  // three workgroups for two CUs.  us, staged / straight to registers (bf16 rows x K x rank x N, adapters; * the rule's):
  //   with A:  4096 x 7168 x 64 x 7168, 8   56.8* / 62.7   x 32  49.2 / 50.8*   x 16  54.0 / 45.8*
  //            2048 x 2048 x 64 x 2048, 16 (f32)  35.5* / 39.0    2048 x 768 x 8 x 768, 60 (f32)  27.0 / 13.7*
  //   with B:  4096 x 7168 x 64 x 7168, 8   56.4* / 67.8   x 16  45.9* / 56.9
  //            2048 x 4096 x 64 x 4096, 16   27.9* / 32.8   x 16  24.2* / 27.6    1024 x 7168 x 64 x 7168, 4  25.7* / 28.5
  //            2048 x 2048 x 64 x 2048, 16 (f32)  42.8 / 35.4*   (f16)  24.4 / 20.6*    512 x 4096 x 32 x 4096, 16  16.5 / 12.8*
  //   both at 16 rows an adapter: 517 x 2048 x 8 x 768, 32  17.2 / 8.9*
  // `each` counts adapters that are there, not those with rows, which only the device knows: 4096 rows of four of 256 adapters
  // take 114 us in 16-row tiles, of four of 64 60.6.
  const bool staged_a = each >= 32 && a.R > 32 && a.K * size % 16 == 0 && ((uintptr_t)a.x | (uintptr_t)a.a) % 16 == 0 &&
                        (uint64_t)a.M * a.K * size < MOE_LDS_OOB && (uint64_t)a.R * a.K * size < MOE_LDS_OOB;
  const bool staged_b = each >= 32 && 2L * ceil_div(a.M, 64) * ceil_div(a.N, 256) >= 3 * n_cu && a.R <= 64 &&
                        a.R * size % 16 == 0 && (uintptr_t)a.b % 16 == 0 && (uint64_t)a.N * a.R * size < MOE_LDS_OOB;
  // no larger a tile than the adapters' rows fill
  const int BM = each <= 16 ? 16 : adapters_tile(a.M), groups = ceil_div(a.N, staged_b ? 256 : 128);
  auto tiles_of = [&](int rows) { return (a.M + (long)matrices * (rows - 1)) / rows; };
  const long tiles_a = tiles_of(staged_a ? 64 : BM), tiles_b = tiles_of(staged_b ? 64 : BM);
  a.splits = adapters_splits(a.M, a.K, a.R, n_cu);
  a.piece = ceil_div(ceil_div(a.K, a.splits), 64) * 64;
  // several groups of columns for one reading of mid, as long as there are four workgroups a CU
  const long wide = (long)ceil_div(a.M, BM) * groups / (4 * n_cu);
  a.col_groups = wide < 1 || staged_b ? 1 : wide < groups ? (int)wide : groups;
  a.col_blocks = ceil_div(groups, a.col_groups);
  a.nt = (size_t)a.M * a.N * (a.out_type == MOE_GGML_F32 ? 4 : 2) > MOE_LAYER_STREAM_BYTES;
  if (!fits(tiles_a * a.splits, 1024) || !fits(tiles_b * a.col_blocks, 256)) return false;
  with_type(a.type, [&](auto t) {
    typedef decltype(t) T;
    constexpr int NBUF = 5;
    if (staged_a)
      hipLaunchKernelGGL((k_adapters_shrink_staged<T, NBUF>), dim3((unsigned)(tiles_a * a.splits), ceil_div(a.R, 64)), dim3(256),
                         NBUF * 128 * 128, st, a);
    else if (BM == 16) launch_shrink<T, 1>(a, tiles_a, st);
    else launch_shrink<T, 2>(a, tiles_a, st);
    with_type(a.out_type, [&](auto to) {
      typedef decltype(to) TO;
      if (staged_b)
        hipLaunchKernelGGL((k_adapters_expand_staged<T, TO>), dim3((unsigned)(tiles_b * a.col_blocks)), dim3(256), 0, st, a);
      else if (BM == 16) launch_expand<T, TO, 1>(a, tiles_b, st);
      else launch_expand<T, TO, 2>(a, tiles_b, st);
    });
  });
  return true;
}
