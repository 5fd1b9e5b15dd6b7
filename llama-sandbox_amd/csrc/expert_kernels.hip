// expert_kernels.hip -- the kernels around the expert products (kernels_dispatch.h,
// kernels_i8.h) and their launches: which variant a call takes, and its grid.
#include "expert_kernels.h"

#include "../../include/moe_block.h"
#include "kernels_dispatch.h"
#include "kernels_i8.h"

#include <cmath>

static int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

// A grid's x dimension holds fewer than 2^32 threads.
static bool fits(long blocks, int threads) { return blocks * threads < (1L << 32); }

// f(T{}) for the element type t.
template <typename F>
static void with_type(int t, F f) {
  if (t == MOE_GGML_F32) f(float{});
  else if (t == MOE_GGML_F16) f(_Float16{});
  else f(bf16_t{});
}

// Elements a thread takes at once: 16 bytes, or 8 elements where a side has 16 bits.
template <typename A, typename B>
constexpr int vec_of() { return sizeof(A) == 4 && sizeof(B) == 4 ? 4 : 8; }

// Rows of more than this go past the caches (non-temporal): they displace what
// the next kernels could find in the 256 MiB cache, and the plain form spends its
// bandwidth on writing back what it displaced.  Measured with H = 7168, us
// plain / non-temporal: dispatch of 59 MB 11.6 / 12.4, 117 MB 28.4 / 24.7, 470 MB
// 108 / 95; combine 59 MB 11.9 / 12.5, 117 MB 29.0 / 25.8, 470 MB 110 / 98;
// combine_grad (read and written) 59 MB 12.1 / 13.3, 117 MB 27.6 / 25.2, 940 MB 207 / 195.
static constexpr size_t MOE_STREAM_BYTES = (size_t)96 << 20;

// Pairs below which 4 waves share one of combine_grad's (H = 7168, bf16, us with 1
// wave / 4: 128 pairs 6.0 / 3.7, 512 7.7 / 5.4, 1024 8.8 / 8.4, 2048 12.1 / 13.3).
static constexpr long MOE_FEW_PAIRS = 1024;

// Workgroups a token of nv vectors: enough for the chip, no more than have work.
static int row_splits(int T, int nv) {
  const int most = ceil_div(nv, 256), want = ceil_div(2048, T);
  return most < want ? most : want;
}

bool launch_dispatch(const void *x, int x_type, const int32_t *inv, int T, int k, int H, int n_rows, void *rows,
                     int rows_type, hipStream_t st) {
  if (!fits(T, 256)) return false;
  with_type(x_type, [&](auto ti) {
    with_type(rows_type, [&](auto to) {
      typedef decltype(ti) TI;
      typedef decltype(to) TO;
      constexpr int V = vec_of<TI, TO>();
      const bool nt = (size_t)T * k * H * sizeof(TO) > MOE_STREAM_BYTES;
      hipLaunchKernelGGL((nt ? k_dispatch<TI, TO, V, true> : k_dispatch<TI, TO, V, false>),
                         dim3(T, row_splits(T, ceil_div(H, V))), dim3(256), 0, st, (const TI *)x, inv, k, H, n_rows,
                         (TO *)rows);
    });
  });
  return true;
}

bool launch_combine_rows(const void *rows, int rows_type, int n_rows, const float *wts, const int32_t *inv, int T, int k,
                         int H, void *out, int out_type, hipStream_t st) {
  if (!fits(T, 256)) return false;
  with_type(rows_type, [&](auto ti) {
    with_type(out_type, [&](auto to) {
      typedef decltype(ti) TI;
      typedef decltype(to) TO;
      constexpr int V = vec_of<TI, TO>();
      const bool nt = (size_t)T * k * H * sizeof(TI) > MOE_STREAM_BYTES;
      hipLaunchKernelGGL((nt ? k_combine_rows<TI, TO, V, true> : k_combine_rows<TI, TO, V, false>),
                         dim3(T, row_splits(T, ceil_div(H, V))), dim3(256), 0, st, (const TI *)rows, wts, inv, k, H, n_rows,
                         (TO *)out);
    });
  });
  return true;
}

bool launch_combine_grad(const void *dout, int dout_type, const void *rows, int rows_type, int n_rows, const float *wts,
                         const int32_t *inv, int T, int k, int H, void *drows, float *dwts, hipStream_t st) {
  const long P = (long)T * k;
  if (!fits((P + 7) / 8, 512)) return false;
  with_type(dout_type, [&](auto td) {
    with_type(rows_type, [&](auto tr) {
      typedef decltype(td) TD;
      typedef decltype(tr) TR;
      constexpr int V = vec_of<TD, TR>();
      const bool nt = 2 * (size_t)P * H * sizeof(TR) > MOE_STREAM_BYTES, few = P < MOE_FEW_PAIRS && H >= 256 * V;
      hipLaunchKernelGGL((few ? k_combine_grad<TD, TR, V, 4, false> : nt ? k_combine_grad<TD, TR, V, 1, true>
                                                                         : k_combine_grad<TD, TR, V, 1, false>),
                         dim3((unsigned)(few ? (P + 1) / 2 : (P + 7) / 8)), dim3(512), 0, st, (const TD *)dout,
                         (const TR *)rows, wts, inv, P, k, H, n_rows, (TR *)drows, dwts);
    });
  });
  return true;
}

template <typename T, int LANES, int VPT>
static void launch_quantize(const T *x, int M, int K, int8_t *q, float *scale, hipStream_t st) {
  constexpr int rows = LANES < 256 ? 256 / LANES : 1;
  hipLaunchKernelGGL((k_quantize_i8<T, LANES, VPT>), dim3(ceil_div(M, rows)), dim3(LANES < 256 ? 256 : LANES), 0, st, x, M,
                     K, q, scale);
}

// One vector a thread where the rows are too few to fill the chip (a row is
// then spread as wide as it goes), else as many rows at once as registers allow.
bool launch_quantize_i8(const void *x, int x_type, int M, int K, int8_t *q, float *scale, int n_cu, hipStream_t st) {
  if (!fits(M, K > 8192 ? 1024 : 256)) return false;
  with_type(x_type, [&](auto t) {
    typedef decltype(t) T;
    const T *p = (const T *)x;
    if (M < 2 * n_cu && K > 512 && K <= 8192) {
      if (K <= 2048) launch_quantize<T, 256, 1>(p, M, K, q, scale, st);
      else launch_quantize<T, 1024, 1>(p, M, K, q, scale, st);
    }
    else if (K <= 256) launch_quantize<T, 32, 1>(p, M, K, q, scale, st);
    else if (K <= 512) launch_quantize<T, 64, 1>(p, M, K, q, scale, st);
    else if (K <= 768 && M >= 8 * n_cu) launch_quantize<T, 32, 3>(p, M, K, q, scale, st);
    else if (K <= 1024) launch_quantize<T, 64, 2>(p, M, K, q, scale, st);
    else if (K <= 2048) launch_quantize<T, 64, 4>(p, M, K, q, scale, st);
    else if (K <= 4096) launch_quantize<T, 256, 2>(p, M, K, q, scale, st);
    else if (K <= 6144) launch_quantize<T, 256, 3>(p, M, K, q, scale, st);
    else if (K <= 8192) launch_quantize<T, 256, 4>(p, M, K, q, scale, st);
    else if (K <= 32768) launch_quantize<T, 1024, 4>(p, M, K, q, scale, st);
    else hipLaunchKernelGGL((k_quantize_i8_long<T>), dim3(M), dim3(256), 0, st, p, K, q, scale);
  });
  return true;
}

// Tiles of at most BM rows that M rows of E experts can make.
static long i8_tiles(const i8_mm &a, int BM) {
  const long n = a.offsets ? (a.M < a.E ? a.M : a.E) : 1;  // matrices: each rounds up
  return (a.M + n * (BM - 1)) / BM;
}

// The launch of a product by one kernel; false: more workgroups than a grid takes.
typedef bool (*i8_launch)(const i8_mm &, hipStream_t);

template <int M, int C, int U>
static bool launch_few(const i8_mm &a, hipStream_t st) {
  const int nt = ceil_div(a.swiglu ? a.N / 2 : a.N, a.swiglu ? C / 2 : C);
  const long n = i8_tiles(a, M) * nt;
  if (!fits(n, 64)) return false;
  hipLaunchKernelGGL((k_mv_i8<M, C, U>), dim3((unsigned)n), dim3(64), 0, st, a, nt);
  return true;
}

// The launch of a call whose rows are few enough for k_mv_i8 (else NULL).  More rows a tile read
// the weights less often, fewer spread them wider.  us, rows x K x N:
//   rows a tile, channels:   1, 2    1, 4    2, 4    4, 2   staged
//   1 x 4096 x 4096          5.14    5.40    5.62    5.76    7.29
//   2 x 2048 x 7168          6.31    5.68    5.47    5.58    6.51
//   4 x 4096 x 4096          7.36    7.09    6.34    6.01    7.29
//   4 x 7168 x 7168          29.5    26.2    15.9    14.4    13.5
//   8 x 7168 x 512           4.46    4.74    5.15    5.41    7.05
//   8 x 2048 x 1024          4.27    3.71    3.69    3.75    4.48
//   8 x 7168 x 2048          10.2     8.6     7.0     7.1     7.2
//   32 x 7168 x 256          5.86    5.61    5.43    5.60    6.97
//   2 tokens' 8 experts of 2048 x 7168, and 4's:
//                            51.5    37.4    37.4    52.5    42.8
//                            98.7    70.4    69.6    98.4    75.5
// Grouped rows are taken one a tile, up to 16 of them: an expert's weights are then read
// as often as it has rows (128 rows of 16 tokens, Zipf, 7168 x 4096: 280 us against 165 staged).  So
// where an expert has 2 rows or more on average, only matrices that the second read finds in L2, and
// up to 4 rows.  us, one a tile / staged, random experts, weights from HBM where they are more than the caches hold:
//   rows, experts:       16, 1       16, 2       16, 4        16, 8        16, 12       16, 16       4, 2
//   7168 x 7168      88.5 / 13.6  90.0 / 19.9  95.1 / 34.1  98.2 / 57.1  101.7 / 79.1  104 / 82  27.2 / 19.8
//   7168 x 2048           -       13.5 / 7.7   20.0 / 13.7  20.2 / 19.6   24.0 / 30.9  26.2 / 31.5  7.2 / 7.7
//   2048 x 4096           -       10.0 / 6.4   11.0 / 9.2   14.0 / 12.7   15.4 / 16.3  16.8 / 18.5  5.9 / 6.5
//   1024 x 4096           -        6.8 / 5.0    7.1 / 6.7    7.8 / 7.8     9.5 / 10.8   9.7 / 11.1  4.7 / 5.1
//   7168 x 512            -        5.5 / 6.1    5.9 / 6.3    6.7 / 7.1     8.3 / 10.0   8.8 / 10.8  4.7 / 6.1
static i8_launch few_rows(const i8_mm &a) {
  if (a.N > 1 << 22) return nullptr;
  if (a.offsets) {
    const bool again = a.M >= 2 * a.E && (a.M > 4 * a.E || (size_t)a.N * a.K > (size_t)4 << 20);
    return a.M > 16 || again ? nullptr : a.K <= 1024 ? launch_few<1, 8, 1> : launch_few<1, 4, 2>;
  }
  const long n = (long)a.M * a.N;
  if (a.M == 1 || n <= 4096) return launch_few<1, 2, 4>;
  if (a.M == 2 || n <= 8192) return launch_few<2, 4, 2>;
  if (a.M <= 4 && (size_t)a.N * a.K <= (size_t)32 << 20) return launch_few<4, 2, 2>;
  return nullptr;
}

template <int BM, int BN, int WM, int WN, int WK, int NBUF>
static bool launch_tiles(const i8_mm &a, hipStream_t st) {
  const int nt = ceil_div(a.N, BN);
  const long n = i8_tiles(a, BM) * nt;
  if (!fits(n, 64 * WM * WN * WK)) return false;
  hipLaunchKernelGGL((a.stream ? k_mm_i8<BM, BN, WM, WN, WK, NBUF, true> : k_mm_i8<BM, BN, WM, WN, WK, NBUF, false>),
                     dim3((unsigned)n), dim3(64 * WM * WN * WK), (i8_lds_bytes<BM, BN, WM, WN, WK, NBUF>()), st, a, nt);
  return true;
}

// The tile shapes, and what they cost.  A call of `rounds` tiles one after the other
// on a CU takes about
//   call + rounds * (tile + K / 128 * (k + k_share * tiles that share the CU))  us,
// fitted to 83 dense products of 1 to 8192 rows, K and N from 640 to 7168, on each of
// 25 shapes, before the present order of LDS reads: then the shape of the least cost was on average 0.6% slower
// than the fastest of the 25 (at most 12%), and 2.8% (24%) over 72 grouped calls of 4 to
// 32764 rows, where the rows of each expert are not known here.  It serves to choose, not to predict: with
// weights from HBM a call takes 10 to 35% more than it says (256x256 less).  The present kernels, weights from
// HBM, the chosen one marked (its bracket: the weights of the call before, from the cache):
//   rows x 7168 x 7168, us:  16x16  32x32  64x32  64x64  128x64  64x128  128x128  128x256  256x128  256x256
//                      16:   13.5*   12.8   13.6   18.0    20.8    28.9     30.3     43.9     41.8     75.0  (10.8)
//                      64:    33.4   22.2   16.6*  21.7    22.3    31.7     32.8     50.1     43.7     78.9  (12.4)
//                     256:     118   69.1   46.1   34.6    26.3*   31.0     36.4     53.8     53.1     95.1  (20.3)
//                     512:     231    132   77.7   59.4    45.3    41.3     36.4*    52.8     52.1     89.6  (29.1)
//                    1024:     457    258    149    102    84.6    79.2     59.6     55.4*    55.0     87.6  (50.8)
//                    4096:    1803   1009    580    386     299     271      212      207      201      173* (164)
// A last round that is partly filled costs less than
// a whole one, once there are several: its tiles have the memory to themselves.
// 128x128 stands twice (the table: the faster one): 3 stages for one workgroup a CU, 2 for two.  Eight waves a
// workgroup in all but the smallest: with 4 the same tiles took up to a third longer.
struct i8_shape {
  int BM, BN, threads, lds;
  float call, tile, k, k_share;
  i8_launch launch;
};
template <int BM, int BN, int WM, int WN, int WK, int NBUF>
static constexpr i8_shape shape_of(float call, float tile, float k, float k_share) {
  return {BM, BN, 64 * WM * WN * WK, i8_lds_bytes<BM, BN, WM, WN, WK, NBUF>(), call, tile, k, k_share, launch_tiles<BM, BN, WM, WN, WK, NBUF>};
}
static const i8_shape i8_shapes[] = {
    shape_of<16, 16, 1, 1, 4, 4>(2.11f, 1.81f, 0.031f, 0.039f),
    shape_of<32, 32, 2, 1, 4, 4>(1.81f, 2.36f, 0.112f, 0.0f),
    shape_of<64, 32, 4, 1, 2, 4>(1.68f, 2.27f, 0.165f, 0.0f),
    shape_of<64, 64, 2, 2, 2, 3>(1.30f, 2.77f, 0.225f, 0.0f),
    shape_of<128, 64, 4, 2, 1, 4>(1.27f, 2.80f, 0.350f, 0.0f),
    shape_of<64, 128, 2, 4, 1, 3>(1.57f, 2.41f, 0.134f, 0.253f),
    shape_of<128, 128, 4, 2, 1, 3>(0.0f, 4.09f, 0.504f, 0.0f),
    shape_of<128, 128, 2, 4, 1, 2>(0.0f, 2.95f, 0.509f, 0.264f),
    shape_of<128, 256, 2, 4, 1, 3>(0.0f, 5.55f, 0.775f, 0.0f),
    shape_of<256, 128, 4, 2, 1, 3>(0.0f, 5.59f, 0.779f, 0.0f),
    shape_of<256, 256, 2, 4, 1, 2>(0.0f, 5.95f, 1.544f, 0.0f),
};

// The launch of the least cost, of the shapes whose tiles a grid takes (NULL: none; the largest
// take every product whose output fits the memory).
static i8_launch choose_shape(const i8_mm &a, int n_cu) {
  const i8_shape *best = nullptr;
  float least = 0.0f;
  // experts: as many as can have rows, of the same number each
  const float matrices = a.offsets ? (float)(a.M < a.E ? a.M : a.E) : 1.0f, rows = a.M / matrices;
  for (const i8_shape &s : i8_shapes) {
    if (!fits(i8_tiles(a, s.BM) * ceil_div(a.N, s.BN), s.threads)) continue;
    const float row_tiles = !a.offsets ? (float)ceil_div(a.M, s.BM) : rows <= s.BM ? 1.0f : rows / s.BM + 0.5f;
    const float tiles = matrices * row_tiles * (float)ceil_div(a.N, s.BN);
    const int fit = (160 << 10) / s.lds, occ = fit < 4 ? fit : 4;
    const float each = tiles / (float)(n_cu * occ), per_cu = ceilf(tiles / (float)n_cu);
    const float rounds = each <= 3.0f ? ceilf(each) : fminf(ceilf(each), each + 0.5f);
    const float cost = s.call + rounds * (s.tile + a.K / 128.0f * (s.k + s.k_share * (per_cu < occ ? per_cu : occ)));
    if (!best || cost < least) {
      best = &s;
      least = cost;
    }
  }
  return best ? best->launch : nullptr;
}

static constexpr long MOE_GRID_Y = 65535;  // most blocks along a grid's y and z dimensions

bool launch_matmul_i8(const i8_mm &args, int n_cu, hipStream_t st) {
  i8_mm a = args;
  // the tiles: 16-byte loads at 32-bit offsets (a smaller row count is a uniform matter of the operands)
  const bool aligned = a.K % 16 == 0 && ((uintptr_t)a.q | (uintptr_t)a.w) % 16 == 0;
  const bool offsets32 = (uint64_t)a.n_src * a.K < MOE_I8_OOB && (uint64_t)a.N * a.K < MOE_I8_OOB;
  if (aligned && offsets32) {
    // weights of more than the caches hold from call to call, each read by one tile: past the caches.  Measured:
    // 939 MB against 16 rows 164 us with plain loads, 146 without (5.75 and 6.5 TB/s)
    a.stream = (size_t)a.N * a.K * (a.M < a.E ? a.M : a.E) > MOE_STREAM_BYTES;
    const i8_launch few = few_rows(a), launch = few ? few : choose_shape(a, n_cu);
    return launch && launch(a, st);
  }
  const int nt = a.swiglu ? ceil_div(a.N / 2, 32) : ceil_div(a.N, 64);
  if (!fits(nt, 256)) return false;
  // tiles of rows along y, and along z as often as they do not fit there
  const long mt = i8_tiles(a, 64), y = mt < MOE_GRID_Y ? mt : MOE_GRID_Y;
  hipLaunchKernelGGL(k_mm_i8_any, dim3(nt, (unsigned)y, (unsigned)ceil_div(mt, y)), dim3(256), 0, st, a);
  return true;
}
