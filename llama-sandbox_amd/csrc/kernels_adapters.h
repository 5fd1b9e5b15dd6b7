// kernels_adapters.h -- low-rank adapters of many requests beside a shared projection.
//
//   mid[i] = A[a] x[perm[i]],  out[perm[i]] = base[perm[i]] + scale[a] * B[a] mid[i]
// for the grouped rows i of adapter a, [offsets[a], offsets[a+1]).  mid is f32.
//
// Two launches on 16x16 MFMA tiles of an adapter's rows.  Lane l of an operand holds row l % 16 and V
// consecutive elements of K from V (l / 16) on (V = 8 of 16 bits, 4 of f32); of the result column l % 16 and
// rows 4 (l / 16) + i.  Tokens are the columns, so that a lane's four values are next to each other in mid,
// and, with the weight rows dealt to two tiles four and four, its eight in out (the last kernel: the other way round).
#pragma once

#include "group_tiles.h"
#include "layer_kernels.h"
#include "lds_dma.h"
#include "row_vec.h"
#include "../../include/moe_block.h"

#include <type_traits>

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// 16 bytes of a row, V elements, at the type's own alignment.
template <typename T>
struct frag {
  static constexpr int V = 16 / sizeof(T), STEP = 4 * V;  // elements of K that a wave's 64 lanes hold of 16 rows
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  vec v;
  __device__ __forceinline__ void load(const T *p) { v = *reinterpret_cast<const vec *>(p); }
  // 0 from `left` on; whole: the same for a wave, pieces are there as a whole or not at all
  __device__ __forceinline__ void load(const T *p, int left, bool whole) {
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = (T)0.0f;
    if (left >= V) {
      load(p);
    } else if (!whole) {
#pragma unroll
      for (int i = 0; i < V; i++)
        if (i < left) v[i] = p[i];
    }
  }
};

__device__ __forceinline__ f32x4_t mfma16(const frag<bf16_t> &a, const frag<bf16_t> &b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16((bf16x8_t)a.v, (bf16x8_t)b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma16(const frag<_Float16> &a, const frag<_Float16> &b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16((f16x8_t)a.v, (f16x8_t)b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma16(const frag<float> &a, const frag<float> &b, f32x4_t c) {
#pragma unroll
  for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
  return c;
}

// 8 values of out; nt: past the caches, the same for a whole call.
template <typename TO>
__device__ __forceinline__ void store_out(const adapters_call &a, int row, int n, const float (&f)[8]) {
  TO *to = reinterpret_cast<TO *>(a.out) + (size_t)row * a.N + n;
  if (a.nt) store_v<TO, 8, true>(to, a.N - n, f);
  else store_v<TO, 8>(to, a.N - n, f);
}

// The row of x, base and out that grouped row i is; -1: none.
__device__ __forceinline__ int adapters_row(const adapters_call &a, const row_tile &t, int i) {
  const int row = i < t.n ? a.perm[t.r0 + i] : -1;
  return row < a.M ? row : -1;
}

// mid, as a.splits shares of it, [split][grouped row][R].  grid (tiles * splits, ceil(R / (16 RT))): a workgroup has the share
// of one piece of K of 16 MT grouped rows and 16 RT rows of A; its waves take pieces of U steps in turn and meet in LDS.
// Absent rows read another's (their columns are not written).
// 16 single tokens of 16 adapters of 7168 x 16 (3.7 MB): 4.2 us, the chain of offsets, perm, x; 4096 rows of 7168 x
// 16 14.0, x 64 25.  Bound there by the address unit, which takes a lane a cycle for loads whose neighbours are other
// rows; neither deeper rings nor another order of the loads moved it.
template <typename T, int MT, int RT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_adapters_shrink(adapters_call a) {
  typedef frag<T> F;
  constexpr int U = MT + RT > 4 ? 2 : 4;  // steps in flight, next to each other in memory
  __shared__ f32x4_t part[WAVES][MT * RT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, split = blockIdx.x % a.splits;
  const row_tile t = find_row_tile(a.offsets, a.n, a.M, blockIdx.x / a.splits, 16 * MT);
  if (t.e < 0) return;
  const int r0 = blockIdx.y * 16 * RT, k0 = lane / 16 * F::V;
  const T *x[MT], *w[RT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    const int row = adapters_row(a, t, m * 16 + lane % 16);
    x[m] = reinterpret_cast<const T *>(a.x) + (size_t)(row < 0 ? 0 : row) * a.K + k0;
  }
#pragma unroll
  for (int r = 0; r < RT; r++)
    w[r] = reinterpret_cast<const T *>(a.a) + ((size_t)t.e * a.R + min(r0 + r * 16 + lane % 16, a.R - 1)) * a.K + k0;
  f32x4_t acc[MT][RT] = {};
  const int end = min(a.K, (split + 1) * a.piece);
  for (int k = split * a.piece + wave * U * F::STEP; k < end; k += WAVES * U * F::STEP) {
    F fx[U][MT], fw[U][RT];
    // a row's steps one after the other: two share a cache line, and rows of many lengths share sets of the cache
    if (k + U * F::STEP <= end) {
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int u = 0; u < U; u++) fx[u][m].load(x[m] + k + u * F::STEP);
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int u = 0; u < U; u++) fw[u][r].load(w[r] + k + u * F::STEP);
    } else {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int left = end - k - u * F::STEP - k0;
#pragma unroll
        for (int m = 0; m < MT; m++) fx[u][m].load(x[m] + k + u * F::STEP, left, a.K % F::V == 0);
#pragma unroll
        for (int r = 0; r < RT; r++) fw[u][r].load(w[r] + k + u * F::STEP, left, a.K % F::V == 0);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int r = 0; r < RT; r++) acc[m][r] = mfma16(fw[u][r], fx[u][m], acc[m][r]);
  }
#pragma unroll
  for (int m = 0; m < MT; m++)
#pragma unroll
    for (int r = 0; r < RT; r++) part[wave][m * RT + r][lane] = acc[m][r];
  __syncthreads();
  for (int q = wave; q < MT * RT; q += WAVES) {
    f32x4_t sum = part[0][q][lane];
#pragma unroll
    for (int v = 1; v < WAVES; v++) sum += part[v][q][lane];
    const int i = q / RT * 16 + lane % 16, at = r0 + q % RT * 16 + lane / 16 * 4;
    const float f[4] = {sum[0], sum[1], sum[2], sum[3]};
    if (i < t.n && at < a.R) store_v<float, 4>(a.mid + ((size_t)split * a.M + t.r0 + i) * a.R + at, a.R - at, f);
  }
}

// The same for adapters of many rows: 64 of them a workgroup, 16 a wave.  Loads that give neighbouring lanes
// other rows take a cycle a lane (above: 59 accesses a load); here rows come as runs of 128 bytes, straight to LDS,
// NBUF - 1 stages ahead, and are read from there as operands (chunk c of row r lies at c ^ (r & 7)).  Rows and A of
// whole 16 bytes, below 4 GiB.  4096 rows of 7168 x 64 bf16 (59 MB of x, 62 of A from L2) 22.7 us; more pieces of K
// (3 to 8) move time from here to the reading of the shares, another start in K for each tile does nothing.
template <typename T, int NBUF>
__global__ __launch_bounds__(256) void k_adapters_shrink_staged(adapters_call a) {
  typedef frag<T> F;
  typedef uint32_t chunk_t __attribute__((ext_vector_type(4)));
  constexpr int RT = 4, STAGE = (64 + 64) * 8;  // tiles of A's rows; chunks of a stage
  constexpr int CX = 2, CW = 2;                 // 1 KiB loads a wave: of x, of A
  extern __shared__ __align__(16) uint32_t adapters_lds[];  // NBUF * STAGE chunks
  chunk_t *lds = reinterpret_cast<chunk_t *>(adapters_lds);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), split = blockIdx.x % a.splits;
  const row_tile t = find_row_tile(a.offsets, a.n, a.M, blockIdx.x / a.splits, 64);
  if (t.e < 0) return;
  const int r0 = blockIdx.y * 64, rows_a = min(64, a.R - r0);
  const uint32_t row_bytes = (uint32_t)a.K * sizeof(T), xbytes = (uint32_t)a.M * row_bytes, wbytes = (uint32_t)rows_a * row_bytes;
  const T *w = reinterpret_cast<const T *>(a.a) + ((size_t)t.e * a.R + r0) * a.K;
  const uint32_t begin = (uint32_t)(split * a.piece) * sizeof(T);
  const uint32_t end = min(row_bytes, begin + (uint32_t)a.piece * (uint32_t)sizeof(T));
  const int stages = begin < end ? (int)((end - begin + 127) / 128) : 0;
  const int lr = lane >> 3, lc = ((lane & 7) ^ lr) * 16;
  uint32_t vx[CX], vw[CW];
#pragma unroll
  for (int i = 0; i < CW; i++) {
    const int row = 8 * (wave + 4 * i) + lr;
    vw[i] = row < rows_a ? (uint32_t)row * row_bytes + lc : MOE_LDS_OOB;
  }
  // stage s of this wave's loads into its buffer; past the end they read 0, so that the waits can count on them
  auto load_w = [&](int s) __attribute__((always_inline)) {
    const uint32_t at = begin + s * 128;
    const bool there = s < stages && at + lc < end;
#pragma unroll
    for (int i = 0; i < CW; i++)
      lds_dma(w, wbytes, lds + s % NBUF * STAGE + (64 / 8 + wave + 4 * i) * 64, there ? vw[i] : MOE_LDS_OOB, s < stages ? at : 0);
  };
  auto load_x = [&](int s) __attribute__((always_inline)) {
    const uint32_t at = begin + s * 128;
    const bool there = s < stages && at + lc < end;
#pragma unroll
    for (int i = 0; i < CX; i++)
      lds_dma(a.x, xbytes, lds + s % NBUF * STAGE + (wave + 4 * i) * 64, there ? vx[i] : MOE_LDS_OOB, s < stages ? at : 0);
  };
  // A goes out before the rows are known
#pragma unroll
  for (int s = 0; s < NBUF - 1; s++) load_w(s);
#pragma unroll
  for (int i = 0; i < CX; i++) {
    const int row = adapters_row(a, t, 8 * (wave + 4 * i) + lr);
    vx[i] = row >= 0 ? (uint32_t)row * row_bytes + lc : MOE_LDS_OOB;
  }
#pragma unroll
  for (int s = 0; s < NBUF - 1; s++) load_x(s);
  f32x4_t acc[RT] = {};
  const int fr = lane & 15, fg = lane >> 4;
  for (int s = 0; s < stages; s++) {
    // this stage has landed, and every wave is done with the one before, whose buffer the next loads take
    if (s < NBUF - 2) lds_wait_barrier<(NBUF - 2) * CX>();
    else lds_wait_barrier<(NBUF - 2) * (CX + CW)>();
    load_w(s + NBUF - 1);
    load_x(s + NBUF - 1);
    const chunk_t *x = lds + s % NBUF * STAGE + (wave * 16 + fr) * 8, *wl = lds + s % NBUF * STAGE + (64 + fr) * 8;
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int c = (k * 4 + fg) ^ (fr & 7);
      const F fx = {__builtin_bit_cast(typename F::vec, x[c])};
#pragma unroll
      for (int r = 0; r < RT; r++) acc[r] = mfma16(F{__builtin_bit_cast(typename F::vec, wl[r * 128 + c])}, fx, acc[r]);
    }
  }
  lds_wait_barrier<0>();  // what is on its way has landed
  const int i = wave * 16 + fr;
  if (i >= t.n) return;
  float *to = a.mid + ((size_t)split * a.M + t.r0 + i) * a.R;
#pragma unroll
  for (int r = 0; r < RT; r++) {
    const int at = r0 + r * 16 + fg * 4;
    const float f[4] = {acc[r][0], acc[r][1], acc[r][2], acc[r][3]};
    if (at < a.R) store_v<float, 4>(to + at, a.R - at, f);
  }
}

// mid as the operands that multiply a piece of B: f32 as it is; else as three bf16 parts, each the leading 8 bits of what
// the ones before leave, so that together they are its 24 bits.  (Two would do for an output of 16 bits, but not where
// base and update, or the products of B, cancel; 4096 rows x 64 x 7168 bf16 36.6 us with two, 37.5 with three.)  The
// parts are cut, not rounded: a value next to the largest stays finite.
// A piece of f16 weights is two bf16 pieces, which hold it exactly, at bf16's range: mid may be past f16's.
template <typename T>
struct expand_of {
  typedef bf16_t type;
};
template <>
struct expand_of<float> {
  typedef float type;
};

__device__ __forceinline__ void weight_parts(const frag<float> &w, frag<float> (&p)[1]) { p[0] = w; }
__device__ __forceinline__ void weight_parts(const frag<bf16_t> &w, frag<bf16_t> (&p)[1]) { p[0] = w; }
__device__ __forceinline__ void weight_parts(const frag<_Float16> &w, frag<bf16_t> (&p)[2]) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float f = (float)w.v[i], hi = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, f) & 0xffff0000u);
    p[0].v[i] = (bf16_t)hi;
    p[1].v[i] = (bf16_t)(f - hi);
  }
}

template <typename T>
constexpr int mid_parts() { return sizeof(T) == 4 ? 1 : 3; }

template <typename TE, int N>
using vec_of_n = TE __attribute__((ext_vector_type(N)));

template <int N>
__device__ __forceinline__ void cut_mid(float (&f)[N], vec_of_n<float, N> (&o)[1]) {
#pragma unroll
  for (int j = 0; j < N; j++) o[0][j] = f[j];
}
template <int N>
__device__ __forceinline__ void cut_mid(float (&f)[N], vec_of_n<bf16_t, N> (&o)[3]) {
#pragma unroll
  for (int p = 0; p < 3; p++) {
    vec_of_n<uint16_t, N> top;
#pragma unroll
    for (int j = 0; j < N; j++) {
      const uint32_t u = __builtin_bit_cast(uint32_t, f[j]);
      top[j] = (uint16_t)(u >> 16);
      f[j] -= __builtin_bit_cast(float, u & 0xffff0000u);
    }
    o[p] = __builtin_bit_cast(vec_of_n<bf16_t, N>, top);
  }
}

// mid of ROWS grouped rows of a tile from rc on, its shares added up, in LDS as parts of TE: 64 of R.  256 threads.
template <typename TE, int PARTS, int ROWS, int ROW>
__device__ __forceinline__ void stage_mid(const adapters_call &a, const row_tile &t, int rc, TE (&mid)[PARTS][ROWS][ROW]) {
  // pieces of 4 a thread, and shares of each in flight
  constexpr int RC = 64, PIECES = ROWS * RC / 4 / 256, SHARES = PIECES == 1 ? 4 : 2;
  const size_t share = (size_t)a.M * a.R;
  float f[PIECES][4] = {};
#pragma unroll 1
  for (int s = 0; s < a.splits; s += SHARES) {
    frag<float> g[PIECES][SHARES];
#pragma unroll
    for (int q = 0; q < PIECES; q++) {
      const int i = threadIdx.x + q * 256, m = i / (RC / 4), r = rc + i % (RC / 4) * 4;
      const float *from = a.mid + ((size_t)s * a.M + t.r0 + m) * a.R + r;
#pragma unroll
      for (int v = 0; v < SHARES; v++)
        g[q][v].load(from + v * share, s + v < a.splits && m < t.n ? a.R - r : 0, a.R % 4 == 0);
    }
#pragma unroll
    for (int q = 0; q < PIECES; q++)
#pragma unroll
      for (int v = 0; v < SHARES; v++)
#pragma unroll
        for (int j = 0; j < 4; j++) f[q][j] += g[q][v].v[j];
  }
#pragma unroll
  for (int q = 0; q < PIECES; q++) {
    const int i = threadIdx.x + q * 256;
    vec_of_n<TE, 4> o[PARTS];
    cut_mid(f[q], o);
#pragma unroll
    for (int p = 0; p < PARTS; p++) *reinterpret_cast<vec_of_n<TE, 4> *>(&mid[p][i / (RC / 4)][i % (RC / 4) * 4]) = o[p];
  }
}

// out.  grid (tiles * column blocks): 16 MT grouped rows by a.col_groups times 128 columns of out a workgroup, 32 a wave,
// with the next group's loads in flight; mid's shares are added up and cut into parts in LDS, 64 of R at a time.
// Four workgroups a CU (at most 128 registers) or the chains of loads show: with 208 registers half as slow again.  16
// single tokens x 16 x 4096 4.8 us; 4096 rows x 16 x 7168, which the staged kernel takes, 43.
template <typename T, typename TO, int MT>
__global__ __launch_bounds__(256, 4) void k_adapters_expand(adapters_call a) {
  typedef typename expand_of<T>::type TE;
  typedef frag<TE> F;
  constexpr int RC = 64, STEPS = RC / F::STEP, PARTS = mid_parts<T>();
  constexpr int WP = sizeof(T) == 2 && !std::is_same<T, TE>::value ? 2 : 1;
  constexpr int ROW = RC + F::V;  // a piece more, so that rows lie in different banks
  __shared__ __attribute__((aligned(16))) TE mid[PARTS][16 * MT][ROW];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane % 16, kg = lane / 16;
  const row_tile t = find_row_tile(a.offsets, a.n, a.M, blockIdx.x / a.col_blocks, 16 * MT);
  if (t.e < 0) return;
  const T *b = reinterpret_cast<const T *>(a.b) + (size_t)t.e * a.N * a.R;
  int row[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) row[m] = adapters_row(a, t, m * 16 + col);

  const int first = (blockIdx.x % a.col_blocks * a.col_groups) * 128 + wave * 32;
  // a lane's 8 columns n0 + 8 kg + .. of rows m * 16 + col; absent rows read the first
  raw_v<TO, 8> base[MT];
  auto load_base = [&](int n0) {
    const int n = n0 + kg * 8;
#pragma unroll
    for (int m = 0; m < MT; m++) {
      const TO *p = reinterpret_cast<const TO *>(a.base) + (size_t)(row[m] < 0 ? 0 : row[m]) * a.N + n;
      if (n0 + 32 <= a.N) base[m].v = *reinterpret_cast<const typename raw_v<TO, 8>::vec_t *>(p);
      else base[m].load(p, a.N - n);
    }
  };
  // the pieces of B of one step: 32 rows, dealt to the two tiles four and four
  frag<T> w[2];
  auto load_b = [&](int n0, int r) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const T *p = b + (size_t)min(n0 + col / 4 * 8 + j * 4 + col % 4, a.N - 1) * a.R + r + kg * F::V;
      if (r + F::STEP <= a.R) w[j].load(p);
      else w[j].load(p, a.R - r - kg * F::V, a.R % F::V == 0);
    }
  };
  load_b(first, 0);
  load_base(first);
  const float scale = a.scale ? a.scale[t.e] : 1.0f;
  for (int g = 0; g < a.col_groups; g++) {
    const int n0 = first + g * 128;
    f32x4_t acc[MT][2] = {};
    for (int rc = 0; rc < a.R; rc += RC) {
      if (g == 0 || a.R > RC) {
        if (g || rc) __syncthreads();
        stage_mid<TE, PARTS, 16 * MT, ROW>(a, t, rc, mid);
        __syncthreads();
      }
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        const int r = rc + s * F::STEP, next = r + F::STEP;
        if (r >= a.R) break;
        F fm[MT][PARTS], wp[2][WP];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int p = 0; p < PARTS; p++)
            fm[m][p].v = *reinterpret_cast<const typename F::vec *>(&mid[p][m * 16 + col][s * F::STEP + kg * F::V]);
#pragma unroll
        for (int j = 0; j < 2; j++) weight_parts(w[j], wp[j]);
        if (next < a.R) load_b(n0, next);
        else if (g + 1 < a.col_groups) load_b(n0 + 128, 0);
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int m = 0; m < MT; m++)
#pragma unroll
            for (int p = 0; p < PARTS; p++)
#pragma unroll
              for (int q = 0; q < WP; q++) acc[m][j] = mfma16(wp[j][q], fm[m][p], acc[m][j]);
      }
    }
    const int n = n0 + kg * 8;
    float out[MT][8];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int i = 0; i < 8; i++) out[m][i] = fmaf(scale, acc[m][i / 4][i % 4], (float)base[m].v[i]);
    if (g + 1 < a.col_groups) load_base(n0 + 128);
#pragma unroll
    for (int m = 0; m < MT; m++)
      if (row[m] >= 0 && n < a.N) store_out<TO>(a, row[m], n, out[m]);
  }
}

// out for adapters of many rows and R <= 64: 64 grouped rows, 16 a wave, by 256 columns a workgroup.  B's rows come to LDS
// as runs, all at once, and tokens are the rows of the result: tile j of a group of 128 columns has the columns
// 8 l + j, so that a lane holds 8 next to each other and 16 lanes a run of 128 columns of base and out.
// LDS row 16 j + l of a group is row 8 l + j of B.  B's rows are whole 16 bytes, an adapter's below 4 GiB.  4096 rows of
// 64 x 7168 bf16 (117 MB of base and out) 37.5 us, x 16 30.7: workgroups of one phase after another (offsets; B, mid, base;
// the products; out), three a CU.
template <typename T, typename TO>
__global__ __launch_bounds__(256) void k_adapters_expand_staged(adapters_call a) {
  typedef typename expand_of<T>::type TE;
  typedef frag<TE> F;
  typedef uint32_t chunk_t __attribute__((ext_vector_type(4)));
  constexpr int RC = 64, STEPS = RC / F::STEP, PARTS = mid_parts<T>();
  constexpr int WP = sizeof(T) == 2 && !std::is_same<T, TE>::value ? 2 : 1;
  constexpr int ROW = RC + 4;                        // a piece more, so that rows lie in different banks
  constexpr int BLOCKS = RC * (int)sizeof(T) / 128;  // of 128 bytes of B's rows
  __shared__ chunk_t lds[BLOCKS * 256 * 8];
  __shared__ __attribute__((aligned(16))) float mid[1][64][ROW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fg = lane >> 4;
  const row_tile t = find_row_tile(a.offsets, a.n, a.M, blockIdx.x / a.col_blocks, 64);
  if (t.e < 0) return;
  const int first = blockIdx.x % a.col_blocks * 256;
  const uint32_t row_bytes = (uint32_t)a.R * sizeof(T), bbytes = (uint32_t)a.N * row_bytes;
  const T *b = reinterpret_cast<const T *>(a.b) + (size_t)t.e * a.N * a.R;
  const int lr = lane >> 3, lc = ((lane & 7) ^ lr) * 16;
#pragma unroll
  for (int k = 0; k < BLOCKS; k++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int row = 8 * (wave + 4 * i) + lr, n = first + row / 128 * 128 + row % 16 * 8 + row % 128 / 16;
      const uint32_t at = k * 128 + lc;
      lds_dma(b, bbytes, lds + (k * 32 + wave + 4 * i) * 64, n < a.N && at < row_bytes ? (uint32_t)n * row_bytes + at : MOE_LDS_OOB, 0);
    }
  int row[4];
#pragma unroll
  for (int i = 0; i < 4; i++) row[i] = adapters_row(a, t, wave * 16 + fg * 4 + i);
  raw_v<TO, 8> base[2][4];
#pragma unroll
  for (int g = 0; g < 2; g++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int n = first + g * 128 + fr * 8;
      base[g][i].load(reinterpret_cast<const TO *>(a.base) + (size_t)(row[i] < 0 ? 0 : row[i]) * a.N + n, row[i] < 0 ? 0 : a.N - n);
    }
  const float scale = a.scale ? a.scale[t.e] : 1.0f;
  stage_mid<float, 1, 64, ROW>(a, t, 0, mid);
  lds_wait_barrier<0>();
  // (as f32 in LDS, cut here: a row's parts are one wave's, and three of them in LDS would leave two workgroups a CU)
  F fm[STEPS][PARTS];
#pragma unroll
  for (int s = 0; s < STEPS; s++) {
    float f[F::V];
#pragma unroll
    for (int j = 0; j < F::V; j++) f[j] = mid[0][wave * 16 + fr][s * F::STEP + fg * F::V + j];
    vec_of_n<TE, F::V> o[PARTS];
    cut_mid(f, o);
#pragma unroll
    for (int p = 0; p < PARTS; p++) fm[s][p].v = o[p];
  }
#pragma unroll
  for (int g = 0; g < 2; g++) {
    const int n = first + g * 128 + fr * 8;
    if (first + g * 128 >= a.N) break;
    f32x4_t acc[8] = {};
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        if (s * F::STEP >= a.R) break;
        const int c = s * 4 + fg;  // chunk of the row
        const frag<T> w = {__builtin_bit_cast(typename frag<T>::vec, lds[((c / 8 * 256) + g * 128 + j * 16 + fr) * 8 + ((c & 7) ^ (fr & 7))])};
        F wp[WP];
        weight_parts(w, wp);
#pragma unroll
        for (int p = 0; p < PARTS; p++)
#pragma unroll
          for (int q = 0; q < WP; q++) acc[j] = mfma16(fm[s][p], wp[q], acc[j]);
      }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; j++) f[j] = fmaf(scale, acc[j][i], (float)base[g][i].v[j]);
      if (row[i] >= 0 && n < a.N) store_out<TO>(a, row[i], n, f);
    }
  }
}
