// kernels_adapters.h -- low-rank adapters of many requests beside a shared projection.
//
//   mid[i] = A[a] x[perm[i]],  out[perm[i]] = base[perm[i]] + scale[a] * B[a] mid[i]
// for the grouped rows i of adapter a, [offsets[a], offsets[a+1]).  mid is f32.
//
// Two launches on 16x16 MFMA tiles of an adapter's rows.  Lane l of an operand holds row l % 16 and V
// consecutive elements of K from V (l / 16) on (V = 8 of 16 bits, 4 of f32); of the result column l % 16 and
// rows 4 (l / 16) + i.  Tokens are the columns in both, so that a lane's four values are next to each other in mid,
// and, with the weight rows dealt to two tiles four and four, its eight in out.
#pragma once

#include "group_tiles.h"
#include "layer_kernels.h"
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

// The row of x, base and out that grouped row i is; -1: none.
__device__ __forceinline__ int adapters_row(const adapters_call &a, const row_tile &t, int i) {
  const int row = i < t.n ? a.perm[t.r0 + i] : -1;
  return row < a.M ? row : -1;
}

// mid, as a.splits shares of it, [split][grouped row][R].  grid (tiles * splits, ceil(R / (16 RT))): a workgroup has the share
// of one piece of K of 16 MT grouped rows and 16 RT rows of A; its waves take pieces of U steps in turn and meet in LDS.
// Absent rows read another's (their columns are not written).
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

// A 16-byte piece of mid as the operands that multiply a piece of B: f32 as it is; else as PARTS bf16 parts, each what
// the ones before leave (2: 2^-16 of it is lost, where the output is rounded to 2^-8 of its; 3: 2^-24).
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

// out.  grid (tiles * column blocks): 16 MT grouped rows by a.col_groups times 128 columns of out a workgroup, 32 a wave,
// with the next group's loads in flight; mid's shares are added up and cut into parts in LDS, 64 of R at a time.
template <typename T, typename TO, int MT, int PARTS>
__global__ __launch_bounds__(256, 4) void k_adapters_expand(adapters_call a) {
  typedef typename expand_of<T>::type TE;
  typedef frag<TE> F;
  constexpr int RC = 64, STEPS = RC / F::STEP, WP = sizeof(T) == 2 && !std::is_same<T, TE>::value ? 2 : 1;
  constexpr int ROW = RC + F::V;  // a piece more, so that rows lie in different banks
  __shared__ __attribute__((aligned(16))) TE mid[PARTS][16 * MT][ROW];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane % 16, kg = lane / 16;
  const row_tile t = find_row_tile(a.offsets, a.n, a.M, blockIdx.x / a.col_blocks, 16 * MT);
  if (t.e < 0) return;
  const T *b = reinterpret_cast<const T *>(a.b) + (size_t)t.e * a.N * a.R;
  int row[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) row[m] = adapters_row(a, t, m * 16 + col);

  auto stage = [&](int rc) {
#pragma unroll 1
    for (int i = threadIdx.x; i < 16 * MT * RC / 4; i += 256) {
      const int m = i / (RC / 4), r = rc + i % (RC / 4) * 4;
      const float *from = a.mid + ((size_t)t.r0 + m) * a.R + r;
      const size_t share = (size_t)a.M * a.R;
      const int left = m < t.n ? a.R - r : 0;
      float f[4] = {};
      for (int s = 0; s < a.splits; s += 4, from += 4 * share) {
        frag<float> g[4];
#pragma unroll
        for (int v = 0; v < 4; v++) g[v].load(from + v * share, s + v < a.splits ? left : 0, a.R % 4 == 0);
#pragma unroll
        for (int v = 0; v < 4; v++)
#pragma unroll
          for (int j = 0; j < 4; j++) f[j] += g[v].v[j];
      }
      typedef TE vec4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int p = 0; p < PARTS; p++) {
        vec4 o;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          o[j] = (TE)f[j];
          f[j] -= (float)o[j];
        }
        *reinterpret_cast<vec4 *>(&mid[p][m][i % (RC / 4) * 4]) = o;
      }
    }
  };

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
        stage(rc);
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
      if (row[m] >= 0 && n < a.N) store_v<TO, 8>(reinterpret_cast<TO *>(a.out) + (size_t)row[m] * a.N + n, a.N - n, out[m]);
  }
}
