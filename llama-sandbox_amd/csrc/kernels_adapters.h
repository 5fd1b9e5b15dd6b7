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
  __device__ __forceinline__ void load(const T *p, int left) {  // 0 from `left` on
    if (left >= V) {
      load(p);
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) v[i] = i < left ? p[i] : (T)0.0f;
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
// of one piece of K of 16 MT grouped rows and 16 RT rows of A; its 4 waves take every fourth step of K and meet in LDS.
// Absent rows read another's (their columns are not written).
template <typename T, int MT, int RT>
__global__ __launch_bounds__(256) void k_adapters_shrink(adapters_call a) {
  typedef frag<T> F;
  constexpr int U = MT + RT > 4 ? 2 : 4;  // steps in flight
  __shared__ f32x4_t part[3][MT * RT][64];
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
  const int begin = split * a.piece + wave * F::STEP, end = min(a.K, (split + 1) * a.piece);
  int k = begin;
  // whole steps, U at once
  for (; k + ((U - 1) * 4 + 1) * F::STEP <= end; k += U * 4 * F::STEP) {
    F fx[U][MT], fw[U][RT];
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
      for (int m = 0; m < MT; m++) fx[u][m].load(x[m] + k + u * 4 * F::STEP);
#pragma unroll
      for (int r = 0; r < RT; r++) fw[u][r].load(w[r] + k + u * 4 * F::STEP);
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int r = 0; r < RT; r++) acc[m][r] = mfma16(fw[u][r], fx[u][m], acc[m][r]);
  }
  for (; k < end; k += 4 * F::STEP) {
    F fx[MT], fw[RT];
#pragma unroll
    for (int m = 0; m < MT; m++) fx[m].load(x[m] + k, end - k - k0);
#pragma unroll
    for (int r = 0; r < RT; r++) fw[r].load(w[r] + k, end - k - k0);
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int r = 0; r < RT; r++) acc[m][r] = mfma16(fw[r], fx[m], acc[m][r]);
  }
  if (wave) {
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int r = 0; r < RT; r++) part[wave - 1][m * RT + r][lane] = acc[m][r];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int m = 0; m < MT; m++) {
    const int i = m * 16 + lane % 16;
    if (i >= t.n) continue;
    float *to = a.mid + ((size_t)split * a.M + t.r0 + i) * a.R;
#pragma unroll
    for (int r = 0; r < RT; r++) {
      const f32x4_t sum = (acc[m][r] + part[0][m * RT + r][lane]) + (part[1][m * RT + r][lane] + part[2][m * RT + r][lane]);
      const float f[4] = {sum[0], sum[1], sum[2], sum[3]};
      const int at = r0 + r * 16 + lane / 16 * 4;
      if (at < a.R) store_v<float, 4>(to + at, a.R - at, f);
    }
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

// out.  grid (tiles * column blocks): 16 MT grouped rows by 256 columns of out a workgroup, 64 a wave; mid's shares
// are added up and cut into parts in LDS, 64 of R at a time.
template <typename T, typename TO, int MT, int PARTS>
__global__ __launch_bounds__(256) void k_adapters_expand(adapters_call a) {
  typedef typename expand_of<T>::type TE;
  typedef frag<TE> F;
  constexpr int RC = 64, STEPS = RC / F::STEP, WP = sizeof(T) == 2 && !std::is_same<T, TE>::value ? 2 : 1;
  constexpr int ROW = RC + F::V;  // a piece more, so that rows lie in different banks
  __shared__ __attribute__((aligned(16))) TE mid[PARTS][16 * MT][ROW];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane % 16, kg = lane / 16;
  const row_tile t = find_row_tile(a.offsets, a.n, a.M, blockIdx.x / a.col_blocks, 16 * MT);
  if (t.e < 0) return;
  const int n0 = blockIdx.x % a.col_blocks * 256 + wave * 64;
  const T *b = reinterpret_cast<const T *>(a.b) + (size_t)t.e * a.N * a.R;
  // lane's 8 columns n0 + 32 q + 8 kg + .. of the pairs q of weight tiles, of rows m * 16 + col
  int row[MT];
  raw_v<TO, 8> base[MT][2];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    row[m] = adapters_row(a, t, m * 16 + col);
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const int n = n0 + q * 32 + kg * 8;
      base[m][q].load(reinterpret_cast<const TO *>(a.base) + (size_t)(row[m] < 0 ? 0 : row[m]) * a.N + n,
                      row[m] < 0 ? 0 : a.N - n);
    }
  }
  f32x4_t acc[MT][4] = {};
  for (int rc = 0; rc < a.R; rc += RC) {
    if (rc) __syncthreads();
    for (int i = threadIdx.x; i < 16 * MT * RC; i += 256) {
      const int m = i / RC, r = rc + i % RC;
      float f = 0.0f;
      if (m < t.n && r < a.R) {
        const float *from = a.mid + (size_t)(t.r0 + m) * a.R + r;
#pragma unroll 8
        for (int s = 0; s < a.splits; s++) f += from[(size_t)s * a.M * a.R];
      }
#pragma unroll
      for (int p = 0; p < PARTS; p++) {
        const TE part = (TE)f;
        mid[p][m][i % RC] = part;
        f -= (float)part;
      }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
      const int r = s * F::STEP + kg * F::V;
      if (rc + s * F::STEP >= a.R) break;
      F fm[MT][PARTS];
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int p = 0; p < PARTS; p++) fm[m][p].v = *reinterpret_cast<const typename F::vec *>(&mid[p][m * 16 + col][r]);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int n = min(n0 + j / 2 * 32 + col / 4 * 8 + j % 2 * 4 + col % 4, a.N - 1);
        frag<T> w;
        F wp[WP];
        w.load(b + (size_t)n * a.R + rc + r, a.R - rc - r);
        weight_parts(w, wp);
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int p = 0; p < PARTS; p++)
#pragma unroll
            for (int q = 0; q < WP; q++) acc[m][j] = mfma16(wp[q], fm[m][p], acc[m][j]);
      }
    }
  }
  const float scale = a.scale ? a.scale[t.e] : 1.0f;
#pragma unroll
  for (int m = 0; m < MT; m++) {
    if (row[m] < 0) continue;
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const int n = n0 + q * 32 + kg * 8;
      if (n >= a.N) continue;
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = fmaf(scale, acc[m][2 * q + i / 4][i % 4], (float)base[m][q].v[i]);
      store_v<TO, 8>(reinterpret_cast<TO *>(a.out) + (size_t)row[m] * a.N + n, a.N - n, f);
    }
  }
}
