// kernels_adapters.h -- low-rank adapters of many requests beside a shared projection.
//
//   mid[i] = A[a] x[perm[i]],  out[perm[i]] = base[perm[i]] + scale[a] * B[a] mid[i]
// for the grouped rows i of adapter a, [offsets[a], offsets[a+1]).  mid is f32.
#pragma once

#include "group_tiles.h"
#include "layer_kernels.h"
#include "row_vec.h"
#include "../../include/moe_block.h"

// grid (ceil(R / 4), M): a wave for one grouped row and one row of A.
template <typename T>
__global__ __launch_bounds__(256) void k_adapters_shrink(adapters_call a) {
  const int lane = threadIdx.x & 63, i = blockIdx.y, j = blockIdx.x * 4 + (threadIdx.x >> 6);
  const row_tile t = find_row_tile(a.offsets, a.n, a.M, i, 1);
  if (t.e < 0 || j >= a.R) return;
  const int row = a.perm[t.r0];
  if (row < 0 || row >= a.M) return;
  const T *x = reinterpret_cast<const T *>(a.x) + (size_t)row * a.K;
  const T *w = reinterpret_cast<const T *>(a.a) + ((size_t)t.e * a.R + j) * a.K;
  float sum = 0.0f;
  for (int k = lane; k < a.K; k += 64) sum = fmaf((float)x[k], (float)w[k], sum);
  sum = wave_sum(sum);
  if (lane == 0) a.mid[(size_t)t.r0 * a.R + j] = sum;
}

// grid (ceil(N / 256), M): a thread for one value of one grouped row.
template <typename T, typename TO>
__global__ __launch_bounds__(256) void k_adapters_expand(adapters_call a) {
  const int i = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
  const row_tile t = find_row_tile(a.offsets, a.n, a.M, i, 1);
  if (t.e < 0 || n >= a.N) return;
  const int row = a.perm[t.r0];
  if (row < 0 || row >= a.M) return;
  const T *w = reinterpret_cast<const T *>(a.b) + ((size_t)t.e * a.N + n) * a.R;
  float sum = 0.0f;
  for (int j = 0; j < a.R; j++) sum = fmaf(a.mid[(size_t)t.r0 * a.R + j], (float)w[j], sum);
  if (a.scale) sum *= a.scale[t.e];
  const size_t at = (size_t)row * a.N + n;
  reinterpret_cast<TO *>(a.out)[at] = (TO)((float)reinterpret_cast<const TO *>(a.base)[at] + sum);
}
