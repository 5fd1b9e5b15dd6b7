// kernels_dispatch.h -- tokens' rows to expert order and back, and the gradients.
//
// inv is moe_group's pair -> grouped row map (-1: the pair has no row), pair
// p = t*k + s.  Each kernel walks tokens and goes through inv, so a token's
// row is read (or written) once and nothing depends on how many pairs were
// dropped:
//   dispatch       rows[inv[p]] = x[t]
//   combine        out[t] = sum_s wts[p] * rows[inv[p]]   (slot order, f32)
//   dispatch_grad  combine with unit weights
//   combine_grad   drows[inv[p]] = wts[p] * dout[t], dwts[p] = <dout[t], rows[inv[p]]>
// A row index outside [0, n_rows) is treated as dropped.  Sums are f32 FMAs in
// a fixed order (no atomics); the one rounding to 16 bits is the store.
#pragma once

#include "device_common.h"

typedef __bf16 bf16_t;

// n of the V consecutive elements of a row at p, as floats (the others 0).
// Rows of any length and alignment: a whole vector is one or two 16-byte
// accesses at the type's own alignment, which global memory takes; the last
// vector of a row goes element by element.
template <typename T, int V>
__device__ __forceinline__ void load_v(const T *p, int n, float (&f)[V]) {
  typedef T vec_t __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  if (n >= V) {
    const vec_t v = *reinterpret_cast<const vec_t *>(p);
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = i < n ? (float)p[i] : 0.0f;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_v(T *p, int n, const float (&f)[V]) {
  typedef T vec_t __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  if (n >= V) {
    vec_t v;
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = (T)f[i];
    *reinterpret_cast<vec_t *>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (i < n) p[i] = (T)f[i];
  }
}

// grid (T, ny): workgroup (t, y) takes the vectors y*256 + tid, + ny*256, ...
template <typename TI, typename TO, int V>
__global__ __launch_bounds__(256) void k_dispatch(const TI *__restrict__ x, const int32_t *__restrict__ inv, int k, int H,
                                                  int n_rows, TO *__restrict__ rows) {
  const int t = blockIdx.x, nv = (H + V - 1) / V;
  const int32_t *iv = inv + (size_t)t * k;
  for (int v = blockIdx.y * 256 + threadIdx.x; v < nv; v += gridDim.y * 256) {
    float f[V];
    load_v<TI, V>(x + (size_t)t * H + (size_t)v * V, H - v * V, f);
    for (int s = 0; s < k; s++) {
      const int r = iv[s];
      if (r >= 0 && r < n_rows) store_v<TO, V>(rows + (size_t)r * H + (size_t)v * V, H - v * V, f);
    }
  }
}

// grid (T, ny) as above; wts NULL: unit weights.
template <typename TI, typename TO, int V>
__global__ __launch_bounds__(256) void k_combine_rows(const TI *__restrict__ rows, const float *__restrict__ wts,
                                                      const int32_t *__restrict__ inv, int k, int H, int n_rows,
                                                      TO *__restrict__ out) {
  const int t = blockIdx.x, nv = (H + V - 1) / V;
  const int32_t *iv = inv + (size_t)t * k;
  for (int v = blockIdx.y * 256 + threadIdx.x; v < nv; v += gridDim.y * 256) {
    float acc[V] = {};
    for (int s = 0; s < k; s++) {
      const int r = iv[s];
      if (r < 0 || r >= n_rows) continue;
      const float w = wts ? wts[(size_t)t * k + s] : 1.0f;
      float f[V];
      load_v<TI, V>(rows + (size_t)r * H + (size_t)v * V, H - v * V, f);
#pragma unroll
      for (int i = 0; i < V; i++) acc[i] = fmaf(w, f[i], acc[i]);
    }
    store_v<TO, V>(out + (size_t)t * H + (size_t)v * V, H - v * V, acc);
  }
}

// One wave per pair; dwts may be NULL.
template <typename TD, typename TR, int V>
__global__ __launch_bounds__(256) void k_combine_grad(const TD *__restrict__ dout, const TR *__restrict__ rows,
                                                      const float *__restrict__ wts, const int32_t *__restrict__ inv,
                                                      long P, int k, int H, int n_rows, TR *__restrict__ drows,
                                                      float *__restrict__ dwts) {
  const int lane = threadIdx.x & 63, nv = (H + V - 1) / V;
  const long p = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (p >= P) return;
  const int r = inv[p];
  float dot = 0.0f;
  if (r >= 0 && r < n_rows) {
    const float w = wts[p];
    const TD *d = dout + (size_t)(p / k) * H;
    const TR *y = rows + (size_t)r * H;
    TR *dy = drows + (size_t)r * H;
    for (int v = lane; v < nv; v += 64) {
      float a[V], b[V];
      load_v<TD, V>(d + (size_t)v * V, H - v * V, a);
      load_v<TR, V>(y + (size_t)v * V, H - v * V, b);
#pragma unroll
      for (int i = 0; i < V; i++) {
        dot = fmaf(a[i], b[i], dot);
        a[i] *= w;
      }
      store_v<TR, V>(dy + (size_t)v * V, H - v * V, a);
    }
  }
  dot = wave_sum(dot);
  if (lane == 0 && dwts) dwts[p] = dot;
}
