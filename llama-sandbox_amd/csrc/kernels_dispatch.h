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

// V consecutive elements of a row, or as many as are left of it (the others
// 0).  Rows of any length and alignment: a whole vector is one or two 16-byte
// accesses at the type's own alignment, which global memory takes; the last
// vector of a row goes element by element.  raw: loaded, not yet converted, so
// that several can be in flight.
template <typename T, int V, bool NT = false>
struct raw_v {
  typedef T vec_t __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  vec_t v;
  __device__ __forceinline__ void load(const T *p, int left) {
    if (left >= V) {
      v = NT ? __builtin_nontemporal_load(reinterpret_cast<const vec_t *>(p)) : *reinterpret_cast<const vec_t *>(p);
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) v[i] = i < left ? p[i] : (T)0.0f;
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ void load_v(const T *p, int left, float (&f)[V]) {
  raw_v<T, V> r;
  r.load(p, left);
#pragma unroll
  for (int i = 0; i < V; i++) f[i] = (float)r.v[i];
}

template <typename T, int V, bool NT = false>
__device__ __forceinline__ void store_v(T *p, int left, const float (&f)[V]) {
  typedef typename raw_v<T, V>::vec_t vec_t;
  if (left >= V) {
    vec_t v;
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = (T)f[i];
    if (NT) __builtin_nontemporal_store(v, reinterpret_cast<vec_t *>(p));
    else *reinterpret_cast<vec_t *>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (i < left) p[i] = (T)f[i];
  }
}

// grid (T, ny): workgroup (t, y) takes the vectors y*256 + tid, + ny*256, ...
// Bound by memory: a row is read once and its k copies leave from registers,
// which a walk over the grouped rows could not do.  ny > 1 only where tokens
// are too few to fill the chip.  4096 tokens to 8 experts, 7168 bf16 (529 MB)
// 93 us, 5.7 TB/s; one token 2.6 us, a launch.
template <typename TI, typename TO, int V, bool NT>
__global__ __launch_bounds__(256) void k_dispatch(const TI *__restrict__ x, const int32_t *__restrict__ inv, int k, int H,
                                                  int n_rows, TO *__restrict__ rows) {
  const int t = blockIdx.x, nv = (H + V - 1) / V;
  const int32_t *iv = inv + (size_t)t * k;
  for (int v = blockIdx.y * 256 + threadIdx.x; v < nv; v += gridDim.y * 256) {
    float f[V];
    load_v<TI, V>(x + (size_t)t * H + (size_t)v * V, H - v * V, f);
    for (int s = 0; s < k; s++) {
      const int r = iv[s];
      if (r >= 0 && r < n_rows) store_v<TO, V, NT>(rows + (size_t)r * H + (size_t)v * V, H - v * V, f);
    }
  }
}

// grid (T, ny) as above; wts NULL: unit weights.  Bound by memory, by its
// latency where tokens are few: the rows of 8 slots are asked for before the
// first is added.  2048 tokens of 8 slots, 7168 f32 (529 MB) 97 us, 5.5 TB/s
// (110 with one row at a time and through the caches); 37 of 6, 5120 f16 3.4 us.
template <typename TI, typename TO, int V, bool NT>
__global__ __launch_bounds__(256) void k_combine_rows(const TI *__restrict__ rows, const float *__restrict__ wts,
                                                      const int32_t *__restrict__ inv, int k, int H, int n_rows,
                                                      TO *__restrict__ out) {
  constexpr int S = 8;
  const int t = blockIdx.x, nv = (H + V - 1) / V;
  const int32_t *iv = inv + (size_t)t * k;
  for (int v = blockIdx.y * 256 + threadIdx.x; v < nv; v += gridDim.y * 256) {
    float acc[V] = {};
    for (int s0 = 0; s0 < k; s0 += S) {
      raw_v<TI, V, NT> y[S];
      int r[S];
#pragma unroll
      for (int s = 0; s < S; s++) {
        r[s] = s0 + s < k ? iv[s0 + s] : -1;
        r[s] = r[s] < n_rows ? r[s] : -1;
        if (r[s] >= 0) y[s].load(rows + (size_t)r[s] * H + (size_t)v * V, H - v * V);
      }
#pragma unroll
      for (int s = 0; s < S; s++) {
        if (r[s] < 0) continue;
        const float w = wts ? wts[(size_t)t * k + s0 + s] : 1.0f;
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] = fmaf(w, (float)y[s].v[i], acc[i]);
      }
    }
    store_v<TO, V>(out + (size_t)t * H + (size_t)v * V, H - v * V, acc);
  }
}

// WPP waves per pair, 8 waves a workgroup (a token's pairs next to each other:
// dout comes from L2 after the first), 4 vectors of each row in flight.  Bound
// by memory: drows and the dot product share one pass over dout and rows.
// 4096 tokens of 8 slots, 7168 bf16 (999 MB) 196 us, 5.1 TB/s; 301 of 4, 2048
// f32 (17 MB) 5.2 us, most of it latency.
template <typename TD, typename TR, int V, int WPP, bool NT>
__global__ __launch_bounds__(512) void k_combine_grad(const TD *__restrict__ dout, const TR *__restrict__ rows,
                                                      const float *__restrict__ wts, const int32_t *__restrict__ inv,
                                                      long P, int k, int H, int n_rows, TR *__restrict__ drows,
                                                      float *__restrict__ dwts) {
  constexpr int S = 4;
  __shared__ float part[8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nv = (H + V - 1) / V;
  const long p = (long)blockIdx.x * (8 / WPP) + wave / WPP;
  const int r = p < P ? inv[p] : -1;
  float dot = 0.0f;
  if (r >= 0 && r < n_rows) {
    const float w = wts[p];
    const TD *d = dout + (size_t)(p / k) * H;
    const TR *y = rows + (size_t)r * H;
    TR *dy = drows + (size_t)r * H;
    for (int v0 = wave % WPP * 64 + lane; v0 < nv; v0 += 64 * WPP * S) {
      raw_v<TD, V> a[S];
      raw_v<TR, V, NT> b[S];
#pragma unroll
      for (int u = 0; u < S; u++) {
        const int v = v0 + 64 * WPP * u;
        if (v < nv) {
          a[u].load(d + (size_t)v * V, H - v * V);
          b[u].load(y + (size_t)v * V, H - v * V);
        }
      }
#pragma unroll
      for (int u = 0; u < S; u++) {
        const int v = v0 + 64 * WPP * u;
        if (v >= nv) break;
        float f[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
          f[i] = (float)a[u].v[i];
          dot = fmaf(f[i], (float)b[u].v[i], dot);
          f[i] *= w;
        }
        store_v<TR, V, NT>(dy + (size_t)v * V, H - v * V, f);
      }
    }
  }
  dot = wave_sum(dot);
  if constexpr (WPP > 1) {
    if (lane == 0) part[wave] = dot;
    __syncthreads();
    dot = 0.0f;
#pragma unroll
    for (int i = 0; i < WPP; i++) dot += part[wave / WPP * WPP + i];
  }
  if (p < P && wave % WPP == 0 && lane == 0) dwts[p] = dot;
}
