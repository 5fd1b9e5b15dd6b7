// kernels_i8.h -- rows quantised to 8 bits, and products of 8-bit rows with
// 8-bit weights, dense or over the experts' grouped rows.
//
//   scale[r] = fl32(amax_k |x[r,k]| / 127), q[r,k] = x[r,k] / scale[r] to the
//   nearest whole number, ties to even
//   y[r,n] = (sum_k q[r,k] * w[n,k]) * scale[r] * w_scale[n]
// The sum is exact in int32 (K <= MOE_I8_MAX_K); the three roundings after it
// (to f32, and one a scale) are f32's, and one more to 16 bits where out is.
#pragma once

#include "expert_kernels.h"
#include "kernels_dispatch.h"



typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

// ---- quantisation --------------------------------------------------------------

// The code of x: nearest whole number to x / s, ties to even, from a quotient
// that is off by less than one.  r = x - q*s is exact (q*s and x are multiples
// of one power of two, r is at most 0.5 s), so comparing |r| with s/2 decides
// the neighbour and the ties as exact arithmetic would.
__device__ __forceinline__ int i8_code(float x, float s, float inv) {
  float q = __builtin_rintf(x * inv);
  const float r = fmaf(-q, s, x), a = fabsf(r), h = 0.5f * s;
  const bool odd = (int)q & 1;
  if (a > h || (a == h && odd)) q += copysignf(1.0f, r);
  return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// What a row's codes need, from the bits of its largest |x| (as integers, NaN
// above infinity above every finite value): the row's scale; x is multiplied
// by pre and divided by s = scale * pre, where pre = 2^64 keeps tiny rows
// clear of denormal quotients.  A row that holds a NaN or an infinity gets a
// NaN scale and codes 0: every product of it is NaN, none is silently wrong.
struct i8_row {
  float scale, pre, s, inv;
};
__device__ __forceinline__ i8_row i8_row_of(uint32_t amax_bits) {
  i8_row w;
  const float amax = __builtin_bit_cast(float, amax_bits);
  if (amax_bits >= 0x7f800000u) {
    w.scale = __builtin_nanf("");
    w.pre = w.s = w.inv = 0.0f;
    return w;
  }
  w.scale = __fdiv_rn(amax, 127.0f);
  w.pre = amax < 0x1p-60f ? 0x1p64f : 1.0f;
  w.s = w.scale * w.pre;
  w.inv = w.s > 0.0f ? __fdiv_rn(1.0f, w.s) : 0.0f;
  return w;
}
__device__ __forceinline__ int i8_code_in(const i8_row &w, float x) {
  return w.inv > 0.0f ? i8_code(x * w.pre, w.s, w.inv) : 0;
}

__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = (uint32_t)__shfl_xor((int)v, o);
    v = u > v ? u : v;
  }
  return v;
}

// Any K and alignment: one workgroup per row, two passes over it.
template <typename T>
__global__ __launch_bounds__(256) void k_quantize_i8_any(const T *__restrict__ x, int K, int8_t *__restrict__ q,
                                                         float *__restrict__ scale) {
  __shared__ uint32_t part[4];
  const int tid = threadIdx.x;
  const T *xr = x + (size_t)blockIdx.x * K;
  uint32_t m = 0;
  for (int i = tid; i < K; i += 256) {
    const uint32_t b = __builtin_bit_cast(uint32_t, (float)xr[i]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  m = wave_max_u(m);
  if ((tid & 63) == 0) part[tid >> 6] = m;
  __syncthreads();
  m = max(max(part[0], part[1]), max(part[2], part[3]));
  const i8_row w = i8_row_of(m);
  for (int i = tid; i < K; i += 256) q[(size_t)blockIdx.x * K + i] = (int8_t)i8_code_in(w, (float)xr[i]);
  if (tid == 0) scale[blockIdx.x] = w.scale;
}

// ---- products --------------------------------------------------------------------

// The rows of one tile: expert e (-1: none left), rows [r0, r0 + n).
struct i8_tile {
  int e, r0, n;
};

// Tile `item` of the grouped rows cut into tiles of at most BM: expert e has
// ceil(c_e / BM) of them, in expert order.  Every wave finds it for itself:
// lane l holds the tile counts of 16 consecutive experts (E <= 1024), one scan
// over the lanes, and the owner broadcasts.  Offsets are held to [0, M].
__device__ __forceinline__ i8_tile i8_find_tile(const i8_mm &a, int item, int BM) {
  if (!a.offsets) {
    const int r0 = item * BM;
    return {r0 < a.M ? 0 : -1, r0, a.M - r0 < BM ? a.M - r0 : BM};
  }
  const int lane = threadIdx.x & 63, per = (a.E + 63) / 64;
  int n = 0;
  for (int i = 0; i < per; i++) {
    const int e = lane * per + i;
    if (e >= a.E) break;
    const int lo = min(max(a.offsets[e], 0), a.M), hi = min(max(a.offsets[e + 1], 0), a.M);
    n += hi > lo ? (hi - lo + BM - 1) / BM : 0;
  }
  int sum = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(sum, o);
    if (lane >= o) sum += u;
  }
  int first = sum - n;
  const uint64_t here = __ballot(first <= item && item < sum);
  i8_tile t = {-1, 0, 0};
  if (!here) return t;
  if (first <= item && item < sum) {
    for (int i = 0; i < per; i++) {
      const int e = lane * per + i;
      if (e >= a.E) break;
      const int lo = min(max(a.offsets[e], 0), a.M), hi = min(max(a.offsets[e + 1], 0), a.M);
      const int c = hi > lo ? (hi - lo + BM - 1) / BM : 0;
      if (item < first + c) {
        const int r0 = lo + (item - first) * BM;
        t = {e, r0, hi - r0 < BM ? hi - r0 : BM};
        break;
      }
      first += c;
    }
  }
  const int owner = __ffsll((unsigned long long)here) - 1;
  t.e = __builtin_amdgcn_readlane(t.e, owner);
  t.r0 = __builtin_amdgcn_readlane(t.r0, owner);
  t.n = __builtin_amdgcn_readlane(t.n, owner);
  return t;
}

// Source row of grouped row r (-1 where perm points outside).
__device__ __forceinline__ int i8_src(const i8_mm &a, int r) {
  if (!a.perm) return r < a.n_src ? r : -1;
  const int p = a.perm[r];
  const int s = p >= 0 ? p / a.k : -1;
  return s < a.n_src ? s : -1;
}

__device__ __forceinline__ float i8_swiglu(float g, float u, float L) {
  if (L > 1e-6f) {  // comparisons, so that a NaN stays one
    g = g > L ? L : g;
    u = u > L ? L : (u < -L ? -L : u);
  }
  return g / (1.0f + __expf(-g)) * u;
}

template <typename T>
__device__ __forceinline__ void i8_store(const i8_mm &a, int r, int n, float v) {
  const int No = a.swiglu ? a.N / 2 : a.N;
  reinterpret_cast<T *>(a.out)[(size_t)r * No + n] = (T)v;
}

// 16 bytes of a row at k, any alignment; bytes from K on are 0.
__device__ __forceinline__ v4i i8_bytes(const int8_t *row, int k, int K) {
  v4i v = {0, 0, 0, 0};
  if (k + 16 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else {
    int8_t b[16];
#pragma unroll
    for (int i = 0; i < 16; i++) b[i] = k + i < K ? row[k + i] : (int8_t)0;
    __builtin_memcpy(&v, b, 16);
  }
  return v;
}

// Any K and alignment: tiles of 64 rows x 64 channels, 64 bytes of K a step
// through registers into LDS.  Wave (wm, wn) multiplies 32 rows with two
// 16-channel tiles, wn*16 of each half of the 64 (SwiGLU: the halves are gate
// and up, so a lane holds both of its channels).
// 16x16x64 MFMA, weights as A, rows as B: lane l holds K bytes [16 (l/16), +16)
// of A row (B column) l % 16; D lane l holds column l % 16, rows 4 (l/16) + i.
template <typename TO>
__global__ __launch_bounds__(256) void k_mm_i8_any(i8_mm a) {
  __shared__ v4i xs[64][5], wsh[64][5];  // 4 chunks of 16 bytes a row, and one of padding
  const i8_tile t = i8_find_tile(a, blockIdx.y, 64);
  if (t.e < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  const int half = a.swiglu ? a.N / 2 : 32, per = a.swiglu ? 32 : 64;  // channels a workgroup: per of each half
  const int n0 = blockIdx.x * per, n_end = a.swiglu ? a.N / 2 : a.N;
  const int row = tid >> 2, ch = tid & 3;
  // this thread's LDS row of weights: channel n0 + row, or gate / up channel n0 + row % 32
  const int wc = a.swiglu ? n0 + (row & 31) : n0 + row;
  const int wrow = a.swiglu ? (row >> 5) * half + wc : wc;
  const int src = row < t.n ? i8_src(a, t.r0 + row) : -1;
  const int8_t *xr = a.q + (size_t)max(src, 0) * a.K;
  const int8_t *wr = a.w + ((size_t)t.e * a.N + (wc < n_end ? wrow : 0)) * a.K;
  v4i acc[2][2] = {};
  for (int k0 = 0; k0 < a.K; k0 += 64) {
    const v4i z = {0, 0, 0, 0};
    const v4i xv = src >= 0 ? i8_bytes(xr, k0 + 16 * ch, a.K) : z, wv = wc < n_end ? i8_bytes(wr, k0 + 16 * ch, a.K) : z;
    __syncthreads();
    xs[row][ch] = xv;
    wsh[row][ch] = wv;
    __syncthreads();
    v4i A[2], B[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      A[j] = wsh[32 * j + 16 * wn + (lane & 15)][lane >> 4];
      B[j] = xs[32 * wm + 16 * j + (lane & 15)][lane >> 4];
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[i], B[j], acc[i][j], 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const int m = 32 * wm + 16 * j + (lane & 15);
    if (m >= t.n) continue;
    const int r = t.r0 + m, s = i8_src(a, r);
    const float sx = s >= 0 ? a.qs[s] : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int nl = 16 * wn + 4 * (lane >> 4) + i;
      const float *wsc = a.ws + (size_t)t.e * a.N;
      if (a.swiglu) {
        const int n = n0 + nl;
        if (n < n_end)
          i8_store<TO>(a, r, n, i8_swiglu((float)acc[0][j][i] * sx * wsc[n], (float)acc[1][j][i] * sx * wsc[half + n], a.clamp));
      } else {
        if (n0 + nl < n_end) i8_store<TO>(a, r, n0 + nl, (float)acc[0][j][i] * sx * wsc[n0 + nl]);
        if (n0 + 32 + nl < n_end) i8_store<TO>(a, r, n0 + 32 + nl, (float)acc[1][j][i] * sx * wsc[n0 + 32 + nl]);
      }
    }
  }
}
