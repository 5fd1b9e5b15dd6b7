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
#include "../../include/moe_block.h"
#include "group_tiles.h"
#include "lds_dma.h"
#include "row_vec.h"

#include <type_traits>

typedef int v4i __attribute__((ext_vector_type(4)));

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

// What the code of x is more than u - 1.5 * 2^23, the whole number at most one off; as
// above, without branches and for rows that need no pre.
__device__ __forceinline__ int i8_correction(const i8_row &w, float x, float u) {
  const float r = fmaf(0x1.8p23f - u, w.s, x), past = fabsf(r) - 0.5f * w.s;
  const bool odd = __builtin_bit_cast(uint32_t, u) & 1;
  return (past > 0.0f) | ((past == 0.0f) & odd) ? (r < 0.0f ? -1 : 1) : 0;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
  v = dpp_max<0xB1>(v);   // quad_perm [1,0,3,2]
  v = dpp_max<0x4E>(v);   // quad_perm [2,3,0,1]
  v = dpp_max<0x141>(v);  // row_half_mirror
  v = dpp_max<0x140>(v);  // row_mirror: every lane holds its row of 16's
  const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)v, 0), b = (uint32_t)__builtin_amdgcn_readlane((int)v, 16);
  const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)v, 32), d = (uint32_t)__builtin_amdgcn_readlane((int)v, 48);
  return max(max(a, b), max(c, d));
}

// Of the 32 lanes that a lane is one of.
__device__ __forceinline__ uint32_t half_wave_max_u(uint32_t v) {
  v = dpp_max<0xB1>(v);
  v = dpp_max<0x4E>(v);
  v = dpp_max<0x141>(v);
  v = dpp_max<0x140>(v);
  return max(v, (uint32_t)__shfl_xor((int)v, 16));
}

// Largest |x| of a vector as it was loaded, as the bits of a float: bits without the
// sign grow with the value, NaN above infinity above every finite one.
template <typename T, int V>
__device__ __forceinline__ uint32_t abs_bits(const raw_v<T, V> &r) {
  uint32_t m = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; i++) {
      const float e = r.v[i];  // (a bit cast of the vector's element itself reads element 0)
      m = max(m, __builtin_bit_cast(uint32_t, e) & 0x7fffffffu);
    }
    return m;
  } else {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 p = {0, 0};
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const T e0 = r.v[i], e1 = r.v[i + 1];
      const u16x2 w = {(uint16_t)(__builtin_bit_cast(uint16_t, e0) & 0x7fff), (uint16_t)(__builtin_bit_cast(uint16_t, e1) & 0x7fff)};
      p = __builtin_elementwise_max(p, w);
    }
    const uint16_t h = p.x > p.y ? p.x : p.y;
    return __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(T, h));
  }
}

// A row's codes in one pass: LANES threads hold it in registers, VPT vectors of 8 each
// (K <= 8 LANES VPT); 256 / LANES rows a workgroup where that is more than one.
// Memory bound (2 to 4 bytes in, 1 out) only while the codes are cheap: x * inv, before
// it is rounded, is within 127 * 2^-24 = 7.6e-6 of x / s, so it decides all but those next
// to a tie, and only waves that hold one look at the remainders: one vector in a hundred
// of f32 values, most of 16-bit ones (their quotients have small denominators, and meet ties
// exactly).  x * inv + 1.5 * 2^23 is rounded once, to a whole number, ties to even,
// with the code in its low byte.  4096 rows of 7168 bf16 (88 MB) 18.8 to 20.0 us, 4.4 to 4.7 TB/s
// (22.1 where a tie took the whole quotient again, with branches); 32764 of 768 (76 MB)
// 17.8, between products 21.5, two rows a wave (23.5 with one row and a third of the lanes idle); one row
// 2.3, a launch.  Workgroups that walk rows with the next one's loads in flight took 24
// to 29 us for the first.
template <typename T, int LANES, int VPT>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void k_quantize_i8(const T *__restrict__ x, int M, int K,
                                                                           int8_t *__restrict__ q, float *__restrict__ scale) {
  constexpr int RPW = LANES < 256 ? 256 / LANES : 1, WPR = LANES / 64;  // rows a workgroup, waves a row
  __shared__ uint32_t part[LANES < 256 ? 4 : WPR];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, in_row = tid % LANES;
  const long row = (long)blockIdx.x * RPW + tid / LANES;
  const T *xr = x + (row < M ? row : 0) * K;
  raw_v<T, 8> r[VPT];
#pragma unroll
  for (int v = 0; v < VPT; v++) {
    const int c = (in_row + v * LANES) * 8;
    r[v].load(xr + c, row < M ? K - c : 0);
  }
  uint32_t m = 0;
#pragma unroll
  for (int v = 0; v < VPT; v++) m = max(m, abs_bits(r[v]));
  m = LANES == 32 ? half_wave_max_u(m) : wave_max_u(m);
  if constexpr (WPR > 1) {
    if (lane == 0) part[wave] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WPR; i++) m = max(m, part[wave / WPR * WPR + i]);
  }
  if (row >= M) return;
  const i8_row w = i8_row_of(m);
#pragma unroll
  for (int v = 0; v < VPT; v++) {
    const int c = (in_row + v * LANES) * 8;
    if (c >= K) break;
    uint32_t code[8];
    float far = 0.0f;  // the largest distance of a quotient from its whole number
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float e = (float)r[v].v[i], u = fmaf(e, w.inv, 0x1.8p23f);
      far = fmaxf(far, fabsf(fmaf(e, w.inv, 0x1.8p23f - u)));
      code[i] = __builtin_bit_cast(uint32_t, u);
    }
    if (w.pre != 1.0f) {
#pragma unroll
      for (int i = 0; i < 8; i++) code[i] = (uint32_t)i8_code_in(w, (float)r[v].v[i]);
    } else if (__any(far > 0.49999f)) {
#pragma unroll
      for (int i = 0; i < 8; i++) code[i] += i8_correction(w, (float)r[v].v[i], __builtin_bit_cast(float, code[i]));
    }
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2), aligned(1)));
    int8_t *to = q + row * K + c;
    if (c + 8 <= K) {
      u32x2 o;
#pragma unroll
      for (int h = 0; h < 2; h++)
        o[h] = (code[4 * h] & 255) | (code[4 * h + 1] & 255) << 8 | (code[4 * h + 2] & 255) << 16 | code[4 * h + 3] << 24;
      *reinterpret_cast<u32x2 *>(to) = o;
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (c + i < K) to[i] = (int8_t)code[i];
    }
  }
  if (in_row == 0) scale[row] = w.scale;
}

// Rows too long for registers: one workgroup a row, two passes over it.
template <typename T>
__global__ __launch_bounds__(256) void k_quantize_i8_long(const T *__restrict__ x, int K, int8_t *__restrict__ q,
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

__device__ __forceinline__ row_tile i8_find_tile(const i8_mm &a, int item, int BM) {
  if (!a.offsets) {
    const int r0 = item * BM;
    return {r0 < a.M ? 0 : -1, r0, a.M - r0 < BM ? a.M - r0 : BM, a.M <= BM};
  }
  return find_row_tile(a.offsets, a.E, a.M, item, BM);
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

// The type is the same for a whole call: a uniform branch.
__device__ __forceinline__ void i8_store(const i8_mm &a, int r, int n, float v) {
  const size_t at = (size_t)r * (a.swiglu ? a.N / 2 : a.N) + n;
  if (a.out_type == MOE_GGML_F32) reinterpret_cast<float *>(a.out)[at] = v;
  else if (a.out_type == MOE_GGML_F16) reinterpret_cast<_Float16 *>(a.out)[at] = (_Float16)v;
  else reinterpret_cast<bf16_t *>(a.out)[at] = (bf16_t)v;
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

// Any K and alignment: tiles of 64 rows x 64 channels, 128 bytes of K a step
// through registers (unaligned 16-byte loads, a step ahead) into LDS.  Wave (wm, wn)
// multiplies 32 rows with two 16-channel tiles, wn*16 of each half of the 64
// (SwiGLU: the halves are gate and up, so a lane holds both of its channels).
// 16x16x64 MFMA, channels as A, rows as B: lane l holds K bytes [16 (l/16), +16)
// of A row (B column) l % 16; D lane l holds column l % 16, rows 4 (l/16) + i.
// Bound by the loads' latency where the tiles are few, by the small tile's traffic
// where they are many: K = 1765 against K = 1776 on the other kernels, 4096 channels, weights from the
// caches: 1 row 11.7 and 3.2 us, 300 rows 19 and 8.0, 4096 rows 126 and 34.
// (nt along x and row tiles along y and z, not one index that is divided: 20000 x 101 x 300 17.5 us, 20.3 with a division.)
__global__ __launch_bounds__(256) void k_mm_i8_any(i8_mm a) {
  __shared__ v4i xs[64][9], wsh[64][9];  // 8 chunks of 16 bytes a row, and one of padding
  const row_tile t = i8_find_tile(a, blockIdx.z * gridDim.y + blockIdx.y, 64);
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
  v4i xv[2], wv[2];
  auto fetch = [&](int k0) __attribute__((always_inline)) {
    const v4i z = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int k = k0 + 16 * (ch + 4 * i);
      xv[i] = src >= 0 ? i8_bytes(xr, k, a.K) : z;
      wv[i] = wc < n_end ? i8_bytes(wr, k, a.K) : z;
    }
  };
  fetch(0);
  for (int k0 = 0; k0 < a.K; k0 += 128) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; i++) {
      xs[row][ch + 4 * i] = xv[i];
      wsh[row][ch + 4 * i] = wv[i];
    }
    __syncthreads();
    if (k0 + 128 < a.K) fetch(k0 + 128);
#pragma unroll
    for (int kk = 0; kk < 2; kk++) {
      v4i A[2], B[2];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        A[j] = wsh[32 * j + 16 * wn + (lane & 15)][4 * kk + (lane >> 4)];
        B[j] = xs[32 * wm + 16 * j + (lane & 15)][4 * kk + (lane >> 4)];
      }
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[i], B[j], acc[i][j], 0, 0, 0);
    }
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
          i8_store(a, r, n, i8_swiglu((float)acc[0][j][i] * sx * wsc[n], (float)acc[1][j][i] * sx * wsc[half + n], a.clamp));
      } else {
        if (n0 + nl < n_end) i8_store(a, r, n0 + nl, (float)acc[0][j][i] * sx * wsc[n0 + nl]);
        if (n0 + 32 + nl < n_end) i8_store(a, r, n0 + 32 + nl, (float)acc[1][j][i] * sx * wsc[n0 + 32 + nl]);
      }
    }
  }
}

// Few rows: up to M a tile, straight from memory to registers.  A workgroup is one wave
// and takes C channels (SwiGLU: C / 2 columns, gate and up by turns); lane l multiplies
// bytes [16 l, +16) of every 1024 of K, U times 1024 in flight for all channels and
// rows, 4 products an instruction; the lanes' sums meet by DPP.  No LDS and no barrier: where the
// weights are small the staged tiles spend 4 us on the turns of their loop, and
// where they are large this streams as well (us, staged / this; rows x K x N):
// 1 x 7168 x 512 6.8 / 3.4, 1 x 4096 x 4096 7.3 / 5.1, 1 x 7168 x 4096 8.4 / 7.0, 1 x 5120 x 32000 30.1 / 27.3,
// one token's 8 experts of 7168 x 4096 39.3 / 36.6 (6.4 TB/s).
template <int M, int C, int U>
__global__ __launch_bounds__(64) void k_mv_i8(i8_mm a, int nt) {
  const int lane = threadIdx.x;
  const row_tile t = i8_find_tile(a, blockIdx.x / nt, M);
  if (t.e < 0) return;
  const int half = a.N / 2, n_end = a.swiglu ? half : a.N, cols = a.swiglu ? C / 2 : C;
  const int n0 = blockIdx.x % nt * cols;
  const int8_t *w[C], *x[M];
#pragma unroll
  for (int c = 0; c < C; c++) {  // past the end: the last one again
    const int n = min(n0 + (a.swiglu ? c / 2 : c), n_end - 1);
    w[c] = a.w + ((size_t)t.e * a.N + (a.swiglu && c % 2 ? half + n : n)) * a.K;
  }
  // lane m * cols + o ends up with row m's column o; the scales are asked for first
  const int m_lane = lane >> (a.swiglu ? __builtin_ctz(C) - 1 : __builtin_ctz(C)), n = n0 + (lane & (cols - 1));
  const float *ws = a.ws + (size_t)t.e * a.N + min(n, n_end - 1);
  const float s_n = ws[0], s_up = a.swiglu ? ws[half] : 0.0f;
  int acc[M][C] = {}, src[M], row = -1;
#pragma unroll
  for (int m = 0; m < M; m++) {
    src[m] = __builtin_amdgcn_readfirstlane(m < t.n ? i8_src(a, t.r0 + m) : -1);
    x[m] = a.q + (size_t)max(src[m], 0) * a.K;
    if (m_lane == m) row = src[m];
  }
  const float s_row = row >= 0 ? a.qs[row] : 0.0f;
  auto sums = [&](auto once) __attribute__((always_inline)) {
    for (int k0 = 0; k0 < a.K; k0 += 1024 * U) {
      v4i wv[C][U], xv[M][U];
#pragma unroll
      for (int u = 0; u < U; u++) {  // past K: the last 16 bytes, against zeros
        const int at = min(k0 + 1024 * u + 16 * lane, a.K - 16);
#pragma unroll
        for (int c = 0; c < C; c++) {
          const v4i *p = reinterpret_cast<const v4i *>(w[c] + at);
          wv[c][u] = decltype(once)::value ? __builtin_nontemporal_load(p) : *p;
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int k = k0 + 1024 * u + 16 * lane;
#pragma unroll
        for (int m = 0; m < M; m++) {
          const v4i v = *reinterpret_cast<const v4i *>(x[m] + min(k, a.K - 16));
#pragma unroll
          for (int i = 0; i < 4; i++) xv[m][u][i] = k < a.K ? v[i] : 0;
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
          for (int m = 0; m < M; m++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[m][c] = __builtin_amdgcn_sdot4(wv[c][u][i], xv[m][u][i], acc[m][c], false);
    }
  };
  if (a.stream && t.only) sums(std::true_type{});
  else sums(std::false_type{});
  int s0 = 0, s1 = 0;
#pragma unroll
  for (int m = 0; m < M; m++)
#pragma unroll
    for (int c = 0; c < C; c++) {
      const int s = src[m] < 0 ? 0 : __builtin_amdgcn_readlane(wave_scan(acc[m][c]), 63);
      if (lane == m * cols + (a.swiglu ? c / 2 : c)) (a.swiglu && c % 2 ? s1 : s0) = s;
    }
  if (m_lane >= t.n || m_lane >= M || n >= n_end) return;
  const float y = (float)s0 * s_row * s_n;
  i8_store(a, t.r0 + m_lane, n, a.swiglu ? i8_swiglu(y, (float)s1 * s_row * s_up, a.clamp) : y);
}

// ---- staged tiles -------------------------------------------------------------------
//
// K % 16 == 0 and 16-byte aligned rows.  A workgroup multiplies BM rows with BN
// channels; both go to LDS by direct loads, 128 bytes of K a row and block,
// NBUF stages around.  A 1 KiB load is 8 rows; the 16-byte chunk c of row r lies
// at c ^ (r & 7), so that the 16 rows that an MFMA operand reads at one chunk fall
// on all banks.  Waves: WM x WN over the tile, and WK over K (a stage is WK blocks
// of 128 bytes, wave k takes block k; the sums meet in LDS after the loop).
// 16x16x64 MFMA, channels as A and rows as B: D lane l holds row l % 16 of its
// row tile and channels 4 (l / 16) + i of its channel tile.
// Bound by, and measured (kernel alone):
//   4096 x 7168 x 7168, 256x256: 171 to 187 us, 2.46 to 2.25 PO/s; 8192 x 8192 x 8192 421 us, 2.61.  A
//     tile's start and end are a tenth; of the launch's cycles the MFMA pipes are busy for 57% (65%
//     of those in which a CU has one of its 1.75 tiles), the LDS reads for 23%; waves wait for LDS in 4% of
//     theirs: the rest is mostly the wait at each stage's barrier.  Waves of 128 rows x 64 channels 187 us, of
//     64 x 128 191; a non-temporal choice at every load, which cut the loop into blocks, 204.
//     16x16x64 from registers alone reaches 3.8 PO/s here, 32x32x32 3.3.
//   16 or 4096 rows over the experts, 64x128: the weights' stream from HBM, 6.2 to
//     6.5 TB/s (32x128 to 128x64 within a few percent).
//   32764 x 768 x 2048 to f32, 256x256: 116 us, the output's 262 MB and the start
//     of short tiles (13 thousand cycles before the first MFMA, 21 of K, 16 of output).
//     A workgroup that takes tile after tile, the next one's loads behind the output,
//     was slower in every shape (the stores delay the waits for those loads).
//   16 rows x 7168 x 4096: 8.6 us, latency: 16x16 tiles, K over 4 waves.
// Load i of this wave's share (loads wave, wave + NW, ...) of the N_LOAD 1 KiB loads
// of a stage from K byte k0 on, R rows a block of 128 bytes.  vo: lane offsets at
// K 0.  Lanes past K, and every lane of a stage past the end, are out of range:
// they read 0, and the waits can count on the loads.
template <int R, int N_LOAD, int NW, bool ONCE>
__device__ __forceinline__ void i8_load(int i, const int8_t *base, uint32_t bytes, uint32_t vo, v4i *buf, int wave, int k0,
                                        int k_lane, int K) {
  const int u = wave + NW * i;
  const uint32_t at = k0 + 8 * u / R * 128 + k_lane < K ? vo : MOE_LDS_OOB;
  if (N_LOAD % NW == 0 || u < N_LOAD) {  // uniform over the wave
    if constexpr (ONCE) lds_dma_once(base, bytes, buf + u * 64, at, k0 < K ? k0 : 0);
    else lds_dma(base, bytes, buf + u * 64, at, k0 < K ? k0 : 0);
  }
}

// A wave's rows on their way out: 16 rows of up to 128 bytes, and 16 between them.
#define MOE_I8_OUT 128
#define MOE_I8_OUT_BYTES (16 * (MOE_I8_OUT + 16))

// The stages; over them, after the loop, the sums of the waves along K and the rows on their way
// out; the rows' and channels' scales.
template <int BM, int BN, int WM, int WN, int WK, int NBUF>
constexpr int i8_lds_bytes() {
  const int ring = NBUF * (BM + BN) * WK * 128, after = (WK - 1) * BM * BN * 4 + WM * WN * MOE_I8_OUT_BYTES;
  return (ring > after ? ring : after) + 4 * (BM + BN);
}

// Row `row` (0..15) of a wave's channel tile j is this column of its output
// columns.  SwiGLU: gate and up tiles alternate (one tile alone holds 8 rows of
// each).  The 4 rows that a lane holds of two output tiles are 8 columns side by
// side, and the lane stores them at once; a last tile without a partner is in order.
template <int NI>
__device__ __forceinline__ int i8_column(int swiglu, int j, int row) {
  if (swiglu && NI == 1) return row % 8;
  const int o = swiglu ? j / 2 : j, outs = swiglu ? NI / 2 : NI;
  return outs % 2 && o == outs - 1 ? o * 16 + row : o / 2 * 32 + 8 * (row / 4) + 4 * (o & 1) + row % 4;
}
template <int NI>
__device__ __forceinline__ bool i8_is_up(int j, int row) { return NI == 1 ? row >= 8 : j & 1; }

// 16 rows x COLS columns of T that a wave holds (`value`: part p's V columns of this
// lane, from column 4 V p + V (lane / 16) of its row lane % 16 on) to out's rows r0
// on, columns c0 on; `rows` and `left` of them exist.  Through LDS, 128 bytes of a row
// at a time: a lane's columns are one row's, and neighbouring lanes hold other rows;
// stored from there, a quad of lanes touches 4 rows (256 KiB of f32 took 20 thousand
// cycles that way, 15 so).
template <typename T, int COLS, int V, typename F>
__device__ __forceinline__ void i8_rows_out(T *out, int8_t *reg, int lane, size_t r0, int rows, int pitch, int c0, int left,
                                            F value) {
  constexpr int ES = sizeof(T), RUN = COLS * ES < MOE_I8_OUT ? COLS : MOE_I8_OUT / ES;  // columns at a time
  constexpr int ROW = RUN * ES + 16, PIECES = RUN * ES / 16, PARTS = RUN < 4 * V ? 1 : RUN / (4 * V);
  typedef T quad_t __attribute__((ext_vector_type(4)));
  typedef T piece_t __attribute__((ext_vector_type(16 / ES)));
  typedef T any_t __attribute__((ext_vector_type(16 / ES), aligned(ES)));
  const int fr = lane & 15, fg = lane >> 4;
#pragma unroll
  for (int n = 0; n < COLS / RUN; n++) {
    asm volatile("" ::: "memory");
#pragma unroll
    for (int p = 0; p < PARTS; p++) {
      float f[V];
      value(n * PARTS + p, f);
      if (RUN < 4 * V && fg >= RUN / V) continue;  // (one tile of 8 gate and 8 up rows: two lane groups hold them)
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        quad_t w;
#pragma unroll
        for (int v = 0; v < 4; v++) w[v] = (T)f[q + v];
        *reinterpret_cast<quad_t *>(reg + fr * ROW + (p * 4 * V + fg * V + q) * ES) = w;
      }
    }
    asm volatile("" ::: "memory");
#pragma unroll
    for (int u0 = 0; u0 < 16 * PIECES; u0 += 64) {
      const int u = u0 + lane, r = u / PIECES, c = n * RUN + u % PIECES * (16 / ES);
      if (16 * PIECES % 64 && u >= 16 * PIECES) break;
      if (r >= rows || c >= left) continue;
      const piece_t w = *reinterpret_cast<const piece_t *>(reg + r * ROW + u % PIECES * 16);
      T *to = out + (r0 + r) * (size_t)pitch + c0 + c;
      if (c + 16 / ES <= left) {
        *reinterpret_cast<any_t *>(to) = w;
      } else {
#pragma unroll
        for (int v = 0; v < 16 / ES; v++)
          if (c + v < left) to[v] = w[v];
      }
    }
  }
}

// The rest of k_mm_i8 for one tile; ONCE: no other workgroup reads its weights.
template <int BM, int BN, int WM, int WN, int WK, int NBUF, bool ONCE>
__device__ __forceinline__ void i8_multiply(const i8_mm &a, int nt, const row_tile &t, v4i *lds) {
  constexpr int NW = WM * WN * WK, TM = BM / WM, TN = BN / WN, MI = TM / 16, NI = TN / 16;
  constexpr int STAGE = (BM + BN) * WK * 8;          // 16-byte chunks of a stage
  constexpr int XI = BM * WK / 8, WI = BN * WK / 8;  // 1 KiB loads of a stage
  constexpr int NX = (XI + NW - 1) / NW, NWI = (WI + NW - 1) / NW;
  constexpr int CX = XI / NW, CNT = CX + WI / NW;    // loads of every wave, at least
  constexpr int LDS = i8_lds_bytes<BM, BN, WM, WN, WK, NBUF>();
  float *scales = reinterpret_cast<float *>(lds + LDS / 16) - (BM + BN);  // rows, channels
  static_assert(NI == 1 || NI % 4 == 0 || NI == 2, "output tiles in pairs, or one");
  static_assert(64 * NW >= BM && 64 * NW >= BN, "a thread for each scale");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = wave % WK, wn = wave / WK % WN, wm = wave / (WK * WN);
  const int half = a.N / 2, n_end = a.swiglu ? half : a.N, cols = a.swiglu ? TN / 2 : TN;  // a wave's output columns
  const uint32_t xbytes = (uint32_t)a.n_src * (uint32_t)a.K, wbytes = (uint32_t)a.N * (uint32_t)a.K;
  const int stages = (a.K + 128 * WK - 1) / (128 * WK);

  const int c0 = blockIdx.x % nt * WN * cols;  // the workgroup's first column
  const int8_t *wbase = a.w + (size_t)t.e * a.N * a.K;
  // weight row of channel row j of the tile; past the end where its column does not exist
  auto channel = [&](int j) __attribute__((always_inline)) {
    const int jt = j % TN / 16, c = c0 + j / TN * cols + i8_column<NI>(a.swiglu, jt, j % 16);
    return c < n_end ? (a.swiglu && i8_is_up<NI>(jt, j % 16) ? half + c : c) : a.N;
  };
  // lane offsets of this wave's loads at K 0: row lr of the load's 8, chunk swizzled by it
  const int lr = lane >> 3, lc = (lane & 7) ^ lr;
  uint32_t vx[NX], vw[NWI];
#pragma unroll
  for (int i = 0; i < NWI; i++) {
    const int rr = 8 * (wave + NW * i), w = channel(rr % BN + lr);
    vw[i] = w < a.N ? (uint32_t)w * (uint32_t)a.K + rr / BN * 128 + lc * 16 : MOE_LDS_OOB;
  }
  // loads l of this wave's of stage s, into buffer b: the rows' WK blocks of BM x 128 bytes, then the channels'
  auto load_x = [&](int l, int s, int b) __attribute__((always_inline)) {
    i8_load<BM, XI, NW, false>(l, a.q, xbytes, vx[l], lds + b * STAGE, wave, s * 128 * WK, lc * 16, a.K);
  };
  auto load_w = [&](int l, int s, int b) __attribute__((always_inline)) {
    i8_load<BN, WI, NW, ONCE>(l, wbase, wbytes, vw[l], lds + b * STAGE + BM * WK * 8, wave, s * 128 * WK, lc * 16, a.K);
  };
  // the weights go out before the rows are known (a load and a division away)
#pragma unroll
  for (int s = 0; s < NBUF; s++)
#pragma unroll
    for (int l = 0; l < NWI; l++) load_w(l, s, s);
  const int srow = tid < BM && tid < t.n ? i8_src(a, t.r0 + tid) : -1, schannel = tid < BN ? channel(tid) : a.N;
#pragma unroll
  for (int i = 0; i < NX; i++) {
    const int rr = 8 * (wave + NW * i), row = rr % BM + lr, s = row < t.n ? i8_src(a, t.r0 + row) : -1;
    vx[i] = s >= 0 ? (uint32_t)s * (uint32_t)a.K + rr / BM * 128 + lc * 16 : MOE_LDS_OOB;
  }
  const float row_scale = srow >= 0 ? a.qs[srow] : 0.0f;
  const float channel_scale = schannel < a.N ? a.ws[(size_t)t.e * a.N + schannel] : 0.0f;
#pragma unroll
  for (int s = 0; s < NBUF; s++)
#pragma unroll
    for (int l = 0; l < NX; l++) load_x(l, s, s);
  if (tid < BM) scales[tid] = row_scale;
  if (tid < BN) scales[BM + tid] = channel_scale;

  v4i acc[NI][MI];
  const int fr = lane & 15, fg = lane >> 4;  // this lane's row of an operand, and its chunk of 4
  // Two MFMA steps a stage, 64 bytes of K each; their operands alternate between two sets of
  // registers, a step ahead of the MFMAs (over the stages' border too).
  v4i A[2][NI], B[2][MI];
  // the operands of step kk of the stage in buffer b, in MI parts
  auto read = [&](int i, int set, int b, int kk) __attribute__((always_inline)) {
    const v4i *xb = lds + b * STAGE + (wk * BM + wm * TM + fr) * 8;
    const v4i *wb = lds + b * STAGE + (BM * WK + wk * BN + wn * TN + fr) * 8;
    const int c = (kk * 4 + fg) ^ (fr & 7);
    B[set][i] = xb[i * 128 + c];
#pragma unroll
    for (int j = 0; j < NI; j++)
      if (j * MI / NI == i) A[set][j] = wb[j * 128 + c];
  };
  lds_wait_barrier<(NBUF - 1) * CX>();
#pragma unroll
  for (int i = 0; i < MI; i++) read(i, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < NI; j++)
#pragma unroll
    for (int i = 0; i < MI; i++) acc[j][i] = v4i{0, 0, 0, 0};
  int cur = 0;
#pragma unroll 1
  for (int s = 0; s < stages; s++) {
    const int next = cur + 1 == NBUF ? 0 : cur + 1;
#pragma unroll
    for (int kk = 0; kk < 2; kk++) {
      // Before a stage's last step: the next stage has landed, and every wave
      // holds the rest of this one in registers, so its buffer is free.  (The
      // first NBUF stages' weights were all asked for before their rows.)
      if (kk == 1) {
        if (NBUF > 2 && s < NBUF - 2) lds_wait_barrier<(NBUF - 2) * CX>();
        else lds_wait_barrier<(NBUF - 2) * CNT>();
      }
#pragma unroll
      for (int i = 0; i < MI; i++) {
        read(i, kk ^ 1, kk ? next : cur, kk ^ 1);
#pragma unroll
        for (int j = 0; j < NI; j++) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[kk][j], B[kk][i], acc[j][i], 0, 0, 0);
        // this order, where the compiler would gather a step's LDS reads before the barrier and wait for them there
        __builtin_amdgcn_sched_group_barrier(0x100, 1 + NI / MI, 0);  // LDS reads
        __builtin_amdgcn_sched_group_barrier(0x008, NI, 0);           // MFMA
        // spread between the MFMAs: a wave that waits to issue a load issues nothing else
        if (kk == 1) {
#pragma unroll
          for (int l = 0; l < NWI; l++)
            if (l * MI / NWI == i) load_w(l, s + NBUF, cur);
#pragma unroll
          for (int l = 0; l < NX; l++)
            if (l * MI / NX == i) load_x(l, s + NBUF, cur);
        }
      }
    }
    cur = next;
  }
  if constexpr (WK > 1) {
    lds_wait_barrier<0>();  // the last loads, out of range as they are, have landed: the stages are free
    v4i *part = lds + ((wm * WN + wn) * MI * NI) * 64 + lane;
    if (wk > 0) {
#pragma unroll
      for (int j = 0; j < NI; j++)
#pragma unroll
        for (int i = 0; i < MI; i++) part[((wk - 1) * WM * WN * MI * NI + j * MI + i) * 64] = acc[j][i];
    }
    lds_wait_barrier<0>();
    if (wk > 0) return;
    for (int q = 0; q < WK - 1; q++)
#pragma unroll
      for (int j = 0; j < NI; j++)
#pragma unroll
        for (int i = 0; i < MI; i++) acc[j][i] += part[(q * WM * WN * MI * NI + j * MI + i) * 64];
  } else {
    lds_wait_barrier<0>();
  }

  int8_t *reg = reinterpret_cast<int8_t *>(lds) + (WK - 1) * BM * BN * 4 + (wm * WN + wn) * MOE_I8_OUT_BYTES;
  const int cw = c0 + wn * cols;  // this wave's first column
  const float *sr = scales + wm * TM + fr, *sc = scales + BM + wn * TN + 4 * fg;
  // value v of channel tile j of row tile i, scaled; its 4 channels' scales lie side by side
  auto value = [&](int i, int j, int v, float sx) __attribute__((always_inline)) { return (float)acc[j][i][v] * sx * sc[j * 16 + v]; };
#pragma unroll
  for (int i = 0; i < MI; i++) {
    const int m0 = wm * TM + i * 16, rows = t.n - m0 < 16 ? t.n - m0 : 16;
    if (rows <= 0) break;
    const float sx = sr[i * 16];
    auto plain = [&](auto width) __attribute__((always_inline)) {
      constexpr int V = decltype(width)::value;
      return [&](int p, float(&f)[V]) __attribute__((always_inline)) {
#pragma unroll
        for (int v = 0; v < V; v++) f[v] = value(i, p * V / 4 + v / 4, v % 4, sx);
      };
    };
    auto gated = [&](auto width) __attribute__((always_inline)) {
      constexpr int V = decltype(width)::value;
      return [&](int p, float(&f)[V]) __attribute__((always_inline)) {
#pragma unroll
        for (int v = 0; v < V; v++) {
          if constexpr (NI == 1) {  // lanes 0-31 hold gate, 32-63 up
            const float y = value(i, 0, v, sx);
            f[v] = i8_swiglu(y, __shfl_xor(y, 32), a.clamp);
          } else {
            const int j = 2 * (p * V / 4 + v / 4);
            f[v] = i8_swiglu(value(i, j, v % 4, sx), value(i, j + 1, v % 4, sx), a.clamp);
          }
        }
      };
    };
    auto to = [&](auto zero) __attribute__((always_inline)) {
      typedef decltype(zero) T;
      T *o = reinterpret_cast<T *>(a.out);
      constexpr int VP = NI % 2 ? 4 : 8, VG = NI < 4 ? 4 : 8;  // columns side by side in a lane
      if (!a.swiglu)
        i8_rows_out<T, TN, VP>(o, reg, lane, t.r0 + m0, rows, n_end, cw, n_end - cw, plain(std::integral_constant<int, VP>{}));
      else
        i8_rows_out<T, TN / 2, VG>(o, reg, lane, t.r0 + m0, rows, n_end, cw, n_end - cw, gated(std::integral_constant<int, VG>{}));
    };
    if (a.out_type == MOE_GGML_F32) to(float{});
    else if (a.out_type == MOE_GGML_F16) to((_Float16)0.0f);
    else to((bf16_t)0.0f);
  }
}

// STREAM: the weights are more than the caches hold from call to call, and tiles that alone read
// their weights read them past the caches.  A kernel of its own: a choice at every
// load would cut the loop into blocks that the compiler schedules one by one.
template <int BM, int BN, int WM, int WN, int WK, int NBUF, bool STREAM>
__global__ __launch_bounds__(64 * WM * WN * WK) void k_mm_i8(i8_mm a, int nt) {
  // one dynamic array: for a static one the compiler would make every LDS read wait for every load in flight
  extern __shared__ v4i lds[];
  const row_tile t = i8_find_tile(a, blockIdx.x / nt, BM);
  if (t.e < 0) return;
  if (STREAM && t.only) i8_multiply<BM, BN, WM, WN, WK, NBUF, true>(a, nt, t, lds);
  else i8_multiply<BM, BN, WM, WN, WK, NBUF, false>(a, nt, t, lds);
}
