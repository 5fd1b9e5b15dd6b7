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

// A row's codes in one pass: WPR waves hold it in registers, VPT vectors of 8 a
// thread (K <= 512 WPR VPT); 256 / (64 WPR) rows a workgroup where WPR < 4.
// Memory bound (2 to 4 bytes in, 1 out) only while the codes are cheap: a
// quotient x * inv is within 1.6e-5 of x / s, so it decides all but those next
// to a tie, and the exact comparison runs only for waves that hold one (about
// one vector in ten).
template <typename T, int WPR, int VPT>
__global__ __launch_bounds__(WPR < 4 ? 256 : 64 * WPR) void k_quantize_i8(const T *__restrict__ x, int M, int K,
                                                                          int8_t *__restrict__ q, float *__restrict__ scale) {
  constexpr int RPW = WPR < 4 ? 4 / WPR : 1;  // rows a workgroup
  __shared__ uint32_t part[WPR < 4 ? 4 : WPR];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, in_row = tid % (64 * WPR);
  const long row = (long)blockIdx.x * RPW + wave / WPR;
  const T *xr = x + (row < M ? row : 0) * K;
  float f[VPT][8];
  uint32_t m = 0;
#pragma unroll
  for (int v = 0; v < VPT; v++) {
    const int c = (in_row + v * 64 * WPR) * 8;
    load_v<T, 8>(xr + c, row < M ? K - c : 0, f[v]);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t b = __builtin_bit_cast(uint32_t, f[v][i]) & 0x7fffffffu;
      m = b > m ? b : m;
    }
  }
  m = wave_max_u(m);
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
    const int c = (in_row + v * 64 * WPR) * 8;
    if (c >= K) break;
    int8_t code[8];
    bool near = w.pre != 1.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float t = f[v][i] * w.inv, r = __builtin_rintf(t);
      near |= fabsf(t - r) > 0.4999f;
      code[i] = (int8_t)(int)r;
    }
    if (__any(near)) {
#pragma unroll
      for (int i = 0; i < 8; i++) code[i] = (int8_t)i8_code_in(w, f[v][i]);
    }
    typedef int8_t c8 __attribute__((ext_vector_type(8), aligned(1)));
    int8_t *to = q + row * K + c;
    if (c + 8 <= K) {
      c8 o;
#pragma unroll
      for (int i = 0; i < 8; i++) o[i] = code[i];
      *reinterpret_cast<c8 *>(to) = o;
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (c + i < K) to[i] = code[i];
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

// The rows of one tile: expert e (-1: none left), rows [r0, r0 + n).
struct i8_tile {
  int e, r0, n;
};

// Tile `item` of the grouped rows cut into tiles of at most BM: expert e has
// ceil(c_e / BM) of them, in expert order.  Every wave finds it for itself,
// 64 experts at a time (E <= 1024: all offsets are asked for at once), with a
// scan over the lanes.  Offsets are held to [0, M].
__device__ __forceinline__ i8_tile i8_find_tile(const i8_mm &a, int item, int BM) {
  if (!a.offsets) {
    const int r0 = item * BM;
    return {r0 < a.M ? 0 : -1, r0, a.M - r0 < BM ? a.M - r0 : BM};
  }
  const int lane = threadIdx.x & 63;
  int lo[16], hi[16];
#pragma unroll
  for (int j = 0; j < 16; j++)
    if (64 * j < a.E) {
      const int e = min(64 * j + lane, a.E - 1);
      lo[j] = a.offsets[e];
      hi[j] = a.offsets[e + 1];
    }
  int first = 0;
#pragma unroll
  for (int j = 0; j < 16; j++)
    if (64 * j < a.E) {
      const int l = min(max(lo[j], 0), a.M), h = min(max(hi[j], 0), a.M);
      const int c = 64 * j + lane < a.E && h > l ? (h - l + BM - 1) / BM : 0;
      int sum = c;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(sum, o);
        if (lane >= o) sum += u;
      }
      const int at = first + sum - c;
      const uint64_t here = __ballot(at <= item && item < at + c);
      if (here) {
        const int r0 = l + (item - at) * BM, n = h - r0 < BM ? h - r0 : BM;
        const int owner = __ffsll((unsigned long long)here) - 1;
        return {64 * j + owner, __builtin_amdgcn_readlane(r0, owner), __builtin_amdgcn_readlane(n, owner)};
      }
      first += __builtin_amdgcn_readlane(sum, 63);
    }
  return {-1, 0, 0};
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

// Any K and alignment: tiles of 64 rows x 64 channels, 64 bytes of K a step
// through registers into LDS.  Wave (wm, wn) multiplies 32 rows with two
// 16-channel tiles, wn*16 of each half of the 64 (SwiGLU: the halves are gate
// and up, so a lane holds both of its channels).
// 16x16x64 MFMA, weights as A, rows as B: lane l holds K bytes [16 (l/16), +16)
// of A row (B column) l % 16; D lane l holds column l % 16, rows 4 (l/16) + i.
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
          i8_store(a, r, n, i8_swiglu((float)acc[0][j][i] * sx * wsc[n], (float)acc[1][j][i] * sx * wsc[half + n], a.clamp));
      } else {
        if (n0 + nl < n_end) i8_store(a, r, n0 + nl, (float)acc[0][j][i] * sx * wsc[n0 + nl]);
        if (n0 + 32 + nl < n_end) i8_store(a, r, n0 + 32 + nl, (float)acc[1][j][i] * sx * wsc[n0 + 32 + nl]);
      }
    }
  }
}

// ---- staged tiles -------------------------------------------------------------------
//
// K % 16 == 0 and 16-byte aligned rows.  A workgroup multiplies BM rows with BN
// channels; both go to LDS by direct loads, 128 bytes of K a row, NBUF stages
// around.  A 1 KiB load is 8 rows; the 16-byte chunk c of row r lies at c ^ (r & 7),
// so the 16 or 32 rows that an MFMA operand reads at one chunk fall on all banks.
// Waves: WM x WN over the tile, and WK over K (wave k takes every WK-th 128
// bytes; the sums meet in LDS after the loop).
// MF x MF MFMA with the rows as A and the channels as B: a D lane holds one
// channel (gate and up of one column are in one lane: the wave's channel tiles
// alternate) and 4 consecutive rows an element quad.
#define MOE_I8_OOB 0xffffff00u  // a lane offset past any buffer: the load returns 0
#define MOE_I8_RSRC 0x00020000  // raw buffer, 32-bit dwords, no swizzle

template <int MF>
struct i8_frag;
template <>
struct i8_frag<16> {
  typedef v4i acc_t;
  static constexpr int KC = 4, NACC = 4;  // 16-byte chunks of K an MFMA takes; values a lane holds
  static __device__ __forceinline__ acc_t mfma(v4i a, v4i b, acc_t c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ int row(int lane, int i) { return 4 * (lane >> 4) + i; }
};
template <>
struct i8_frag<32> {
  typedef v16i acc_t;
  static constexpr int KC = 2, NACC = 16;
  static __device__ __forceinline__ acc_t mfma(v4i a, v4i b, acc_t c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ int row(int lane, int i) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }
};

// Waits for vmcnt <= n only (gfx9 encoding), then for every wave's LDS reads.
template <int N>
__device__ __forceinline__ void i8_wait_barrier() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x70 | 0xF00);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 64 lanes' 16 bytes at base + vo + so into the 1 KiB at buf.
__device__ __forceinline__ void i8_dma(const int8_t *base, uint32_t bytes, v4i *buf, uint32_t vo, uint32_t so) {
  typedef __attribute__((address_space(3))) void *lds_t;
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)bytes, MOE_I8_RSRC);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_t)buf, 16, vo, so, 0, 0);
}

// This wave's share of the N_LOAD 1 KiB loads of `span` bytes of K, from k0 on, of
// R rows a 128-byte block: loads wave, wave + NW, ...  vo: lane offsets at K 0.
// Lanes past K, and every lane of a stage past the end, are out of range: they
// read 0, and the waits can count on the loads.
template <int R, int N_LOAD, int NW>
__device__ __forceinline__ void i8_stage(const int8_t *base, uint32_t bytes, const uint32_t (&vo)[(N_LOAD + NW - 1) / NW],
                                         v4i *buf, int wave, int k0, int span, int k_lane, int K) {
  constexpr int N = (N_LOAD + NW - 1) / NW;
  if (k0 + span <= K) {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (N_LOAD % NW == 0 || wave + NW * i < N_LOAD) i8_dma(base, bytes, buf + (wave + NW * i) * 64, vo[i], k0);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++)
      if (N_LOAD % NW == 0 || wave + NW * i < N_LOAD) {
        const int u = wave + NW * i;
        i8_dma(base, bytes, buf + u * 64, k0 + 8 * u / R * 128 + k_lane < K ? vo[i] : MOE_I8_OOB, k0 < K ? k0 : 0);
      }
  }
}

// Floats from a row to the next in a wave's region of LDS on the way out.
template <int TN>
constexpr int i8_out_stride() { return TN + 4; }

// The stages; then, over them, the sums of the waves along K and each wave's rows on their way out; the rows' scales.
template <int BM, int BN, int WM, int WN, int WK, int NBUF, int MF>
constexpr int i8_lds_bytes() {
  const int ring = NBUF * (BM + BN) * WK * 128, part = (WK - 1) * BM * BN * 4 + WM * WN * MF * i8_out_stride<BN / WN>() * 4;
  return (ring > part ? ring : part) + 4 * BM;
}

template <int BM, int BN, int WM, int WN, int WK, int NBUF, int MF, int OCC>
__global__ __launch_bounds__(64 * WM * WN * WK, OCC) void k_mm_i8(i8_mm a, int nt) {
  typedef i8_frag<MF> F;
  constexpr int NW = WM * WN * WK, TM = BM / WM, TN = BN / WN, MI = TM / MF, NI = TN / MF;
  constexpr int STAGE = (BM + BN) * WK * 8;                     // 16-byte chunks of a stage
  constexpr int XI = BM * WK / 8, WI = BN * WK / 8;             // 1 KiB loads of a stage
  constexpr int NX = (XI + NW - 1) / NW, NWI = (WI + NW - 1) / NW;
  constexpr int CNT = XI / NW + WI / NW;                        // of every wave, at least
  // one dynamic array: for a static one the compiler would make every LDS read wait for every load in flight
  static_assert(NI % 2 == 0, "gate and up of a column are channel tiles of one wave");
  extern __shared__ v4i lds[];
  float *sxs = reinterpret_cast<float *>(lds + i8_lds_bytes<BM, BN, WM, WN, WK, NBUF, MF>() / 16) - BM;  // the rows' scales
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = wave % WK, wn = wave / WK % WN, wm = wave / (WK * WN);
  const int nb = blockIdx.x % nt;
  const i8_tile t = i8_find_tile(a, blockIdx.x / nt, BM);
  if (t.e < 0) return;
  const int half = a.N / 2, n_end = a.swiglu ? half : a.N;
  // output column of channel row j of the tile, and its weight row
  auto column = [&](int j) {
    const int jj = j % TN;
    return a.swiglu ? nb * (BN / 2) + j / TN * (TN / 2) + jj / (2 * MF) * MF + jj % MF : nb * BN + j;
  };
  auto weight_row = [&](int j) { return a.swiglu && (j % TN / MF & 1) ? half + column(j) : column(j); };

  // lane offsets of this wave's loads: row of the 8, chunk swizzled by it
  const int lr = lane >> 3, lc = (lane & 7) ^ lr;
  uint32_t vx[NX], vw[NWI];
  for (int i = tid; i < BM; i += 64 * NW) {
    const int s = i < t.n ? i8_src(a, t.r0 + i) : -1;
    sxs[i] = s >= 0 ? a.qs[s] : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < NX; i++) {
    const int rr = 8 * (wave + NW * i), row = rr % BM + lr, s = row < t.n ? i8_src(a, t.r0 + row) : -1;
    vx[i] = s >= 0 ? (uint32_t)s * (uint32_t)a.K + rr / BM * 128 + lc * 16 : MOE_I8_OOB;
  }
#pragma unroll
  for (int i = 0; i < NWI; i++) {
    const int rr = 8 * (wave + NW * i), j = rr % BN + lr;
    vw[i] = column(j) < n_end ? (uint32_t)weight_row(j) * (uint32_t)a.K + rr / BN * 128 + lc * 16 : MOE_I8_OOB;
  }
  const int8_t *wbase = a.w + (size_t)t.e * a.N * a.K;
  const uint32_t xbytes = (uint32_t)a.n_src * (uint32_t)a.K, wbytes = (uint32_t)a.N * (uint32_t)a.K;
  const int stages = (a.K + 128 * WK - 1) / (128 * WK);
  typename F::acc_t acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; i++)
#pragma unroll
    for (int j = 0; j < NI; j++) acc[i][j] = typename F::acc_t{};
  const int fr = lane % MF, fg = lane / MF;  // this lane's row of an operand, and which chunk of the MFMA's
  // stage s into buffer b: the rows' WK blocks of BM x 128 bytes, then the channels'
  auto issue = [&](int s, int b) __attribute__((always_inline)) {
    const int k0 = s * 128 * WK;
    i8_stage<BM, XI, NW>(a.q, xbytes, vx, lds + b * STAGE, wave, k0, 128 * WK, lc * 16, a.K);
    i8_stage<BN, WI, NW>(wbase, wbytes, vw, lds + b * STAGE + BM * WK * 8, wave, k0, 128 * WK, lc * 16, a.K);
  };
#pragma unroll
  for (int s = 0; s < NBUF - 1; s++) issue(s, s);
  int cur = 0;
#pragma unroll 1
  for (int s = 0; s < stages; s++) {
    i8_wait_barrier<(NBUF - 2) * CNT>();
    issue(s + NBUF - 1, cur == 0 ? NBUF - 1 : cur - 1);
    const v4i *xb = lds + cur * STAGE + (wk * BM + wm * TM + fr) * 8;
    const v4i *wb = lds + cur * STAGE + (BM * WK + wk * BN + wn * TN + fr) * 8;
#pragma unroll
    for (int kk = 0; kk < 8 / F::KC; kk++) {
      const int c = (kk * F::KC + fg) ^ (fr & 7);
      v4i A[MI], B[NI];
#pragma unroll
      for (int i = 0; i < MI; i++) A[i] = xb[i * MF * 8 + c];
#pragma unroll
      for (int j = 0; j < NI; j++) B[j] = wb[j * MF * 8 + c];
#pragma unroll
      for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NI; j++) acc[i][j] = F::mfma(A[i], B[j], acc[i][j]);
    }
    cur = cur + 1 == NBUF ? 0 : cur + 1;
  }
  if constexpr (WK > 1) {
    i8_wait_barrier<0>();  // the last loads, out of range as they are, have landed: the stages are free
    typename F::acc_t *part = reinterpret_cast<typename F::acc_t *>(lds);
    const int tile = (wm * WN + wn) * MI * NI;
    if (wk > 0) {
#pragma unroll
      for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NI; j++) part[((wk - 1) * WM * WN * MI * NI + tile + i * NI + j) * 64 + lane] = acc[i][j];
    }
    i8_wait_barrier<0>();
    if (wk > 0) return;
    for (int q = 0; q < WK - 1; q++)
#pragma unroll
      for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NI; j++) acc[i][j] += part[(q * WM * WN * MI * NI + tile + i * NI + j) * 64 + lane];
  } else {
    i8_wait_barrier<0>();
  }
  // through LDS a block of MF rows at a time, in a region of the wave's own: a
  // D lane holds one channel, a store wants a row's channels side by side
  float *reg = reinterpret_cast<float *>(lds + (WK > 1 ? (WK - 1) * BM * BN / 4 : 0)) + (wm * WN + wn) * MF * i8_out_stride<TN>();
  const float *ws = a.ws + (size_t)t.e * a.N;
  float sw[NI];
#pragma unroll
  for (int j = 0; j < NI; j++) {
    const int jr = wn * TN + j * MF + fr;
    sw[j] = column(jr) < n_end ? ws[weight_row(jr)] : 0.0f;
  }
  const int wide = a.swiglu ? TN / 2 : TN, c0 = column(wn * TN);  // the wave's columns, and the first
  const int left = n_end - c0 < wide ? n_end - c0 : wide;
#pragma unroll
  for (int i = 0; i < MI; i++) {
    const int m0 = wm * TM + i * MF;
    if (m0 >= t.n) break;
    asm volatile("" ::: "memory");
#pragma unroll
    for (int v = 0; v < F::NACC; v++) {
      const float sx = sxs[m0 + F::row(lane, v)];
      float *to = reg + F::row(lane, v) * i8_out_stride<TN>() + fr;
      if (!a.swiglu) {
#pragma unroll
        for (int j = 0; j < NI; j++) to[j * MF] = (float)acc[i][j][v] * sx * sw[j];
      } else if constexpr (NI > 1) {
#pragma unroll
        for (int j = 0; j < NI; j += 2)
          to[j / 2 * MF] = i8_swiglu((float)acc[i][j][v] * sx * sw[j], (float)acc[i][j + 1][v] * sx * sw[j + 1], a.clamp);
      }
    }
    asm volatile("" ::: "memory");
    const int rows = t.n - m0 < MF ? t.n - m0 : MF, per = wide / 4;
    for (int u = lane; u < rows * per; u += 64) {
      const int r = u / per, c = u % per * 4;
      const float *from = reg + r * i8_out_stride<TN>() + c;
      const float f[4] = {from[0], from[1], from[2], from[3]};
      const size_t at = (size_t)(t.r0 + m0 + r) * n_end + c0 + c;
      if (c >= left) continue;
      if (a.out_type == MOE_GGML_F32) store_v<float, 4>(reinterpret_cast<float *>(a.out) + at, left - c, f);
      else if (a.out_type == MOE_GGML_F16) store_v<_Float16, 4>(reinterpret_cast<_Float16 *>(a.out) + at, left - c, f);
      else store_v<bf16_t, 4>(reinterpret_cast<bf16_t *>(a.out) + at, left - c, f);
    }
  }
}
