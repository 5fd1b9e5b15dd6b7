// kernels_norm.h -- root-mean-square norm of rows, with the residual's addition
// and an output in 8 bits, and its gradient.
//
//   h = x + res (rounded to res's type: what the next layers read is what is normalised)
//   r = (mean h^2 + eps)^-1/2, y = h * r * w
//   8 bits: s = fl32(max |h w| r / 127), q = h w r / s to the nearest whole number, ties to even
//   with u = h r, g = dy w:  dx = r (g - u mean(g u)) + dres,  dw = sum_t dy u
//
// The sum of squares is in 64 bits, so that any finite row has its norm (squares
// of f32 values pass f32's range) and codes do not hang on the order of the sum.
#pragma once

#include "layer_kernels.h"
#include "row_vec.h"
#include "../../include/moe_block.h"

#include <type_traits>

// Element i of a row operand whose type is the same for a whole call: a uniform branch.
__device__ __forceinline__ float load_any(const void *p, int type, size_t i) {
  if (type == MOE_GGML_F32) return reinterpret_cast<const float *>(p)[i];
  if (type == MOE_GGML_F16) return (float)reinterpret_cast<const _Float16 *>(p)[i];
  return (float)reinterpret_cast<const bf16_t *>(p)[i];
}
__device__ __forceinline__ void store_any(void *p, int type, size_t i, float v) {
  if (type == MOE_GGML_F32) reinterpret_cast<float *>(p)[i] = v;
  else if (type == MOE_GGML_F16) reinterpret_cast<_Float16 *>(p)[i] = (_Float16)v;
  else reinterpret_cast<bf16_t *>(p)[i] = (bf16_t)v;
}
__device__ __forceinline__ float round_any(int type, float v) {
  if (type == MOE_GGML_F16) return (float)(_Float16)v;
  if (type == MOE_GGML_BF16) return (float)(bf16_t)v;
  return v;
}

// 8 elements of a row of S bytes each, as they were loaded.  The kernels are made for sizes, and take
// the type at their conversions (a uniform branch): three types of four operands would be 81
// of each.
template <int S>
struct raw8 {
  typedef typename std::conditional<S == 4, float, uint16_t>::type elem;
  raw_v<elem, 8> r;
  __device__ __forceinline__ void load(const void *p, size_t i, int left) { r.load(reinterpret_cast<const elem *>(p) + i, left); }
  __device__ __forceinline__ void get(int type, float (&f)[8]) const {
    if constexpr (S == 4) {
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = r.v[i];
    } else if (type == MOE_GGML_F16) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const uint16_t e = r.v[i];
        f[i] = (float)__builtin_bit_cast(_Float16, e);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = __builtin_bit_cast(float, (uint32_t)r.v[i] << 16);
    }
  }
};
// ... of any type: the gain, read by every row and found in the caches.
__device__ __forceinline__ void load8_any(const void *p, int type, size_t i, int left, float (&f)[8]) {
  if (type == MOE_GGML_F32) {
    raw8<4> r;
    r.load(p, i, left);
    r.get(type, f);
  } else {
    raw8<2> r;
    r.load(p, i, left);
    r.get(type, f);
  }
}
template <bool NT>
__device__ __forceinline__ void store8_type(void *p, int type, size_t i, int left, const float (&f)[8]) {
  if (type == MOE_GGML_F32) store_v<float, 8, NT>(reinterpret_cast<float *>(p) + i, left, f);
  else if (type == MOE_GGML_F16) store_v<_Float16, 8, NT>(reinterpret_cast<_Float16 *>(p) + i, left, f);
  else store_v<bf16_t, 8, NT>(reinterpret_cast<bf16_t *>(p) + i, left, f);
}
// nt: past the caches, the same for a whole call.
__device__ __forceinline__ void store8_any(void *p, int type, size_t i, int left, const float (&f)[8], int nt = 0) {
  if (nt) store8_type<true>(p, type, i, left, f);
  else store8_type<false>(p, type, i, left, f);
}

__device__ __forceinline__ double add_d(double a, double b) { return a + b; }
// NaN wins: a row that holds one has no largest value.
__device__ __forceinline__ double max_nan(double a, double b) { return a > b || a != a ? a : b; }

__device__ __forceinline__ double readlane_d(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Over the LANES lanes (16 or 64) that a lane is one of; every one gets it.
template <int LANES, typename F>
__device__ __forceinline__ double lanes_reduce_d(double v, F f) {
  static_assert(LANES == 16 || LANES == 64, "a row of 16 lanes, or the wave");
  v = f(v, dpp_d<0xB1>(v));   // quad_perm [1,0,3,2]
  v = f(v, dpp_d<0x4E>(v));   // quad_perm [2,3,0,1]
  v = f(v, dpp_d<0x141>(v));  // row_half_mirror
  v = f(v, dpp_d<0x140>(v));  // row_mirror: every lane holds its row of 16's
  if constexpr (LANES == 64) v = f(f(readlane_d(v, 0), readlane_d(v, 16)), f(readlane_d(v, 32), readlane_d(v, 48)));
  return v;
}

// Over the LANES threads of a row.  part: a double for each wave of the workgroup, not used
// again before a barrier of the caller's.
template <int LANES, typename F>
__device__ __forceinline__ double row_reduce_d(double v, double *part, F f) {
  v = lanes_reduce_d<(LANES < 64 ? LANES : 64)>(v, f);
  if constexpr (LANES > 64) {
    constexpr int W = LANES / 64;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) part[wave] = v;
    __syncthreads();
    v = part[wave / W * W];
#pragma unroll
    for (int i = 1; i < W; i++) v = f(v, part[wave / W * W + i]);
  }
  return v;
}

// A row's 8-bit scale from its largest |y|; what has none (NaN, infinity) gets NaN.
__device__ __forceinline__ float norm_scale(double amax) {
  const float s = (float)(amax / 127.0);
  return s < INFINITY ? s : __builtin_nanf("");
}

// A row in one pass: LANES threads hold it in registers, VPT vectors of 8 each (H <= 8 LANES
// VPT); 256 / LANES rows a workgroup where that is more than one.  SX, SR: bytes of an element of x and of the residual
// (0: none).  Bound by memory: 4096 rows of 7168 bf16 with residual (235 MB) 45.7 us, 5.1 TB/s, as a large copy; 512
// rows 7.3; 8191 of 2048 25.6.  To 8 bits the same 4096 rows (205 MB) take 48.1, 4.3 TB/s: products, maxima and codes in
// 64 bits are 14 instructions a value (with 20, 52.5).  One row 3.6 us: a launch, the loads, two barriers.
template <int SX, int SR, int LANES, int VPT>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void k_rms_norm(norm_call a) {
  constexpr int NT = LANES < 256 ? 256 : LANES;
  __shared__ double part[2][NT / 64];
  const int in_row = threadIdx.x % LANES;
  const long row = (long)blockIdx.x * (NT / LANES) + threadIdx.x / LANES;
  const bool there = row < a.T;
  const size_t at = (size_t)(there ? row : 0) * a.H;
  raw8<SX> x[VPT];
  raw8<(SR ? SR : 2)> res[VPT];
#pragma unroll
  for (int v = 0; v < VPT; v++) {
    const int i = (in_row + v * LANES) * 8, left = there ? a.H - i : 0;
    x[v].load(a.x, at + i, left);
    if constexpr (SR != 0) res[v].load(a.res, at + i, left);
  }
  // asked for before the barrier; the longest rows have no registers for it, and read it where it is used
  constexpr bool EARLY = LANES * VPT <= 2048;
  float w_early[EARLY ? VPT : 1][8];
  auto load_w = [&](int v, float(&f)[8]) {
    const int i = (in_row + v * LANES) * 8;
    load8_any(a.w, a.w_type, i, a.H - i, f);
  };
  if constexpr (EARLY) {
#pragma unroll
    for (int v = 0; v < VPT; v++) load_w(v, w_early[v]);
  }
  auto gain = [&](int v, float(&f)[8]) {
    if constexpr (EARLY) {
#pragma unroll
      for (int j = 0; j < 8; j++) f[j] = w_early[v][j];
    } else {
      load_w(v, f);
    }
  };
  float h[VPT][8];
  double sum = 0.0;
#pragma unroll
  for (int v = 0; v < VPT; v++) {
    const int i = (in_row + v * LANES) * 8;
    x[v].get(a.x_type, h[v]);
    if constexpr (SR != 0) {
      float e[8];
      res[v].get(a.res_type, e);
#pragma unroll
      for (int j = 0; j < 8; j++) h[v][j] += e[j];
      if (SR == 2) {
        if (a.res_type == MOE_GGML_F16) {
#pragma unroll
          for (int j = 0; j < 8; j++) h[v][j] = (float)(_Float16)h[v][j];
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) h[v][j] = (float)(bf16_t)h[v][j];
        }
      }
      if (there && i < a.H) store8_any(a.total, a.res_type, at + i, a.H - i, h[v], a.nt);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) sum = fma((double)h[v][j], (double)h[v][j], sum);  // (past the end: 0)
  }
  sum = row_reduce_d<LANES>(sum, part[0], add_d);
  const double r = 1.0 / sqrt(sum / a.H + (double)a.eps);
  if (a.rstd && there && in_row == 0) a.rstd[row] = (float)r;
  if (a.y && there) {
    const float r32 = (float)r;
#pragma unroll
    for (int v = 0; v < VPT; v++) {
      const int i = (in_row + v * LANES) * 8;
      if (i >= a.H) break;
      float y[8], w[8];
      gain(v, w);
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] = h[v][j] * r32 * w[j];
      store8_any(a.y, a.y_type, at + i, a.H - i, y, a.nt);
    }
  }
  if (!a.q) return;
  double m = 0.0;
  // NaN where the gain has a value that is not finite; one of h shows in r, as a NaN or, of an infinity, as 0
  float odd = 0.0f;
#pragma unroll
  for (int v = 0; v < VPT; v++) {
    float w[8];
    gain(v, w);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      m = fmax(m, fabs((double)h[v][j] * (double)w[j]));
      odd = fmaf(w[j], 0.0f, odd);
    }
  }
  m = row_reduce_d<LANES>(odd == odd && r > 0.0 ? m : __builtin_nan(""), part[1], max_nan);
  if (!there) return;
  const float s = norm_scale(m * r);
  if (in_row == 0) a.scale[row] = s;
  const double g = s > 0.0f ? r / (double)s : 0.0;
#pragma unroll
  for (int v = 0; v < VPT; v++) {
    const int i = (in_row + v * LANES) * 8;
    if (i >= a.H) break;
    float w[8];
    gain(v, w);
    uint32_t code[8];
    // + 1.5 * 2^52 rounds to a whole number, ties to even, with it in the low word; past 127 only by a denormal scale
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const double u = fma((double)h[v][j] * (double)w[j], g, 0x1.8p52);
      code[j] = (uint32_t)min(max((int)(uint32_t)__builtin_bit_cast(uint64_t, u), -127), 127);
    }
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2), aligned(1)));
    int8_t *to = a.q + at + i;
    if (!(s > 0.0f)) {
#pragma unroll
      for (int j = 0; j < 8; j++) code[j] = 0;
    }
    if (i + 8 <= a.H) {
      u32x2 o;
#pragma unroll
      for (int k = 0; k < 2; k++)
        o[k] = (code[4 * k] & 255) | (code[4 * k + 1] & 255) << 8 | (code[4 * k + 2] & 255) << 16 | code[4 * k + 3] << 24;
      if (a.nt) __builtin_nontemporal_store(o, reinterpret_cast<u32x2 *>(to));
      else *reinterpret_cast<u32x2 *>(to) = o;
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (i + j < a.H) to[j] = (int8_t)code[j];
    }
  }
}

// Rows too long for registers: one workgroup a row, three passes over it.
__global__ __launch_bounds__(256) void k_rms_norm_long(norm_call a) {
  __shared__ double part[2][4];
  const size_t at = (size_t)blockIdx.x * a.H;
  const int tid = threadIdx.x;
  const void *hp = a.res ? a.total : a.x;
  const int ht = a.res ? a.res_type : a.x_type;
  double sum = 0.0;
  for (int i = tid; i < a.H; i += 256) {
    float h = load_any(a.x, a.x_type, at + i);
    if (a.res) {
      h = round_any(a.res_type, h + load_any(a.res, a.res_type, at + i));
      store_any(a.total, a.res_type, at + i, h);
    }
    sum = fma((double)h, (double)h, sum);
  }
  sum = row_reduce_d<256>(sum, part[0], add_d);
  const double r = 1.0 / sqrt(sum / a.H + (double)a.eps);
  if (a.rstd && tid == 0) a.rstd[blockIdx.x] = (float)r;
  if (a.y)
    for (int i = tid; i < a.H; i += 256)
      store_any(a.y, a.y_type, at + i, load_any(hp, ht, at + i) * (float)r * load_any(a.w, a.w_type, i));
  if (!a.q) return;
  double m = 0.0;
  for (int i = tid; i < a.H; i += 256) m = max_nan(m, fabs((double)load_any(hp, ht, at + i) * (double)load_any(a.w, a.w_type, i)));
  m = row_reduce_d<256>(m, part[1], max_nan);
  const float s = norm_scale(m * r);
  if (tid == 0) a.scale[blockIdx.x] = s;
  const double g = s > 0.0f ? r / (double)s : 0.0;
  for (int i = tid; i < a.H; i += 256) {
    const double y = (double)load_any(hp, ht, at + i) * (double)load_any(a.w, a.w_type, i) * g;
    a.q[at + i] = s > 0.0f ? (int8_t)fmin(fmax(__builtin_rint(y), -127.0), 127.0) : (int8_t)0;
  }
}

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  static_assert(LANES == 16 || LANES == 64, "a row of 16 lanes, or the wave");
  return LANES == 16 ? row16_sum(v) : wave_sum(v);
}

// The gradient in one pass over the rows: LANES threads hold one, G of them a workgroup, which walks
// rows in steps of the grid, with the next row's loads in flight while it sums this one's, and keeps
// its share of dw in registers; k_rms_norm_dw adds the shares up (part: one of H values a workgroup;
// a single workgroup writes dw itself).  SD, SH, SX: bytes of an element of dy, h, dx and dres.
// One workgroup of 1024 threads a CU: two of 512 with two vectors a thread need 148 registers and ran one at a time
// (4096 rows of 7168 bf16 64 us).  Bound by memory: those rows (235 MB, and 7 of shares written and read) 49.6 us and
// 4.8 for the shares; 301 of 2048 f32 5.2 and 2.6, latency; 1000 of 12000 (no row ahead) 39.
template <int SD, int SH, int SX, int LANES, int VPT, int G>
__global__ __launch_bounds__(LANES *G) void k_rms_norm_grad(norm_grad_call a) {
  constexpr int NT = LANES * G, W = LANES > 64 ? LANES / 64 : 1;
  __shared__ float sums[2][NT / 64];
  __shared__ float share[G > 1 ? G : 1][G > 1 ? LANES * 8 + 4 : 1];  // of dw, of the groups
  const int in_row = threadIdx.x % LANES, group = threadIdx.x / LANES, wave = threadIdx.x >> 6;
  const int step = gridDim.x * G;
  // rows of several vectors a thread leave no registers for the gain and the next row
  constexpr bool AHEAD = VPT == 1;
  float w[AHEAD ? VPT : 1][8], acc[VPT][8] = {};
  auto load_w = [&](int v, float(&f)[8]) {
    const int i = (in_row + v * LANES) * 8;
    load8_any(a.w, a.w_type, i, a.H - i, f);
  };
  if constexpr (AHEAD) load_w(0, w[0]);
  raw8<SD> d[VPT];
  raw8<SH> h[VPT];
  raw8<SX> s[VPT];
  float r = 0.0f;
  auto load = [&](long row) {
    const bool there = row < a.T;
    const size_t at = (size_t)(there ? row : 0) * a.H;
    r = there ? a.rstd[row] : 0.0f;
#pragma unroll
    for (int v = 0; v < VPT; v++) {
      const int i = (in_row + v * LANES) * 8, left = there ? a.H - i : 0;
      d[v].load(a.dy, at + i, left);
      h[v].load(a.h, at + i, left);
      if (a.dres) s[v].load(a.dres, at + i, left);
    }
  };
  long row = (long)blockIdx.x * G + group;
  if constexpr (AHEAD) load(row);
  int turn = 0;
  for (long first = (long)blockIdx.x * G; first < a.T; first += step, row += step, turn ^= 1) {
    float g[VPT][8], u[VPT][8], res[VPT][8], dot = 0.0f;
    if constexpr (!AHEAD) load(row);
    const float rr = r;
#pragma unroll
    for (int v = 0; v < VPT; v++) {
      if constexpr (!AHEAD) load_w(v, w[0]);
      d[v].get(a.dy_type, g[v]);
      h[v].get(a.h_type, u[v]);
      if (a.dres) s[v].get(a.dx_type, res[v]);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        u[v][j] *= rr;
        acc[v][j] = fmaf(g[v][j], u[v][j], acc[v][j]);
        g[v][j] *= w[0][j];
        dot = fmaf(g[v][j], u[v][j], dot);
      }
    }
    if constexpr (AHEAD) load(row + step);
    dot = lanes_sum<(LANES < 64 ? LANES : 64)>(dot);
    if constexpr (W > 1) {
      if ((threadIdx.x & 63) == 0) sums[turn][wave] = dot;
      __syncthreads();
      dot = sums[turn][wave / W * W];
#pragma unroll
      for (int i = 1; i < W; i++) dot += sums[turn][wave / W * W + i];
    }
    const float c = dot / (float)a.H;
    if (row < a.T) {
#pragma unroll
      for (int v = 0; v < VPT; v++) {
        const int i = (in_row + v * LANES) * 8;
        if (i >= a.H) break;
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          o[j] = rr * fmaf(-u[v][j], c, g[v][j]);
          if (a.dres) o[j] += res[v][j];
        }
        store8_any(a.dx, a.dx_type, (size_t)row * a.H + i, a.H - i, o, a.nt);
      }
    }
  }
  float *to = gridDim.x > 1 ? a.part + (size_t)blockIdx.x * a.H : a.dw;
#pragma unroll
  for (int v = 0; v < VPT; v++) {
    const int first = v * LANES * 8;
    if constexpr (G == 1) {
      const int i = first + in_row * 8;
      if (i < a.H) store_v<float, 8>(to + i, a.H - i, acc[v]);
    } else {
      if (v > 0) __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; j++) share[group][in_row * 8 + j] = acc[v][j];
      __syncthreads();
      for (int i = threadIdx.x; i < LANES * 8 && first + i < a.H; i += NT) {
        float sum = share[0][i];
        for (int q = 1; q < G; q++) sum += share[q][i];
        to[first + i] = sum;
      }
    }
  }
}

// dw from the n workgroups' shares: 64 columns a workgroup, each of its 16 waves adds 4 shares at once,
// 16 lanes with 4 columns each.
__global__ __launch_bounds__(1024) void k_rms_norm_dw(const float *__restrict__ part, int n, int H, float *__restrict__ dw) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = blockIdx.x * 64 + lane % 16 * 4;
  float sum[4] = {};
#pragma unroll 4
  for (int p = wave * 4 + lane / 16; p < n; p += 64) {
    float f[4];
    load_v<float, 4>(part + (size_t)p * H + i, H - i, f);
#pragma unroll
    for (int j = 0; j < 4; j++) sum[j] += f[j];
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    sum[j] += __shfl_xor(sum[j], 16);
    sum[j] += __shfl_xor(sum[j], 32);
    if (lane < 16) sums[wave][lane * 4 + j] = sum[j];
  }
  __syncthreads();
  if (wave || blockIdx.x * 64 + lane >= H) return;
  float s = sums[0][lane];
#pragma unroll
  for (int q = 1; q < 16; q++) s += sums[q][lane];
  dw[blockIdx.x * 64 + lane] = s;
}

// The gradient of rows too long for registers: dx of one row a workgroup.
__global__ __launch_bounds__(256) void k_rms_norm_dx_long(norm_grad_call a) {
  __shared__ double part[4];
  const size_t at = (size_t)blockIdx.x * a.H;
  const int tid = threadIdx.x;
  const float r = a.rstd[blockIdx.x];
  double sum = 0.0;
  for (int i = tid; i < a.H; i += 256) {
    const float g = load_any(a.dy, a.dy_type, at + i) * load_any(a.w, a.w_type, i);
    sum = fma((double)g, (double)(load_any(a.h, a.h_type, at + i) * r), sum);
  }
  sum = row_reduce_d<256>(sum, part, add_d);
  const float c = (float)(sum / a.H);
  for (int i = tid; i < a.H; i += 256) {
    const float g = load_any(a.dy, a.dy_type, at + i) * load_any(a.w, a.w_type, i);
    float d = r * fmaf(-(load_any(a.h, a.h_type, at + i) * r), c, g);
    if (a.dres) d += load_any(a.dres, a.dx_type, at + i);
    store_any(a.dx, a.dx_type, at + i, d);
  }
}

// dw of 64 columns a workgroup: wave v takes rows v, v + 4, ..., a quarter of all after each other, so the sums are in 64
// bits (in 32 they would be off by up to T / 4 half steps, where k_rms_norm_grad's chains are T / 256 and tens).  Rows
// this long have no fast form: 1000 of 17000 bf16 384 us for dx and dw, as with sums in 32 bits.
__global__ __launch_bounds__(256) void k_rms_norm_dw_long(norm_grad_call a) {
  __shared__ double part[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = blockIdx.x * 64 + lane;
  double sum = 0.0;
  if (i < a.H)
    for (int t = wave; t < a.T; t += 4)
      sum = fma((double)load_any(a.dy, a.dy_type, (size_t)t * a.H + i),
                (double)(load_any(a.h, a.h_type, (size_t)t * a.H + i) * a.rstd[t]), sum);
  part[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && i < a.H) a.dw[i] = (float)((part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]));
}
