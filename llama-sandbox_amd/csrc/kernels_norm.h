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

template <typename F>
__device__ __forceinline__ double wave_reduce_d(double v, F f) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = f(v, __shfl_xor(v, off));
  return v;
}

// Over a workgroup of WAVES waves; every thread gets it.  part: WAVES doubles, read before the
// next use only after a barrier of the caller's.
template <int WAVES, typename F>
__device__ __forceinline__ double block_reduce_d(double v, double *part, F f) {
  v = wave_reduce_d(v, f);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int i = 1; i < WAVES; i++) v = f(v, part[i]);
  return v;
}

// NaN wins: a row that holds one has no largest value.
__device__ __forceinline__ double max_nan(double a, double b) { return a > b || a != a ? a : b; }

// A row's 8-bit scale from its largest |y|; what has none (NaN, infinity) gets NaN.
__device__ __forceinline__ float norm_scale(double amax) {
  const float s = (float)(amax / 127.0);
  return s < INFINITY ? s : __builtin_nanf("");
}
__device__ __forceinline__ int8_t norm_code(double y, float s) {
  if (!(s > 0.0f)) return 0;
  return (int8_t)fmin(fmax(__builtin_rint(y / (double)s), -127.0), 127.0);
}

// One workgroup a row, three passes over it.
__global__ __launch_bounds__(256) void k_rms_norm_any(norm_call a) {
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
  sum = block_reduce_d<4>(sum, part[0], [](double p, double q) { return p + q; });
  const double r = 1.0 / sqrt(sum / a.H + (double)a.eps);
  if (a.rstd && tid == 0) a.rstd[blockIdx.x] = (float)r;
  if (a.y)
    for (int i = tid; i < a.H; i += 256)
      store_any(a.y, a.y_type, at + i, load_any(hp, ht, at + i) * (float)r * load_any(a.w, a.w_type, i));
  if (!a.q) return;
  double m = 0.0;
  for (int i = tid; i < a.H; i += 256) m = max_nan(m, fabs((double)load_any(hp, ht, at + i) * (double)load_any(a.w, a.w_type, i)));
  m = block_reduce_d<4>(m, part[1], max_nan);
  const float s = norm_scale(m * r);
  if (tid == 0) a.scale[blockIdx.x] = s;
  for (int i = tid; i < a.H; i += 256)
    a.q[at + i] = norm_code((double)load_any(hp, ht, at + i) * (double)load_any(a.w, a.w_type, i) * r, s);
}

// dx of one row a workgroup.
__global__ __launch_bounds__(256) void k_rms_norm_dx_any(norm_grad_call a) {
  __shared__ double part[4];
  const size_t at = (size_t)blockIdx.x * a.H;
  const int tid = threadIdx.x;
  const float r = a.rstd[blockIdx.x];
  double sum = 0.0;
  for (int i = tid; i < a.H; i += 256) {
    const float g = load_any(a.dy, a.dy_type, at + i) * load_any(a.w, a.w_type, i);
    sum = fma((double)g, (double)(load_any(a.h, a.h_type, at + i) * r), sum);
  }
  sum = block_reduce_d<4>(sum, part, [](double p, double q) { return p + q; });
  const float c = (float)(sum / a.H);
  for (int i = tid; i < a.H; i += 256) {
    const float g = load_any(a.dy, a.dy_type, at + i) * load_any(a.w, a.w_type, i);
    float d = r * fmaf(-(load_any(a.h, a.h_type, at + i) * r), c, g);
    if (a.dres) d += load_any(a.dres, a.dx_type, at + i);
    store_any(a.dx, a.dx_type, at + i, d);
  }
}

// dw of 64 columns a workgroup: wave v takes rows v, v + 4, ...
__global__ __launch_bounds__(256) void k_rms_norm_dw_any(norm_grad_call a) {
  __shared__ float part[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = blockIdx.x * 64 + lane;
  float sum = 0.0f;
  if (i < a.H)
    for (int t = wave; t < a.T; t += 4)
      sum = fmaf(load_any(a.dy, a.dy_type, (size_t)t * a.H + i), load_any(a.h, a.h_type, (size_t)t * a.H + i) * a.rstd[t], sum);
  part[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && i < a.H) a.dw[i] = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
}
