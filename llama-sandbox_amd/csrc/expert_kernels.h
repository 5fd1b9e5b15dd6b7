// expert_kernels.h -- launches of expert_kernels.hip, for expert_ops.h.  Arguments are
// checked there; false: more rows than a grid takes; a launch error is left for
// hipGetLastError.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#define MOE_I8_MAX_K 131071          // K * 128 * 128 < 2^31: sums are exact in int32
#define MOE_I8_MAX_M ((1 << 30) - 1) // rows of a product: a tile's first row and last stay in 32 bits

// One call of moe_matmul_i8.  Grouped: offsets [E+1] cut the M rows by expert;
// perm: row r's codes are those of source row perm[r] / k (NULL: row r itself).
// SwiGLU: the N channels are N/2 of gate, then N/2 of up, and out has N/2 columns.
struct i8_mm {
  const int8_t *q;
  const float *qs;
  const int8_t *w;
  const float *ws;
  const int32_t *offsets, *perm;
  void *out;
  int n_src, E, k, M, N, K, swiglu, out_type;
  float clamp;
  int stream = 0;  // set by the launch: a weight that one tile alone reads goes past the caches
};

// element types: moe_block.h's MOE_GGML_F32 / F16 / BF16
bool launch_dispatch(const void *x, int x_type, const int32_t *inv, int T, int k, int H, int n_rows, void *rows,
                     int rows_type, hipStream_t st);
bool launch_combine_rows(const void *rows, int rows_type, int n_rows, const float *wts, const int32_t *inv, int T, int k,
                         int H, void *out, int out_type, hipStream_t st);  // wts NULL: unit weights
bool launch_combine_grad(const void *dout, int dout_type, const void *rows, int rows_type, int n_rows, const float *wts,
                         const int32_t *inv, int T, int k, int H, void *drows, float *dwts, hipStream_t st);
bool launch_quantize_i8(const void *x, int x_type, int M, int K, int8_t *q, float *scale, int n_cu, hipStream_t st);
bool launch_matmul_i8(const i8_mm &a, int n_cu, hipStream_t st);
