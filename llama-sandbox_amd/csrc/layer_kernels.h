// layer_kernels.h -- launches of layer_kernels.hip, for layer_ops.h.  Arguments are
// checked there; false: more rows than a grid takes; a launch error is left for
// hipGetLastError.  Element types: moe_block.h's MOE_GGML_F32 / F16 / BF16.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

// One call of moe_rms_norm; absent operands NULL.
struct norm_call {
  const void *x, *res, *w;
  void *total, *y;
  int8_t *q;
  float *scale, *rstd;
  int x_type, res_type, w_type, y_type, T, H;
  float eps;
  int nt = 0;  // set by the launch: outputs go past the caches
};
bool launch_rms_norm(const norm_call &a, int n_cu, hipStream_t st);

// One call of moe_rms_norm_grad.
struct norm_grad_call {
  const void *dy, *h, *w, *dres;
  const float *rstd;
  void *dx;
  float *dw, *part;
  int dy_type, h_type, w_type, dx_type, T, H;
  int nt = 0;  // set by the launch: dx goes past the caches
};
// Floats of `part` that a call needs, and that every call of at most these sizes can do with.
size_t norm_grad_need(int T, int H, int n_cu);
size_t norm_grad_scratch(int T, int H, int n_cu);
bool launch_rms_norm_grad(const norm_grad_call &a, int n_cu, hipStream_t st);

// One call of moe_route_groups.
struct route_call {
  const void *logits;
  const float *bias;
  int32_t *ids;
  float *wts, *scores;
  int type, T, E, k, mode, n_group, keep, top, norm;
  float scale;
  // set by the launch: experts a group; lanes a group where each takes some; lanes that hold a whole one (0: none do)
  int per = 0, width = 0, lanes = 0;
};
bool launch_route_groups(const route_call &a, hipStream_t st);

// One call of moe_route_grad.
struct route_grad_call {
  const void *logits;
  const int32_t *ids;
  const float *dwts, *dscores;
  void *dlogits;
  int type, out_type, T, E, k, mode, norm;
  float scale;
};
bool launch_route_grad(const route_grad_call &a, hipStream_t st);

// One call of moe_adapters.
struct adapters_call {
  const void *x, *a, *b;
  const float *scale;
  const int32_t *offsets, *perm;
  const void *base;
  void *out;
  float *mid;
  int type, out_type, n, M, K, R, N;
  // set by the launch: shares of mid, elements of K of each, blocks of out's columns, groups of 128 columns in a block;
  // out past the caches
  int splits = 1, piece = 0, col_blocks = 0, col_groups = 1, nt = 0;
};
// As for the gradient: floats of `mid`.
size_t adapters_need(int M, int K, int R, int n_cu);
size_t adapters_scratch(int M, int K, int R, int n_cu);
bool launch_adapters(const adapters_call &a, int n_cu, hipStream_t st);
