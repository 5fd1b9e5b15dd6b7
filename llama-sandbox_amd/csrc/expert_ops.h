// Operators around the expert products: dispatch, combine and their
// gradients, rows quantised to 8 bits and 8-bit products (host code, included
// by moe_block.hip after what it uses).
//
// Nothing here allocates device memory, keeps a call's data or synchronises: a call
// is one launch on the caller's stream, so calls may overlap on several streams,
// threads and captured graphs as long as their buffers do not.  What they
// change in the context, its last message and the profiler's lists, is under moe_ctx::mu.
#pragma once

// The context's device for one call; the caller's current device afterwards.
struct device_scope {
  int prev = -1;
  hipError_t err;
  explicit device_scope(int device) {
    err = hipGetDevice(&prev);
    if (err == hipSuccess && prev != device) err = hipSetDevice(device);
    else prev = -1;
  }
  ~device_scope() {
    if (prev >= 0) (void)hipSetDevice(prev);
  }
};

#define MOE_ROW_MAX (1 << 30)  // elements of a row: indexes within one stay in 32 bits

static size_t type_bytes(int t) { return t == MOE_GGML_F32 ? 4 : t == MOE_GGML_F16 || t == MOE_GGML_BF16 ? 2 : 0; }

// p holds elements of size b (b = 0: an unknown type).
static bool is_array(const void *p, size_t b) { return p && b && (uintptr_t)p % b == 0; }

// A buffer of a call: what is written may overlap nothing else.
struct call_buf {
  const void *p;
  size_t bytes;
  bool written;
};
static bool overlap(std::initializer_list<call_buf> bufs) {
  for (const call_buf &a : bufs)
    for (const call_buf &b : bufs)
      if (&a != &b && a.written && a.p && b.p && (uintptr_t)a.p < (uintptr_t)b.p + b.bytes &&
          (uintptr_t)b.p < (uintptr_t)a.p + a.bytes)
        return true;
  return false;
}

extern "C" moe_status moe_dispatch(moe_ctx *c, const void *x, int x_type, const int32_t *inv, int T, int k, int H,
                                   int n_rows, void *rows, int rows_type, void *stream) {
  if (!c) return MOE_ERR_INVALID_ARG;
  if (!is_array(x, type_bytes(x_type)) || !is_array(rows, type_bytes(rows_type)) || !is_array(inv, 4) || T <= 0 ||
      k <= 0 || k > 64 || H <= 0 || H > MOE_ROW_MAX || n_rows <= 0)
    return fail(c, MOE_ERR_INVALID_ARG, "moe_dispatch: bad arguments");
  if (overlap({{x, (size_t)T * H * type_bytes(x_type), false}, {inv, (size_t)T * k * 4, false},
               {rows, (size_t)n_rows * H * type_bytes(rows_type), true}}))
    return fail(c, MOE_ERR_INVALID_ARG, "moe_dispatch: rows overlaps another buffer");
  device_scope ds(c->device);
  HIPC(c, ds.err);
  {
    prof_scope ps(c, K_DISPATCH, (hipStream_t)stream, true);
    if (!launch_dispatch(x, x_type, inv, T, k, H, n_rows, rows, rows_type, (hipStream_t)stream))
      return fail(c, MOE_ERR_UNSUPPORTED, "moe_dispatch: T = %d tokens", T);
  }
  HIPC(c, hipGetLastError());
  return MOE_OK;
}

static moe_status combine_rows(moe_ctx *c, const char *who, const void *rows, int rows_type, int n_rows, const float *wts,
                               const int32_t *inv, int T, int k, int H, void *out, int out_type, hipStream_t st) {
  if (!is_array(rows, type_bytes(rows_type)) || !is_array(out, type_bytes(out_type)) || !is_array(inv, 4) ||
      (wts && !is_array(wts, 4)) || T <= 0 || k <= 0 || k > 64 || H <= 0 || H > MOE_ROW_MAX ||
      n_rows <= 0)
    return fail(c, MOE_ERR_INVALID_ARG, "%s: bad arguments", who);
  if (overlap({{rows, (size_t)n_rows * H * type_bytes(rows_type), false}, {wts, (size_t)T * k * 4, false},
               {inv, (size_t)T * k * 4, false}, {out, (size_t)T * H * type_bytes(out_type), true}}))
    return fail(c, MOE_ERR_INVALID_ARG, "%s: the output overlaps another buffer", who);
  device_scope ds(c->device);
  HIPC(c, ds.err);
  {
    prof_scope ps(c, K_COMBINE_ROWS, st, true);
    if (!launch_combine_rows(rows, rows_type, n_rows, wts, inv, T, k, H, out, out_type, st))
      return fail(c, MOE_ERR_UNSUPPORTED, "%s: T = %d tokens", who, T);
  }
  HIPC(c, hipGetLastError());
  return MOE_OK;
}

extern "C" moe_status moe_combine(moe_ctx *c, const void *rows, int rows_type, int n_rows, const float *wts,
                                  const int32_t *inv, int T, int k, int H, void *out, int out_type, void *stream) {
  if (!c) return MOE_ERR_INVALID_ARG;
  if (!wts) return fail(c, MOE_ERR_INVALID_ARG, "moe_combine: bad arguments");
  return combine_rows(c, "moe_combine", rows, rows_type, n_rows, wts, inv, T, k, H, out, out_type, (hipStream_t)stream);
}

extern "C" moe_status moe_dispatch_grad(moe_ctx *c, const void *drows, int drows_type, int n_rows, const int32_t *inv,
                                        int T, int k, int H, void *dx, int dx_type, void *stream) {
  if (!c) return MOE_ERR_INVALID_ARG;
  return combine_rows(c, "moe_dispatch_grad", drows, drows_type, n_rows, nullptr, inv, T, k, H, dx, dx_type,
                      (hipStream_t)stream);
}

extern "C" moe_status moe_combine_grad(moe_ctx *c, const void *dout, int dout_type, const void *rows, int rows_type,
                                       int n_rows, const float *wts, const int32_t *inv, int T, int k, int H,
                                       void *drows, float *dwts, void *stream) {
  if (!c) return MOE_ERR_INVALID_ARG;
  const size_t rb = type_bytes(rows_type);
  if (!is_array(dout, type_bytes(dout_type)) || !is_array(rows, rb) || !is_array(drows, rb) || !is_array(wts, 4) ||
      !is_array(inv, 4) || !is_array(dwts, 4) || T <= 0 || k <= 0 || k > 64 || H <= 0 || H > MOE_ROW_MAX ||
      n_rows <= 0)
    return fail(c, MOE_ERR_INVALID_ARG, "moe_combine_grad: bad arguments");
  const size_t nr = (size_t)n_rows * H * rb, np = (size_t)T * k * 4;
  if (overlap({{dout, (size_t)T * H * type_bytes(dout_type), false}, {rows, nr, false}, {wts, np, false}, {inv, np, false},
               {drows, nr, true}, {dwts, np, true}}))
    return fail(c, MOE_ERR_INVALID_ARG, "moe_combine_grad: an output overlaps another buffer");
  device_scope ds(c->device);
  HIPC(c, ds.err);
  {
    prof_scope ps(c, K_COMBINE_GRAD, (hipStream_t)stream, true);
    if (!launch_combine_grad(dout, dout_type, rows, rows_type, n_rows, wts, inv, T, k, H, drows, dwts, (hipStream_t)stream))
      return fail(c, MOE_ERR_UNSUPPORTED, "moe_combine_grad: T = %d tokens of %d slots", T, k);
  }
  HIPC(c, hipGetLastError());
  return MOE_OK;
}

extern "C" moe_status moe_quantize_i8(moe_ctx *c, const void *x, int x_type, int M, int K, int8_t *q, float *scale,
                                      void *stream) {
  if (!c) return MOE_ERR_INVALID_ARG;
  if (!is_array(x, type_bytes(x_type)) || !q || !is_array(scale, 4) || M <= 0 || K <= 0 || K > MOE_ROW_MAX)
    return fail(c, MOE_ERR_INVALID_ARG, "moe_quantize_i8: bad arguments");
  if (overlap({{x, (size_t)M * K * type_bytes(x_type), false}, {q, (size_t)M * K, true}, {scale, (size_t)M * 4, true}}))
    return fail(c, MOE_ERR_INVALID_ARG, "moe_quantize_i8: an output overlaps another buffer");
  device_scope ds(c->device);
  HIPC(c, ds.err);
  {
    prof_scope ps(c, K_QUANT_I8, (hipStream_t)stream, true);
    if (!launch_quantize_i8(x, x_type, M, K, q, scale, c->n_cu, (hipStream_t)stream))
      return fail(c, MOE_ERR_UNSUPPORTED, "moe_quantize_i8: M = %d rows", M);
  }
  HIPC(c, hipGetLastError());
  return MOE_OK;
}

extern "C" moe_status moe_matmul_i8(moe_ctx *c, const int8_t *q, const float *q_scale, int n_src, const int8_t *w,
                                    const float *w_scale, int E, const int32_t *offsets, const int32_t *perm, int k, int M,
                                    int N, int K, uint32_t flags, float clamp, void *out, int out_type, void *stream) {
  if (!c) return MOE_ERR_INVALID_ARG;
  const int swiglu = (flags & MOE_MM_SWIGLU) ? 1 : 0;
  if (!q || !is_array(q_scale, 4) || !w || !is_array(w_scale, 4) || (offsets && !is_array(offsets, 4)) ||
      (perm && !is_array(perm, 4)) || !is_array(out, type_bytes(out_type)) || (flags & ~MOE_MM_SWIGLU) || n_src <= 0 ||
      E <= 0 || E > MOE_GROUP_MAX_E || (!offsets && E != 1) || k <= 0 || (!perm && (k != 1 || n_src < M)) || M <= 0 ||
      N <= 0 || N > MOE_ROW_MAX || K <= 0 || (swiglu && N % 2) || !(clamp >= 0.0f))
    return fail(c, MOE_ERR_INVALID_ARG, "moe_matmul_i8: bad arguments");
  const size_t n_out = (size_t)M * (swiglu ? N / 2 : N) * type_bytes(out_type);
  if (overlap({{q, (size_t)n_src * K, false}, {q_scale, (size_t)n_src * 4, false}, {w, (size_t)E * N * K, false},
               {w_scale, (size_t)E * N * 4, false}, {offsets, ((size_t)E + 1) * 4, false}, {perm, (size_t)M * 4, false},
               {out, n_out, true}}))
    return fail(c, MOE_ERR_INVALID_ARG, "moe_matmul_i8: out overlaps another buffer");
  if (K > MOE_I8_MAX_K)
    return fail(c, MOE_ERR_UNSUPPORTED, "moe_matmul_i8: K = %d: sums of more than %d products can pass 32 bits", K,
                MOE_I8_MAX_K);
  if (M > MOE_I8_MAX_M) return fail(c, MOE_ERR_UNSUPPORTED, "moe_matmul_i8: M = %d rows, at most %d", M, MOE_I8_MAX_M);
  const i8_mm a = {q, q_scale, w, w_scale, offsets, perm, out, n_src, E, k, M, N, K, swiglu, out_type, clamp};
  device_scope ds(c->device);
  HIPC(c, ds.err);
  {
    prof_scope ps(c, K_MM_I8, (hipStream_t)stream, true);
    if (!launch_matmul_i8(a, c->n_cu, (hipStream_t)stream))
      return fail(c, MOE_ERR_UNSUPPORTED, "moe_matmul_i8: M = %d rows of N = %d channels", M, N);
  }
  HIPC(c, hipGetLastError());
  return MOE_OK;
}
