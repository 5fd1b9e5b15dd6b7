// Operators on the way into the experts and beside them: the norm of rows with the
// residual's addition, routing with groups, their gradients, and low-rank adapters
// (host code, included by moe_block.hip after expert_ops.h, whose rules hold here
// too: no allocation, no scratch of the context, no synchronisation).
#pragma once

#define MOE_ADAPTERS_MAX 1024      // adapters of a call: moe_group's experts
#define MOE_ADAPTERS_MAX_RANK 1024

extern "C" moe_status moe_rms_norm(moe_ctx *c, const void *x, int x_type, const void *res, void *total, int res_type,
                                   const void *w, int w_type, float eps, int T, int H, void *y, int y_type, int8_t *q,
                                   float *scale, float *rstd, void *stream) {
  if (!c) return MOE_ERR_INVALID_ARG;
  if (!is_array(x, type_bytes(x_type)) || !is_array(w, type_bytes(w_type)) || !res != !total || !q != !scale || (!y && !q) ||
      (res && (!is_array(res, type_bytes(res_type)) || !is_array(total, type_bytes(res_type)))) ||
      (y && !is_array(y, type_bytes(y_type))) || (scale && !is_array(scale, 4)) || (rstd && !is_array(rstd, 4)) || T <= 0 ||
      H <= 0 || H > MOE_ROW_MAX || !(eps >= FLT_MIN && eps <= FLT_MAX))
    return fail(c, MOE_ERR_INVALID_ARG, "moe_rms_norm: bad arguments");
  const size_t n = (size_t)T * H, rb = n * (res ? type_bytes(res_type) : 0);
  if (overlap({{x, n * type_bytes(x_type), false}, {total == res ? nullptr : res, rb, false}, {total, rb, true},
               {w, (size_t)H * type_bytes(w_type), false}, {y, y ? n * type_bytes(y_type) : 0, true}, {q, n, true},
               {scale, (size_t)T * 4, true}, {rstd, (size_t)T * 4, true}}))
    return fail(c, MOE_ERR_INVALID_ARG, "moe_rms_norm: an output overlaps another buffer");
  const norm_call a = {x, res, w, total, y, q, scale, rstd, x_type, res_type, w_type, y_type, T, H, eps};
  device_scope ds(c->device);
  HIPC(c, ds.err);
  {
    prof_scope ps(c, K_RMS_NORM, (hipStream_t)stream, true);
    if (!launch_rms_norm(a, c->n_cu, (hipStream_t)stream))
      return fail(c, MOE_ERR_UNSUPPORTED, "moe_rms_norm: T = %d rows", T);
  }
  HIPC(c, hipGetLastError());
  return MOE_OK;
}

extern "C" size_t moe_rms_norm_grad_scratch(const moe_ctx *c, int T, int H) {
  return c && T > 0 && H > 0 && H <= MOE_ROW_MAX ? norm_grad_scratch(T, H, c->n_cu) : 0;
}

extern "C" moe_status moe_rms_norm_grad(moe_ctx *c, const void *dy, int dy_type, const void *h, int h_type, const void *w,
                                        int w_type, const float *rstd, const void *dres, int T, int H, void *dx, int dx_type,
                                        float *dw, float *part, size_t part_floats, void *stream) {
  if (!c) return MOE_ERR_INVALID_ARG;
  const size_t db = type_bytes(dx_type);
  if (!is_array(dy, type_bytes(dy_type)) || !is_array(h, type_bytes(h_type)) || !is_array(w, type_bytes(w_type)) ||
      !is_array(rstd, 4) || (dres && !is_array(dres, db)) || !is_array(dx, db) || !is_array(dw, 4) || !is_array(part, 4) ||
      T <= 0 || H <= 0 || H > MOE_ROW_MAX)
    return fail(c, MOE_ERR_INVALID_ARG, "moe_rms_norm_grad: bad arguments");
  const size_t n = (size_t)T * H, need = norm_grad_need(T, H, c->n_cu);
  if (part_floats < need)
    return fail(c, MOE_ERR_INVALID_ARG, "moe_rms_norm_grad: part holds %zu floats, this call needs %zu", part_floats, need);
  if (overlap({{dy, n * type_bytes(dy_type), false}, {h, n * type_bytes(h_type), false}, {w, (size_t)H * type_bytes(w_type), false},
               {rstd, (size_t)T * 4, false}, {dres == dx ? nullptr : dres, n * db, false}, {dx, n * db, true},
               {dw, (size_t)H * 4, true}, {part, need * 4, true}}))
    return fail(c, MOE_ERR_INVALID_ARG, "moe_rms_norm_grad: an output overlaps another buffer");
  const norm_grad_call a = {dy, h, w, dres, rstd, dx, dw, part, dy_type, h_type, w_type, dx_type, T, H};
  device_scope ds(c->device);
  HIPC(c, ds.err);
  {
    prof_scope ps(c, K_RMS_NORM_GRAD, (hipStream_t)stream, true);
    if (!launch_rms_norm_grad(a, c->n_cu, (hipStream_t)stream))
      return fail(c, MOE_ERR_UNSUPPORTED, "moe_rms_norm_grad: T = %d rows of H = %d", T, H);
  }
  HIPC(c, hipGetLastError());
  return MOE_OK;
}

extern "C" moe_status moe_route_groups(moe_ctx *c, const void *logits, int logits_type, const float *bias, int T, int E, int k,
                                       int mode, int n_group, int keep, int top, int norm, float scale, int32_t *ids,
                                       float *wts, float *scores, void *stream) {
  if (!c) return MOE_ERR_INVALID_ARG;
  if (!is_array(logits, type_bytes(logits_type)) || (bias && !is_array(bias, 4)) || !is_array(ids, 4) || !is_array(wts, 4) ||
      (scores && !is_array(scores, 4)) || T <= 0 || E <= 0 || E > MOE_ROUTE_MAX_E || k <= 0 || k > 64 || mode < 0 || mode > 2 ||
      n_group <= 0 || n_group > 64 || E % n_group || keep <= 0 || keep > n_group || k > E / n_group * keep || top < 1 || top > 2)
    return fail(c, MOE_ERR_INVALID_ARG, "moe_route_groups: bad arguments");
  const size_t np = (size_t)T * k * 4, ne = (size_t)T * E;
  if (overlap({{logits, ne * type_bytes(logits_type), false}, {bias, (size_t)E * 4, false}, {ids, np, true}, {wts, np, true},
               {scores, ne * 4, true}}))
    return fail(c, MOE_ERR_INVALID_ARG, "moe_route_groups: an output overlaps another buffer");
  const route_call a = {logits, bias, ids, wts, scores, logits_type, T, E, k, mode, n_group, keep, top, norm, scale};
  device_scope ds(c->device);
  HIPC(c, ds.err);
  {
    prof_scope ps(c, K_ROUTE_GROUPS, (hipStream_t)stream, true);
    if (!launch_route_groups(a, (hipStream_t)stream))
      return fail(c, MOE_ERR_UNSUPPORTED, "moe_route_groups: T = %d tokens", T);
  }
  HIPC(c, hipGetLastError());
  return MOE_OK;
}

extern "C" moe_status moe_route_grad(moe_ctx *c, const void *logits, int logits_type, const int32_t *ids, const float *dwts,
                                     const float *dscores, int T, int E, int k, int mode, int norm, float scale, void *dlogits,
                                     int dlogits_type, void *stream) {
  if (!c) return MOE_ERR_INVALID_ARG;
  if (!is_array(logits, type_bytes(logits_type)) || !is_array(ids, 4) || !is_array(dwts, 4) || (dscores && !is_array(dscores, 4)) ||
      !is_array(dlogits, type_bytes(dlogits_type)) || T <= 0 || E <= 0 || E > MOE_ROUTE_MAX_E || k <= 0 || k > 64 || mode < 0 ||
      mode > 2)
    return fail(c, MOE_ERR_INVALID_ARG, "moe_route_grad: bad arguments");
  const size_t np = (size_t)T * k * 4, ne = (size_t)T * E;
  if (overlap({{logits, ne * type_bytes(logits_type), false}, {ids, np, false}, {dwts, np, false}, {dscores, ne * 4, false},
               {dlogits, ne * type_bytes(dlogits_type), true}}))
    return fail(c, MOE_ERR_INVALID_ARG, "moe_route_grad: dlogits overlaps another buffer");
  const route_grad_call a = {logits, ids, dwts, dscores, dlogits, logits_type, dlogits_type, T, E, k, mode, norm, scale};
  device_scope ds(c->device);
  HIPC(c, ds.err);
  {
    prof_scope ps(c, K_ROUTE_GRAD, (hipStream_t)stream, true);
    if (!launch_route_grad(a, (hipStream_t)stream)) return fail(c, MOE_ERR_UNSUPPORTED, "moe_route_grad: T = %d tokens", T);
  }
  HIPC(c, hipGetLastError());
  return MOE_OK;
}

static bool adapters_sizes(int M, int K, int R) {
  return M > 0 && K > 0 && K <= MOE_ROW_MAX && R > 0 && R <= MOE_ADAPTERS_MAX_RANK;
}

extern "C" size_t moe_adapters_scratch(const moe_ctx *c, int M, int K, int R) {
  return c && adapters_sizes(M, K, R) ? adapters_scratch(M, K, R, c->n_cu) : 0;
}

extern "C" moe_status moe_adapters(moe_ctx *c, const void *x, const void *a, const void *b, int type, const float *scale, int n,
                                   const int32_t *offsets, const int32_t *perm, int M, int K, int R, int N, const void *base,
                                   void *out, int out_type, float *mid, size_t mid_floats, void *stream) {
  if (!c) return MOE_ERR_INVALID_ARG;
  const size_t tb = type_bytes(type), ob = type_bytes(out_type);
  if (!is_array(x, tb) || !is_array(a, tb) || !is_array(b, tb) || (scale && !is_array(scale, 4)) || !is_array(offsets, 4) ||
      !is_array(perm, 4) || !is_array(base, ob) || !is_array(out, ob) || !is_array(mid, 4) || n <= 0 || n > MOE_ADAPTERS_MAX ||
      !adapters_sizes(M, K, R) || N <= 0 || N > MOE_ROW_MAX)
    return fail(c, MOE_ERR_INVALID_ARG, "moe_adapters: bad arguments");
  const size_t need = adapters_need(M, K, R, c->n_cu), no = (size_t)M * N * ob;
  if (mid_floats < need)
    return fail(c, MOE_ERR_INVALID_ARG, "moe_adapters: mid holds %zu floats, this call needs %zu", mid_floats, need);
  if (overlap({{x, (size_t)M * K * tb, false}, {a, (size_t)n * R * K * tb, false}, {b, (size_t)n * N * R * tb, false},
               {scale, (size_t)n * 4, false}, {offsets, ((size_t)n + 1) * 4, false}, {perm, (size_t)M * 4, false},
               {base == out ? nullptr : base, no, false}, {out, no, true}, {mid, need * 4, true}}))
    return fail(c, MOE_ERR_INVALID_ARG, "moe_adapters: an output overlaps another buffer");
  const adapters_call call = {x, a, b, scale, offsets, perm, base, out, mid, type, out_type, n, M, K, R, N};
  device_scope ds(c->device);
  HIPC(c, ds.err);
  {
    prof_scope ps(c, K_ADAPTERS, (hipStream_t)stream, true);
    if (!launch_adapters(call, c->n_cu, (hipStream_t)stream))
      return fail(c, MOE_ERR_UNSUPPORTED, "moe_adapters: M = %d rows of N = %d channels", M, N);
  }
  HIPC(c, hipGetLastError());
  return MOE_OK;
}
