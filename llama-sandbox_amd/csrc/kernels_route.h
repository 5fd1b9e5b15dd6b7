// kernels_route.h -- routing with groups of experts, masked experts and 16-bit logits,
// and the gradient of its weights and scores.
//
// s = softmax(l), sigmoid(l) or sqrt(softplus(l)); an expert with l = -inf is masked: its score is 0 and it is
// not picked.  c = s + bias.  Group score: the sum of the `top` largest c of the group's
// unmasked experts (-inf without any); the `keep` best groups stay, and the k largest c
// of their experts are picked; ties go to the lowest index, NaN comes after every number.
// w = scale * s / max(sum of the picked s, 2^-14).
//
// Which experts are picked hangs on the order of scores that may be close: they are
// compared in 64 bits, or by their logits where that is the same order (no bias, and no sum of two).
// With p = s at the picked, S their sum, D = max(S, 2^-14):
//   dp_i = scale / D (dw_i - [S >= 2^-14] sum_j dw_j p_j / D),  ds = dscores + dp at the picked
//   softmax dl = s (ds - sum s ds), sigmoid dl = ds s (1 - s), sqrt softplus dl = ds sigmoid(l) / (2 s)
#pragma once

#include "layer_kernels.h"
#include "row_vec.h"
#include "../../include/moe_block.h"

#define MOE_ROUTE_GROUPS_MAX_E 1024
#define MOE_ROUTE_FLOOR 6.103515625e-5f  // 2^-14

__device__ __forceinline__ double route_score_d(double l, int mode) {
  return mode == MOE_ROUTE_SIGMOID ? 1.0 / (1.0 + exp(-l)) : sqrt(l > 40.0 ? l : log1p(exp(l)));
}

// a comes before b: larger, or equal and of the lower index; NaN after every number.
__device__ __forceinline__ bool route_before(double a, int ia, double b, int ib) {
  if (a != a || b != b) return a == a ? true : b == b ? false : ia < ib;
  return a > b || (a == b && ia < ib);
}

// The first of a wave's candidates (index -1: none); every lane gets it.
__device__ __forceinline__ void route_first(double &v, int &i) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const double ov = __shfl_xor(v, off);
    const int oi = __shfl_xor(i, off);
    if (oi >= 0 && (i < 0 || route_before(ov, oi, v, i))) {
      v = ov;
      i = oi;
    }
  }
}

// One wave a token.
template <typename T>
__global__ __launch_bounds__(64) void k_route_groups(route_call a) {
  __shared__ double s[MOE_ROUTE_GROUPS_MAX_E], c[MOE_ROUTE_GROUPS_MAX_E];
  __shared__ double gs[64];
  __shared__ uint8_t state[MOE_ROUTE_GROUPS_MAX_E];  // 1: may be picked
  const int t = blockIdx.x, lane = threadIdx.x, E = a.E, per = E / a.n_group;
  const T *l = reinterpret_cast<const T *>(a.logits) + (size_t)t * E;
  double top = -INFINITY, sum = 0.0;
  if (a.mode == MOE_ROUTE_SOFTMAX) {
    for (int e = lane; e < E; e += 64) top = fmax(top, (double)(float)l[e]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = fmax(top, __shfl_xor(top, off));
    if (top == -INFINITY) top = 0.0;
    for (int e = lane; e < E; e += 64) sum += s[e] = exp((double)(float)l[e] - top);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
  }
  const bool by_logit = !a.bias && (a.n_group == 1 || a.top == 1);
  for (int e = lane; e < E; e += 64) {
    const double v = (double)(float)l[e];
    const bool masked = v == -INFINITY;
    double p = a.mode == MOE_ROUTE_SOFTMAX ? s[e] / sum : route_score_d(v, a.mode);
    if (masked) p = 0.0;
    s[e] = p;
    c[e] = by_logit ? v : a.bias ? p + (double)a.bias[e] : p;
    state[e] = !masked;
    if (a.scores) a.scores[(size_t)t * E + e] = (float)p;
  }
  __syncthreads();
  if (a.n_group > 1) {
    if (lane < a.n_group) {
      double v1 = 0.0, v2 = 0.0;
      int i1 = -1, i2 = -1;
      for (int e = lane * per; e < (lane + 1) * per; e++) {
        if (!state[e]) continue;
        if (i1 < 0 || route_before(c[e], e, v1, i1)) {
          v2 = v1;
          i2 = i1;
          v1 = c[e];
          i1 = e;
        } else if (i2 < 0 || route_before(c[e], e, v2, i2)) {
          v2 = c[e];
          i2 = e;
        }
      }
      gs[lane] = i1 < 0 ? -INFINITY : a.top == 2 && i2 >= 0 ? v1 + v2 : v1;
    }
    __syncthreads();
    bool stay = false;
    if (lane < a.n_group) {
      int before = 0;
      for (int g = 0; g < a.n_group; g++) before += g != lane && route_before(gs[g], g, gs[lane], lane);
      stay = before < a.keep;
    }
    const uint64_t kept = __ballot(stay);
    for (int e = lane; e < E; e += 64)
      if (!((kept >> (e / per)) & 1)) state[e] = 0;
    __syncthreads();
  }
  int my_id = -1;
  double my_w = 0.0, total = 0.0;
  for (int j = 0; j < a.k; j++) {
    double v = 0.0;
    int i = -1;
    for (int e = lane; e < E; e += 64)
      if (state[e] && (i < 0 || route_before(c[e], e, v, i))) {
        v = c[e];
        i = e;
      }
    route_first(v, i);
    if (i < 0) break;
    const double w = s[i];
    total += w;
    if (lane == j) {
      my_id = i;
      my_w = w;
    }
    __syncthreads();
    if (lane == 0) state[i] = 0;
    __syncthreads();
  }
  if (a.norm) my_w /= total < (double)MOE_ROUTE_FLOOR ? (double)MOE_ROUTE_FLOOR : total;
  if (a.scale != 0.0f) my_w *= (double)a.scale;
  if (lane < a.k) {
    a.ids[(size_t)t * a.k + lane] = my_id;
    a.wts[(size_t)t * a.k + lane] = (float)my_w;
  }
}

// s and its slope of one logit, element-wise score functions.
__device__ __forceinline__ void route_slope(float l, int mode, float &s, float &slope) {
  const float z = expf(-fabsf(l)), big = __fdiv_rn(1.0f, 1.0f + z), sig = l >= 0.0f ? big : z * big;
  if (mode == MOE_ROUTE_SIGMOID) {
    s = sig;
    slope = big * (z * big);
  } else if (l < -15.0f) {  // softplus is exp(l) up to exp(l) / 2: s = exp(l/2), its slope half of it
    s = expf(0.5f * l);
    slope = 0.5f * s;
  } else {
    s = sqrtf(fmaxf(l, 0.0f) + log1pf(z));
    slope = __fdiv_rn(0.5f * sig, s);
  }
}

// One wave a token.
template <typename T>
__global__ __launch_bounds__(64) void k_route_grad(route_grad_call a) {
  __shared__ float s[MOE_ROUTE_GROUPS_MAX_E], ds[MOE_ROUTE_GROUPS_MAX_E];
  const int t = blockIdx.x, lane = threadIdx.x, E = a.E;
  const T *l = reinterpret_cast<const T *>(a.logits) + (size_t)t * E;
  const float *from = a.dscores ? a.dscores + (size_t)t * E : nullptr;
  const bool soft = a.mode == MOE_ROUTE_SOFTMAX;
  float top = -INFINITY, sum = 0.0f, unused;
  if (soft) {
    for (int e = lane; e < E; e += 64) top = fmaxf(top, (float)l[e]);
    top = wave_max(top);
    if (top == -INFINITY) top = 0.0f;
    for (int e = lane; e < E; e += 64) sum += s[e] = expf((float)l[e] - top);
    sum = wave_sum(sum);
  }
  for (int e = lane; e < E; e += 64) {
    const float v = (float)l[e];
    if (v == -INFINITY) s[e] = 0.0f;
    else if (soft) s[e] = __fdiv_rn(s[e], sum);
    else route_slope(v, a.mode, s[e], unused);
    ds[e] = from ? from[e] : 0.0f;
  }
  __syncthreads();
  const int id = lane < a.k ? a.ids[(size_t)t * a.k + lane] : -1;
  const bool there = id >= 0 && id < E;
  float dw = there ? a.dwts[(size_t)t * a.k + lane] : 0.0f;
  if (a.scale != 0.0f) dw *= a.scale;
  if (a.norm) {
    const float p = there ? s[id] : 0.0f, S = wave_sum(p), D = fmaxf(S, MOE_ROUTE_FLOOR), in = wave_sum(dw * p);
    dw = __fdiv_rn(dw - (S >= MOE_ROUTE_FLOOR ? __fdiv_rn(in, D) : 0.0f), D);
  }
  for (int j = 0; j < a.k; j++) {
    if (lane == j && there) ds[id] += dw;  // in slot order, also where an expert is named twice
    __syncthreads();
  }
  float in = 0.0f;
  if (soft)
    for (int e = lane; e < E; e += 64) in = s[e] != 0.0f ? fmaf(s[e], ds[e], in) : in;
  in = wave_sum(in);
  for (int e = lane; e < E; e += 64) {
    const float v = (float)l[e];
    float slope = s[e], d;
    if (!soft) route_slope(v, a.mode, unused, slope);
    d = soft ? s[e] * (ds[e] - in) : ds[e] * slope;
    if (v == -INFINITY) d = 0.0f;
    const size_t at = (size_t)t * E + e;
    if (a.out_type == MOE_GGML_F32) reinterpret_cast<float *>(a.dlogits)[at] = d;
    else if (a.out_type == MOE_GGML_F16) reinterpret_cast<_Float16 *>(a.dlogits)[at] = (_Float16)d;
    else reinterpret_cast<bf16_t *>(a.dlogits)[at] = (bf16_t)d;
  }
}
