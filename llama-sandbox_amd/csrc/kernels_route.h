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

#include "kernels_norm.h"
#include "layer_kernels.h"
#include "row_vec.h"
#include "../../include/moe_block.h"

#define MOE_ROUTE_GROUPS_MAX_E 1024
#define MOE_ROUTE_FLOOR 6.103515625e-5f  // 2^-14

__device__ __forceinline__ double route_score_d(double l, int mode) {
  return mode == MOE_ROUTE_SIGMOID ? 1.0 / (1.0 + exp(-l)) : sqrt(l > 40.0 ? l : log1p(exp(l)));
}
__device__ __forceinline__ float route_score_f(float l, int mode) {
  if (mode == MOE_ROUTE_SIGMOID) return __fdiv_rn(1.0f, 1.0f + expf(-l));
  return l < -15.0f ? expf(0.5f * l) : sqrtf(fmaxf(l, 0.0f) + log1pf(expf(-fabsf(l))));  // (softplus: exp(l) up to exp(l) / 2)
}

__device__ __forceinline__ float wave_max_k(float v) { return wave_max(v); }
__device__ __forceinline__ double wave_max_k(double v) {
  v = fmax(v, dpp_d<0xB1>(v));
  v = fmax(v, dpp_d<0x4E>(v));
  v = fmax(v, dpp_d<0x141>(v));
  v = fmax(v, dpp_d<0x140>(v));
  return fmax(fmax(readlane_d(v, 0), readlane_d(v, 16)), fmax(readlane_d(v, 32), readlane_d(v, 48)));
}
__device__ __forceinline__ float readlane_k(float v, int lane) { return readlane_f(v, lane); }
__device__ __forceinline__ double readlane_k(double v, int lane) { return readlane_d(v, lane); }
__device__ __forceinline__ double wave_sum_d(double v) { return lanes_reduce_d<64>(v, add_d); }

// What a selection score is compared as: a NaN is -inf, what is -inf the lowest finite value above it.
template <typename K>
__device__ __forceinline__ K route_key(K c) {
  const K low = sizeof(K) == 8 ? (K)-1.7976931348623157e308 : (K)-3.4028234663852886e38f;
  return c != c ? (K)-INFINITY : c < low ? low : c;
}
template <typename K>
__device__ __forceinline__ K route_unkey(K k) {
  const K low = sizeof(K) == 8 ? (K)-1.7976931348623157e308 : (K)-3.4028234663852886e38f;
  return k <= low ? (K)-INFINITY : k;
}

// The two largest of two pairs in order.
template <typename K>
__device__ __forceinline__ void route_merge(K &a1, K &a2, K b1, K b2) {
  a2 = fmax(fmin(a1, b1), fmax(a2, b2));
  a1 = fmax(a1, b1);
}

// Logits [at, at + n) of a token as f32, -inf from `left` on.
template <int N>
__device__ __forceinline__ void route_load(const void *logits, int type, size_t at, int left, float (&l)[N]) {
  auto get = [&](auto t) {
    typedef decltype(t) T;
    const T *p = reinterpret_cast<const T *>(logits) + at;
    if (left >= N) {
      typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
      const vec v = *reinterpret_cast<const vec *>(p);
#pragma unroll
      for (int j = 0; j < N; j++) l[j] = (float)v[j];
    } else {
#pragma unroll
      for (int j = 0; j < N; j++) l[j] = j < left ? (float)p[j] : -INFINITY;
    }
  };
  if (type == MOE_GGML_F32) get(float{});
  else if (type == MOE_GGML_F16) get(_Float16{});
  else get(bf16_t{});
}

// One wave a token, WAVES tokens a workgroup.  Lane i holds experts [NJ i, NJ i + NJ) (E <= 64 NJ), so that of equal
// keys the lowest lane has the lowest index, and a pick is a maximum over the wave and a ballot.  K: the type
// that selection scores are compared in: float where they are the logits.
template <typename K, int NJ, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_route_groups(route_call a) {
  __shared__ K keys[WAVES][64 * NJ];  // for the groups' scores
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, E = a.E, e0 = lane * NJ;
  const long t = (long)blockIdx.x * WAVES + wave;
  if (t >= a.T) return;  // whole waves; no barrier below
  const size_t at = (size_t)t * E;
  const bool soft = a.mode == MOE_ROUTE_SOFTMAX;
  float l[NJ];
  route_load<NJ>(a.logits, a.type, at + e0, E - e0, l);
  float b[NJ];
#pragma unroll
  for (int j = 0; j < NJ; j++) b[j] = sizeof(K) == 8 && a.bias && e0 + j < E ? a.bias[e0 + j] : 0.0f;
  float top = 0.0f, sum = 1.0f;
  double sum_d = 1.0;
  if (soft) {
    top = l[0];
#pragma unroll
    for (int j = 1; j < NJ; j++) top = fmaxf(top, l[j]);
    top = wave_max(top);
    if (top == -INFINITY) top = 0.0f;
    if constexpr (sizeof(K) == 8) {
      sum_d = 0.0;
#pragma unroll
      for (int j = 0; j < NJ; j++) sum_d += exp((double)l[j] - (double)top);
      sum_d = wave_sum_d(sum_d);
      sum = (float)sum_d;
    } else {
      sum = 0.0f;
#pragma unroll
      for (int j = 0; j < NJ; j++) sum += expf(l[j] - top);
      sum = wave_sum(sum);
    }
  }
  if (a.scores) {
#pragma unroll
    for (int j = 0; j < NJ; j++)
      if (e0 + j < E)
        a.scores[at + e0 + j] = l[j] == -INFINITY ? 0.0f : soft ? __fdiv_rn(expf(l[j] - top), sum) : route_score_f(l[j], a.mode);
  }
  K key[NJ];
  uint32_t left = 0;  // bit j: expert e0 + j may be picked
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    if constexpr (sizeof(K) == 8)
      key[j] = route_key((soft ? exp((double)l[j] - (double)top) / sum_d : route_score_d((double)l[j], a.mode)) + (double)b[j]);
    else
      key[j] = route_key(l[j]);
    if (l[j] != -INFINITY) left |= 1u << j;
  }
  if (a.n_group > 1) {
    // lanes g * width .. of group g scan it
    const int per = E / a.n_group, width = a.n_group <= 4 ? 16 : 64 >> (32 - __builtin_clz(a.n_group - 1));
    K v1 = (K)-INFINITY, v2 = (K)-INFINITY;
#pragma unroll
    for (int j = 0; j < NJ; j++) keys[wave][e0 + j] = (left >> j) & 1 ? key[j] : (K)-INFINITY;
    __builtin_amdgcn_wave_barrier();
    const int g = lane / width;
    if (g < a.n_group)
      for (int e = g * per + lane % width; e < (g + 1) * per; e += width) route_merge(v1, v2, keys[wave][e], (K)-INFINITY);
    for (int off = 1; off < width; off <<= 1) {
      const K o1 = __shfl_xor(v1, off), o2 = __shfl_xor(v2, off);
      route_merge(v1, v2, o1, o2);
    }
    // a group without a number: -inf; of one number, that one
    const K score = a.top == 2 && v2 > (K)-INFINITY ? route_unkey(v1) + route_unkey(v2) : route_unkey(v1);
    int before = 0;  // groups that come before this lane's
    for (int o = 0; o < a.n_group; o++) {
      const K s = readlane_k(score, o * width);
      before += s > score || (s == score && o < g);
    }
    const uint64_t stay = __ballot(before < a.keep);
#pragma unroll
    for (int j = 0; j < NJ; j++)
      if (e0 + j < E && !((stay >> ((e0 + j) / per * width)) & 1)) left &= ~(1u << j);
  }
  int my_id = -1;  // lane s: the expert of slot s
  for (int s = 0; s < a.k; s++) {
    K best = (K)-INFINITY;
    int bj = -1;
#pragma unroll
    for (int j = 0; j < NJ; j++)
      if (((left >> j) & 1u) && (bj < 0 || key[j] > best)) {
        best = key[j];
        bj = j;
      }
    const K mx = wave_max_k(best);
    const uint64_t m = __ballot(bj >= 0 && best == mx);
    if (!m) break;
    const int src = __ffsll((unsigned long long)m) - 1, id = src * NJ + __builtin_amdgcn_readlane(bj, src);
    if (lane == src) left &= ~(1u << bj);
    if (lane == s) my_id = id;
  }
  float w = 0.0f;
  if (my_id >= 0) {
    float one[1];
    route_load<1>(a.logits, a.type, at + my_id, 1, one);
    w = soft ? __fdiv_rn(expf(one[0] - top), sum) : route_score_f(one[0], a.mode);
  }
  if (a.norm) {
    const float total = wave_sum(w);
    w = __fdiv_rn(w, total < MOE_ROUTE_FLOOR ? MOE_ROUTE_FLOOR : total);
  }
  if (a.scale != 0.0f) w *= a.scale;
  if (lane < a.k) {
    a.ids[(size_t)t * a.k + lane] = my_id;
    a.wts[(size_t)t * a.k + lane] = w;
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
