// kernels_route.h -- routing with groups of experts, masked experts and 16-bit logits,
// and the gradient of its weights and scores.
//
// s = softmax(l), sigmoid(l) or sqrt(softplus(l)); an expert with l = -inf is masked: its score is 0 and it is
// not picked.  c = s + bias.  Group score: the sum of the `top` largest c of the group's
// experts (numbers of unmasked ones; a group without any comes last); the `keep` best groups stay, and the k
// largest c of their experts are picked; ties go to the lowest index, NaN comes after every number.
// w = scale * s / max(sum of the picked s, 2^-14).
//
// Which experts are picked hangs on the order of scores that may be close: they are compared as
// 64-bit numbers would be, experts without a bias by their logits (the scores rise with them).
// With p = s at the picked, S their sum, D = max(S, 2^-14):
//   dp_i = scale / D (dw_i - [S >= 2^-14] sum_j dw_j p_j / D),  ds = dscores + dp at the picked
//   softmax dl = s (ds - sum s ds), sigmoid dl = ds s (1 - s), sqrt softplus dl = ds sigmoid(l) / (2 s)
#pragma once

#include "kernels_norm.h"
#include "layer_kernels.h"
#include "row_vec.h"
#include "../../include/moe_block.h"

#define MOE_ROUTE_FLOOR 6.103515625e-5f  // 2^-14

__device__ __forceinline__ double route_score_d(double l, int mode) {
  return mode == MOE_ROUTE_SIGMOID ? 1.0 / (1.0 + exp(-l)) : sqrt(l > 40.0 ? l : log1p(exp(l)));
}
// (v_rcp_f32 is off by a step at most; what it takes to 0 is below 2^-126)
__device__ __forceinline__ float route_score_f(float l, int mode) {
  if (mode == MOE_ROUTE_SIGMOID) return __builtin_amdgcn_rcpf(1.0f + expf(-l));
  return l < -15.0f ? expf(0.5f * l) : sqrtf(fmaxf(l, 0.0f) + log1pf(expf(-fabsf(l))));  // (softplus: exp(l) up to exp(l) / 2)
}

__device__ __forceinline__ double wave_sum_d(double v) { return lanes_reduce_d<64>(v, add_d); }
__device__ __forceinline__ double wave_max_d(double v) {
  return lanes_reduce_d<64>(v, [](double a, double b) { return fmax(a, b); });
}

// A score as a whole number that orders as it does (-0 as 0), NaN below every number; 0: no candidate.
__device__ __forceinline__ uint32_t route_key(float c) {
  const uint32_t u = __builtin_bit_cast(uint32_t, c + 0.0f);
  return c != c ? 1u : u & 0x80000000u ? ~u : u | 0x80000000u;
}
// For 64 bits: a NaN is -inf, what is -inf the lowest finite value above it.
#define MOE_ROUTE_LOW (-1.7976931348623157e308)
#define MOE_ROUTE_LOW_F (-3.4028234663852886e38f)
__device__ __forceinline__ double route_key_d(double c) { return c != c ? -INFINITY : c < MOE_ROUTE_LOW ? MOE_ROUTE_LOW : c; }

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max_u(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false));
}
// The largest over the wave, as a scalar: six steps towards lane 63, one read.
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
  v = dpp_max_u<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8: within rows of 16 lanes
  v = dpp_max_u<0x112, 0xF>(v);
  v = dpp_max_u<0x114, 0xF>(v);
  v = dpp_max_u<0x118, 0xF>(v);
  v = dpp_max_u<0x142, 0xA>(v);  // row_bcast15: the last lane of rows 0 and 2 to rows 1 and 3
  v = dpp_max_u<0x143, 0xC>(v);  // row_bcast31: lane 31 to rows 2 and 3
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Logits [at, at + N) of a token as f32, -inf from `left` on.
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

__device__ __forceinline__ float readlane_k(float v, int lane) { return readlane_f(v, lane); }
__device__ __forceinline__ double readlane_k(double v, int lane) { return readlane_d(v, lane); }
template <int CTRL>
__device__ __forceinline__ float dpp_k(float v) { return dpp_f<CTRL>(v); }
template <int CTRL>
__device__ __forceinline__ double dpp_k(double v) { return dpp_d<CTRL>(v); }

// Does the group of this lane stay?  width lanes side by side are a group's, the first n_group * width have one;
// v1, v2: the two largest scores that this lane holds of it, -inf: none, what is -inf itself: the lowest
// finite value.  near: how close two groups in 32 bits may be in another order than in 64; close: set
// where the last that stays and the first that does not are.
template <typename K>
__device__ __forceinline__ bool route_stay(const route_call &a, K v1, K v2, int width, K near, bool &close) {
  const K none = (K)-INFINITY, low = sizeof(K) == 8 ? (K)MOE_ROUTE_LOW : (K)MOE_ROUTE_LOW_F;
  const int lane = threadIdx.x & 63, g = lane / width;
  auto merge = [&](K b1, K b2) {
    v2 = fmax(fmin(v1, b1), fmax(v2, b2));
    v1 = fmax(v1, b1);
  };
  if (width > 1) merge(dpp_k<0xB1>(v1), dpp_k<0xB1>(v2));    // quad_perm [1,0,3,2]
  if (width > 2) merge(dpp_k<0x4E>(v1), dpp_k<0x4E>(v2));    // quad_perm [2,3,0,1]
  if (width > 4) merge(dpp_k<0x141>(v1), dpp_k<0x141>(v2));  // row_half_mirror
  if (width > 8) merge(dpp_k<0x140>(v1), dpp_k<0x140>(v2));  // row_mirror
  K score = v1;
  // 32 bits take -inf and the lowest value for one: the sum with a v1 that counts beside it may be either's
  bool wide = false;
  if (a.top == 2 && v2 > none) {
    const K sum = v1 <= low || v2 <= low ? none : v1 + v2;
    score = sum > low ? sum : low;
    wide = sizeof(K) == 4 && v2 <= low && v1 > (K)0x1p102f;
  }
  int before = 0;  // groups that come before this lane's
  for (int o = 0; o < a.n_group; o++) {
    const K s = readlane_k(score, o * width);
    before += s > score || (s == score && o < g);
  }
  const bool in = before < a.keep;
  if (sizeof(K) == 4 && near > (K)0 && a.keep < a.n_group) {
    const float first_out = wave_max(wide ? INFINITY : in || g >= a.n_group ? -INFINITY : (float)score);
    const float last_in = -wave_max(in && g < a.n_group ? -(float)score : -INFINITY);
    close = last_in > -INFINITY && !(last_in - first_out > (float)near);
  }
  return in;
}

// The same for any groups: c holds the experts' scores by index.  The ballot of the lanes whose groups stay.
template <typename K>
__device__ __forceinline__ uint64_t route_stay_any(const route_call &a, const K *c, K near, bool &close) {
  const int lane = threadIdx.x & 63, g = lane / a.width;
  K v1 = (K)-INFINITY, v2 = (K)-INFINITY;
  if (g < a.n_group)
    for (int e = g * a.per + lane % a.width; e < (g + 1) * a.per; e += a.width) {
      v2 = fmax(v2, fmin(v1, c[e]));
      v1 = fmax(v1, c[e]);
    }
  return __ballot(route_stay(a, v1, v2, a.width, near, close));
}

// One wave a token, WAVES tokens a workgroup.  Lane i holds experts [NJ i, NJ i + NJ) (E <= 64 NJ), so that of equal
// keys the lowest lane has the lowest index, and a pick is a maximum over the wave and a ballot.
// Scores with a bias are compared in 32 bits: that decides unless two that stand next to each other in the
// order come closer than both may be off.  Then those that may be picked are placed by their scores in 64 bits,
// and where it is two groups (or more experts than a wave has lanes) the token is done again in 64 bits.
// Bound by the instructions of a pick, about 35 one after the other (0.12 us alone), and by latency: 256 experts in 8
// groups, bias, top-8: one token 4.6 us, 4096 9.7 (everything in 64 bits 13.4; keys not sorted in their lanes
// 14.3; without bias and groups 5.9).  Lanes hold neighbours, not every 64th expert: a group is then whole lanes.
template <int NJ, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_route_groups(route_call a) {
  // for the groups' scores
  __shared__ float c32[WAVES][64 * NJ];
  __shared__ double c64[WAVES][64 * NJ];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, E = a.E, e0 = lane * NJ;
  const long t = (long)blockIdx.x * WAVES + wave;
  if (t >= a.T) return;  // whole waves; no barrier below
  const size_t at = (size_t)t * E;
  const bool soft = a.mode == MOE_ROUTE_SOFTMAX, sums = a.n_group > 1 && a.top == 2;
  float l[NJ], b[NJ], p[NJ];
  route_load<NJ>(a.logits, a.type, at + e0, E - e0, l);
#pragma unroll
  for (int j = 0; j < NJ; j++) b[j] = a.bias && e0 + j < E ? a.bias[e0 + j] : 0.0f;
  float top = 0.0f, sum = 1.0f;
  if (soft) {
    top = l[0];
#pragma unroll
    for (int j = 1; j < NJ; j++) top = fmaxf(top, l[j]);
    top = wave_max(top);
    if (top == -INFINITY) top = 0.0f;
    float some = 0.0f;
#pragma unroll
    for (int j = 0; j < NJ; j++) some += p[j] = expf(l[j] - top);
    some = wave_sum(some);
    sum = some != 0.0f ? some : 1.0f;  // (0: every expert is masked)
  }
  const float inv_sum = __fdiv_rn(1.0f, sum);
  if (a.bias || a.scores || sums) {
#pragma unroll
    for (int j = 0; j < NJ; j++) p[j] = l[j] == -INFINITY ? 0.0f : soft ? p[j] * inv_sum : route_score_f(l[j], a.mode);
  }
  if (a.scores) {
#pragma unroll
    for (int j = 0; j < NJ; j++)
      if (e0 + j < E) a.scores[at + e0 + j] = p[j];
  }
  // how close two scores in 32 bits may be in another order than in 64: each is off by 7 half steps of f32 (2^-24) of
  // p, softmax's by 33 and twice the size of the exponent, and one of c; those next to 0 by steps of the smallest values.
  // A sum of two is off by what both are and by its own rounding, half a step of |c1 + c2|: as if each c were off by two,
  // which is counted for all.  So two scores are off by `near` together, two groups' sums of `top` by top times as much
  float near = 0.0f;
  if (a.bias || sums) {
    float big = 0.0f, each = 3.5f;  // in double steps, so that no finite c passes f32
    if (soft) {
      float low = 0.0f;
#pragma unroll
      for (int j = 0; j < NJ; j++)
        if (l[j] != -INFINITY) low = fmaxf(low, top - l[j]);
      each = 16.5f + fminf(wave_max(low), 100.0f);
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const float size = fmaf(each, p[j], fabsf(p[j] + b[j]));
      big = l[j] != -INFINITY && size < INFINITY ? fmaxf(big, size) : big;  // (infinities are what they are in 64 bits)
    }
    near = fmaf(wave_max(big), 0x1p-22f, 0x1p-120f);
  }
  uint32_t key[NJ];
#pragma unroll
  for (int j = 0; j < NJ; j++) key[j] = l[j] == -INFINITY ? 0 : route_key(a.bias ? p[j] + b[j] : l[j]);
  const float inv_per = 1.0f / (float)a.per, near_groups = (float)a.top * near;
  bool again = false;
  auto drop = [&](uint64_t stay, auto f) {  // f(j) of the experts whose groups do not stay
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const int g = (int)(((float)(e0 + j) + 0.5f) * inv_per);  // (e0 + j) / per: a half is more than the product is off
      if (e0 + j < E && !((stay >> g * a.width) & 1)) f(j);
    }
  };
  if (a.n_group > 1) {
    float c[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const float v = a.bias ? p[j] + b[j] : sums ? p[j] : l[j];
      c[j] = l[j] == -INFINITY || v != v ? -INFINITY : fmaxf(v, MOE_ROUTE_LOW_F);
    }
    if (a.lanes) {  // whole lanes are a group's
      float v1 = c[0], v2 = -INFINITY;
#pragma unroll
      for (int j = 1; j < NJ; j++) {
        v2 = fmaxf(v2, fminf(v1, c[j]));
        v1 = fmaxf(v1, c[j]);
      }
      const bool in = route_stay<float>(a, v1, v2, a.lanes, near_groups, again);
#pragma unroll
      for (int j = 0; j < NJ; j++) key[j] = in ? key[j] : 0;
    } else {
#pragma unroll
      for (int j = 0; j < NJ; j++) c32[wave][e0 + j] = c[j];
      __builtin_amdgcn_wave_barrier();
      drop(route_stay_any<float>(a, c32[wave], near_groups, again), [&](int j) { key[j] = 0; });
    }
  }
  // lane s: the expert of slot s, and its key
  int my_id = -1;
  uint32_t my_key = 0;
  if (!again) {
    // a lane's keys in order, of equal ones the lower index first: its best left is key[0], and a pick moves the others up
    uint32_t idx[NJ];
    auto either = [](uint32_t mask, uint32_t a, uint32_t b) { return (a & mask) | (b & ~mask); };  // (one v_bfi)
#pragma unroll
    for (int j = 0; j < NJ; j++) idx[j] = e0 + j;
#pragma unroll
    for (int i = 0; i < NJ; i++)
#pragma unroll
      for (int j = i & 1; j + 1 < NJ; j += 2) {
        const uint32_t k0 = key[j], k1 = key[j + 1], swap = k1 > k0 ? ~0u : 0u, i0 = idx[j], i1 = idx[j + 1];
        key[j] = max(k0, k1);
        key[j + 1] = min(k0, k1);
        idx[j] = either(swap, i1, i0);
        idx[j + 1] = either(swap, i0, i1);
      }
    // with a bias, as many more as may belong before the last of the k
    auto value = [](uint32_t k) { return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k); };
    float floor = INFINITY;
    int n = 0;
    for (; n < 64; n++) {
      const uint32_t mx = wave_max_u(key[0]);
      if (mx == 0) break;
      if (n >= a.k - 1) {
        if (n == a.k - 1) floor = mx > 1 && a.bias ? value(mx) - near : INFINITY;
        else if (mx == 1 || !(value(mx) >= floor)) break;
      }
      const int src = __ffsll((unsigned long long)__ballot(key[0] == mx)) - 1;
      const int id = __builtin_amdgcn_readlane((int)idx[0], src);
      if (lane == n) {
        my_id = id;
        my_key = mx;
      }
      const uint32_t win = lane == src ? ~0u : 0u;
#pragma unroll
      for (int j = 0; j < NJ; j++) {
        key[j] = either(win, j + 1 < NJ ? key[j + 1] : 0u, key[j]);
        if (j + 1 < NJ) idx[j] = either(win, idx[j + 1], idx[j]);
      }
    }
    if (a.bias) {
      // two that follow each other, both numbers
      const uint32_t after = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)my_key, 0x130, 0xF, 0xF, false);  // wave_shl 1
      again = n == 64;  // (there may be more that belong among them)
      if (!again && __ballot(my_key > 1 && after > 1 && !(value(my_key) - value(after) > near))) {
        // those picked and those that may belong among them, by their place in 64 bits
        double sum_d = 1.0, c = -INFINITY;
        if (soft) {
          sum_d = 0.0;
#pragma unroll
          for (int j = 0; j < NJ; j++) sum_d += exp((double)l[j] - (double)top);
          sum_d = wave_sum_d(sum_d);
        }
        if (my_id >= 0) {
          float one[1];
          route_load<1>(a.logits, a.type, at + my_id, 1, one);
          c = route_key_d((soft ? exp((double)one[0] - (double)top) / sum_d : route_score_d((double)one[0], a.mode)) +
                          (double)a.bias[my_id]);
        }
        int place = 0;
        for (int o = 0; o < n; o++) {
          const double other = readlane_d(c, o);
          const int other_id = __builtin_amdgcn_readlane(my_id, o);
          place += other > c || (other == c && other_id < my_id);
        }
        my_id = __builtin_amdgcn_ds_permute(4 * (lane < n ? place : lane), my_id);
      }
    }
    if (lane >= a.k) my_id = -1;
  }
  if (again) {
    double kd[NJ], sum_d = 1.0;
    uint32_t left = 0;  // bit j: expert e0 + j may be picked
    if (soft) {
      sum_d = 0.0;
#pragma unroll
      for (int j = 0; j < NJ; j++) sum_d += exp((double)l[j] - (double)top);
      sum_d = wave_sum_d(sum_d);
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      kd[j] = route_key_d((soft ? exp((double)l[j] - (double)top) / sum_d : route_score_d((double)l[j], a.mode)) + (double)b[j]);
      if (l[j] != -INFINITY) left |= 1u << j;
    }
    if (a.n_group > 1) {
#pragma unroll
      for (int j = 0; j < NJ; j++) c64[wave][e0 + j] = (left >> j) & 1 ? kd[j] : -INFINITY;
      __builtin_amdgcn_wave_barrier();
      drop(route_stay_any<double>(a, c64[wave], 0.0, again), [&](int j) { left &= ~(1u << j); });
    }
    if (!a.bias) {
#pragma unroll
      for (int j = 0; j < NJ; j++) kd[j] = route_key_d((double)l[j]);
    }
    my_id = -1;
    for (int s = 0; s < a.k; s++) {
      double best = -INFINITY;
      int bj = -1;
#pragma unroll
      for (int j = 0; j < NJ; j++)
        if (((left >> j) & 1u) && (bj < 0 || kd[j] > best)) {
          best = kd[j];
          bj = j;
        }
      const double mx = wave_max_d(best);
      const uint64_t m = __ballot(bj >= 0 && best == mx);
      if (!m) break;
      const int src = __ffsll((unsigned long long)m) - 1, id = src * NJ + __builtin_amdgcn_readlane(bj, src);
      if (lane == src) left &= ~(1u << bj);
      if (lane == s) my_id = id;
    }
  }
  float w = 0.0f;
  if (my_id >= 0) {
    float one[1];
    route_load<1>(a.logits, a.type, at + my_id, 1, one);
    w = soft ? expf(one[0] - top) * inv_sum : route_score_f(one[0], a.mode);
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
  const float z = expf(-fabsf(l)), big = __builtin_amdgcn_rcpf(1.0f + z), sig = l >= 0.0f ? big : z * big;
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

// One wave a token, WAVES a workgroup, lane i with experts [NJ i, NJ i + NJ) in registers.  The picked
// experts' gradients go to their lanes slot by slot, which adds an expert that is named twice in slot order.
// Latency: 4096 tokens of 256 experts with dscores (12.8 MB) 6.6 us (10.9 with the scores in LDS); 301 of 160 3.4.
template <int NJ, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_route_grad(route_grad_call a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, E = a.E, e0 = lane * NJ;
  const long t = (long)blockIdx.x * WAVES + wave;
  if (t >= a.T) return;  // whole waves
  const size_t at = (size_t)t * E;
  const bool soft = a.mode == MOE_ROUTE_SOFTMAX;
  float l[NJ], ds[NJ], p[NJ], slope[NJ];
  route_load<NJ>(a.logits, a.type, at + e0, E - e0, l);
  if (a.dscores) {
    load_v<float, NJ>(a.dscores + at + e0, E - e0, ds);
  } else {
#pragma unroll
    for (int j = 0; j < NJ; j++) ds[j] = 0.0f;
  }
  // lane s: slot s
  const int id = lane < a.k ? a.ids[(size_t)t * a.k + lane] : -1;
  const bool there = id >= 0 && id < E;
  float dw = there ? a.dwts[(size_t)t * a.k + lane] : 0.0f, mine[1] = {-INFINITY};
  if (there) route_load<1>(a.logits, a.type, at + id, 1, mine);
  float top = 0.0f, inv_sum = 1.0f, own, unused;
  if (soft) {
    top = l[0];
#pragma unroll
    for (int j = 1; j < NJ; j++) top = fmaxf(top, l[j]);
    top = wave_max(top);
    if (top == -INFINITY) top = 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NJ; j++) sum += p[j] = expf(l[j] - top);
    sum = wave_sum(sum);
    inv_sum = __fdiv_rn(1.0f, sum != 0.0f ? sum : 1.0f);  // (0: every expert is masked)
#pragma unroll
    for (int j = 0; j < NJ; j++) p[j] *= inv_sum;
    own = expf(mine[0] - top) * inv_sum;
  } else {
#pragma unroll
    for (int j = 0; j < NJ; j++) route_slope(l[j], a.mode, p[j], slope[j]);
    route_slope(mine[0], a.mode, own, unused);
  }
  if (mine[0] == -INFINITY) own = 0.0f;
  if (a.scale != 0.0f) dw *= a.scale;
  if (a.norm) {
    // (a sum that is NaN is no less than its floor: the weights are NaN, and so is their gradient)
    const float S = wave_sum(own), in = wave_sum(dw * own), D = S < MOE_ROUTE_FLOOR ? MOE_ROUTE_FLOOR : S;
    dw = __fdiv_rn(dw - (S < MOE_ROUTE_FLOOR ? 0.0f : __fdiv_rn(in, D)), D);
  }
  if (!there) dw = 0.0f;
  for (int s = 0; s < a.k; s++) {
    const int e = __builtin_amdgcn_readlane(id, s);
    const float d = readlane_f(dw, s);
#pragma unroll
    for (int j = 0; j < NJ; j++) ds[j] += e0 + j == e ? d : 0.0f;
  }
  float in = 0.0f;
  if (soft) {
#pragma unroll
    for (int j = 0; j < NJ; j++) in = p[j] != 0.0f ? fmaf(p[j], ds[j], in) : in;
    in = wave_sum(in);
  }
  float d[NJ];
#pragma unroll
  for (int j = 0; j < NJ; j++) d[j] = l[j] == -INFINITY ? 0.0f : soft ? p[j] * (ds[j] - in) : ds[j] * slope[j];
  if (e0 >= E) return;
  if (a.out_type == MOE_GGML_F32) store_v<float, NJ>(reinterpret_cast<float *>(a.dlogits) + at + e0, E - e0, d);
  else if (a.out_type == MOE_GGML_F16) store_v<_Float16, NJ>(reinterpret_cast<_Float16 *>(a.dlogits) + at + e0, E - e0, d);
  else store_v<bf16_t, NJ>(reinterpret_cast<bf16_t *>(a.dlogits) + at + e0, E - e0, d);
}
