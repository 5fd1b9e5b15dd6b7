// launch_common.h -- what the launches of expert_kernels.hip and layer_kernels.hip share (host).
#pragma once

#include "../../include/moe_block.h"
#include "row_vec.h"

static inline int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

// A grid's x dimension holds fewer than 2^32 threads.
static inline bool fits(long blocks, int threads) { return blocks * threads < (1L << 32); }

// f(T{}) for the element type t.
template <typename F>
static void with_type(int t, F f) {
  if (t == MOE_GGML_F32) f(float{});
  else if (t == MOE_GGML_F16) f(_Float16{});
  else f(bf16_t{});
}
