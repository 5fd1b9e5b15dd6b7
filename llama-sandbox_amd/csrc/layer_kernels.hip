// layer_kernels.hip -- the kernels on the way into the experts and beside them (kernels_norm.h,
// kernels_route.h, kernels_adapters.h) and their launches.
#include "layer_kernels.h"

#include "../../include/moe_block.h"
#include "kernels_adapters.h"
#include "kernels_norm.h"
#include "kernels_route.h"
#include "launch_common.h"

bool launch_rms_norm(const norm_call &a, int n_cu, hipStream_t st) {
  if (!fits(a.T, 256)) return false;
  hipLaunchKernelGGL(k_rms_norm_any, dim3(a.T), dim3(256), 0, st, a);
  return true;
}

size_t norm_grad_scratch(int T, int H, int n_cu) { return 1; }

bool launch_rms_norm_grad(const norm_grad_call &a, int n_cu, hipStream_t st) {
  if (!fits(a.T, 256)) return false;
  hipLaunchKernelGGL(k_rms_norm_dx_any, dim3(a.T), dim3(256), 0, st, a);
  hipLaunchKernelGGL(k_rms_norm_dw_any, dim3(ceil_div(a.H, 64)), dim3(256), 0, st, a);
  return true;
}

bool launch_route_groups(const route_call &a, hipStream_t st) {
  if (!fits(a.T, 64)) return false;
  with_type(a.type, [&](auto t) {
    hipLaunchKernelGGL((k_route_groups<decltype(t)>), dim3(a.T), dim3(64), 0, st, a);
  });
  return true;
}

bool launch_route_grad(const route_grad_call &a, hipStream_t st) {
  if (!fits(a.T, 64)) return false;
  with_type(a.type, [&](auto t) {
    hipLaunchKernelGGL((k_route_grad<decltype(t)>), dim3(a.T), dim3(64), 0, st, a);
  });
  return true;
}

size_t adapters_scratch(int M, int K, int R, int n_cu) { return (size_t)M * R; }

bool launch_adapters(const adapters_call &a, int n_cu, hipStream_t st) {
  if (a.M > 65535) return false;
  with_type(a.type, [&](auto t) {
    typedef decltype(t) T;
    hipLaunchKernelGGL((k_adapters_shrink<T>), dim3(ceil_div(a.R, 4), a.M), dim3(256), 0, st, a);
    with_type(a.out_type, [&](auto to) {
      hipLaunchKernelGGL((k_adapters_expand<T, decltype(to)>), dim3(ceil_div(a.N, 256), a.M), dim3(256), 0, st, a);
    });
  });
  return true;
}
