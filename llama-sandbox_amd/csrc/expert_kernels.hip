// expert_kernels.hip -- the kernels around the expert products (kernels_dispatch.h,
// kernels_i8.h) and their launches: which variant a call takes, and its grid.
#include "expert_kernels.h"

#include "../../include/moe_block.h"
#include "kernels_dispatch.h"
#include "kernels_i8.h"

static int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

// f(T{}) for the element type t.
template <typename F>
static void with_type(int t, F f) {
  if (t == MOE_GGML_F32) f(float{});
  else if (t == MOE_GGML_F16) f(_Float16{});
  else f(bf16_t{});
}

// Elements a thread takes at once: 16 bytes, or 8 elements where a side has 16 bits.
template <typename A, typename B>
constexpr int vec_of() { return sizeof(A) == 4 && sizeof(B) == 4 ? 4 : 8; }

// Workgroups a token of nv vectors: enough for the chip, no more than have work.
static int row_splits(int T, int nv) {
  const int most = ceil_div(nv, 256), want = ceil_div(2048, T);
  return most < want ? most : want;
}

void launch_dispatch(const void *x, int x_type, const int32_t *inv, int T, int k, int H, int n_rows, void *rows,
                     int rows_type, hipStream_t st) {
  with_type(x_type, [&](auto ti) {
    with_type(rows_type, [&](auto to) {
      typedef decltype(ti) TI;
      typedef decltype(to) TO;
      constexpr int V = vec_of<TI, TO>();
      hipLaunchKernelGGL((k_dispatch<TI, TO, V>), dim3(T, row_splits(T, ceil_div(H, V))), dim3(256), 0, st,
                         (const TI *)x, inv, k, H, n_rows, (TO *)rows);
    });
  });
}

void launch_combine_rows(const void *rows, int rows_type, int n_rows, const float *wts, const int32_t *inv, int T, int k,
                         int H, void *out, int out_type, hipStream_t st) {
  with_type(rows_type, [&](auto ti) {
    with_type(out_type, [&](auto to) {
      typedef decltype(ti) TI;
      typedef decltype(to) TO;
      constexpr int V = vec_of<TI, TO>();
      hipLaunchKernelGGL((k_combine_rows<TI, TO, V>), dim3(T, row_splits(T, ceil_div(H, V))), dim3(256), 0, st,
                         (const TI *)rows, wts, inv, k, H, n_rows, (TO *)out);
    });
  });
}

void launch_combine_grad(const void *dout, int dout_type, const void *rows, int rows_type, int n_rows, const float *wts,
                         const int32_t *inv, int T, int k, int H, void *drows, float *dwts, hipStream_t st) {
  const long P = (long)T * k;
  with_type(dout_type, [&](auto td) {
    with_type(rows_type, [&](auto tr) {
      typedef decltype(td) TD;
      typedef decltype(tr) TR;
      constexpr int V = vec_of<TD, TR>();
      hipLaunchKernelGGL((k_combine_grad<TD, TR, V>), dim3((unsigned)((P + 3) / 4)), dim3(256), 0, st, (const TD *)dout,
                         (const TR *)rows, wts, inv, P, k, H, n_rows, (TR *)drows, dwts);
    });
  });
}

void launch_quantize_i8(const void *x, int x_type, int M, int K, int8_t *q, float *scale, hipStream_t st) {
  with_type(x_type, [&](auto t) {
    typedef decltype(t) T;
    hipLaunchKernelGGL((k_quantize_i8_any<T>), dim3(M), dim3(256), 0, st, (const T *)x, K, q, scale);
  });
}

// Tiles of at most BM rows that M rows of E experts can make.
static long i8_tiles(const i8_mm &a, int BM) {
  return a.offsets ? a.M / BM + (a.M < a.E ? a.M : a.E) : ((long)a.M + BM - 1) / BM;
}

bool launch_matmul_i8(const i8_mm &a, int out_type, int n_cu, hipStream_t st) {
  const int nt = a.swiglu ? ceil_div(a.N / 2, 32) : ceil_div(a.N, 64);
  const long mt = i8_tiles(a, 64);
  if (mt > 65535) return false;
  with_type(out_type, [&](auto t) {
    hipLaunchKernelGGL((k_mm_i8_any<decltype(t)>), dim3(nt, (unsigned)mt), dim3(256), 0, st, a);
  });
  return true;
}
