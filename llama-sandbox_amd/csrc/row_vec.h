// row_vec.h -- vectors of a row's elements, of any row type, length and alignment.
#pragma once

#include "device_common.h"

typedef __bf16 bf16_t;

// V consecutive elements of a row, or as many as are left of it (the others
// 0).  Rows of any length and alignment: a whole vector is one or two 16-byte
// accesses at the type's own alignment, which global memory takes; the last
// vector of a row goes element by element.  raw: loaded, not yet converted, so
// that several can be in flight.
template <typename T, int V, bool NT = false>
struct raw_v {
  typedef T vec_t __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  vec_t v;
  __device__ __forceinline__ void load(const T *p, int left) {
    if (left >= V) {
      v = NT ? __builtin_nontemporal_load(reinterpret_cast<const vec_t *>(p)) : *reinterpret_cast<const vec_t *>(p);
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) v[i] = i < left ? p[i] : (T)0.0f;
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ void load_v(const T *p, int left, float (&f)[V]) {
  raw_v<T, V> r;
  r.load(p, left);
#pragma unroll
  for (int i = 0; i < V; i++) f[i] = (float)r.v[i];
}

template <typename T, int V, bool NT = false>
__device__ __forceinline__ void store_v(T *p, int left, const float (&f)[V]) {
  typedef typename raw_v<T, V>::vec_t vec_t;
  if (left >= V) {
    vec_t v;
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = (T)f[i];
    if (NT) __builtin_nontemporal_store(v, reinterpret_cast<vec_t *>(p));
    else *reinterpret_cast<vec_t *>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (i < left) p[i] = (T)f[i];
  }
}
