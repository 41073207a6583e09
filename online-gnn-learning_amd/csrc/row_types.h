// Element types of the row operators (group_norm.hip, quant_rows.hip, linear_i8.hip): float, bf16 and f16 rows read and written as float,
// V consecutive elements at a time.  Addresses need the alignment of one element only: gfx950 under HSA runs in unaligned-access mode and a
// row such as 602 floats starts at any multiple of 8 bytes, so a 16-byte access is one instruction wherever it falls.
#pragma once
#include "ogl_common.h"

typedef __bf16 ogl_bf16;
typedef _Float16 ogl_f16;

template <typename T, int V>
struct ogl_vec {
  typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T>
struct ogl_vec<T, 1> {
  typedef T type;
};

template <typename T, int V>
__device__ __forceinline__ void row_load(const T* __restrict__ p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = (float)*p;
  } else {
    typename ogl_vec<T, V>::type t;
    __builtin_memcpy(&t, p, sizeof(T) * V);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)t[i];
  }
}
// rounds once, to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
template <typename T, int V>
__device__ __forceinline__ void row_store(T* __restrict__ p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = (T)v[0];
  } else {
    typename ogl_vec<T, V>::type t;
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = (T)v[i];
    __builtin_memcpy(p, &t, sizeof(T) * V);
  }
}

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 as a multiplication: m = ceil(2^(31 + s) / d) with 2^s >= d, so m d = 2^(31 + s) + e, e < d <= 2^s,
// and n m / 2^(31 + s) exceeds n / d by n e / (d 2^(31 + s)) < 1 / d: the floor is the quotient.  m < 2^32.
struct ogl_div {
  uint32_t m, d;
  int s;
  static ogl_div make(uint32_t d) {
    ogl_div r;
    r.d = d;
    r.s = 0;
    while ((1ull << r.s) < d) ++r.s;
    r.m = (uint32_t)(((1ull << (31 + r.s)) + d - 1) / d);
    return r;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * m) >> (31 + s)); }
};
