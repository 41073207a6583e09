// Element types of the row operators (group_norm.hip, quant_rows.hip, linear_i8.hip): float, bf16 and f16 rows read and written as float,
// V consecutive elements at a time.  Addresses need the alignment of one element only: gfx950 under HSA runs in unaligned-access mode and a
// row such as 602 floats starts at any multiple of 8 bytes, so a 16-byte access is one instruction wherever it falls.
#pragma once
#include "ogl_common.h"
#include "ogl_rows.h"

typedef __bf16 ogl_bf16;
typedef _Float16 ogl_f16;

template <typename T, int V>
struct ogl_vec {
  typedef T type __attribute__((ext_vector_type(V)));
};
// rounds once, to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
template <typename T, int V>
__device__ __forceinline__ void row_store(T* __restrict__ p, const float (&v)[V]) {
  typename ogl_vec<T, V>::type t;
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = (T)v[i];
  __builtin_memcpy(p, &t, sizeof(T) * V);
}

// the same past the caches: 16 bytes that nobody reads soon
template <typename T, int V>
__device__ __forceinline__ void row_store_nt(T* __restrict__ p, const float (&v)[V]) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
  typename ogl_vec<T, V>::type t;
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = (T)v[i];
  __builtin_nontemporal_store(__builtin_bit_cast(u4, t), (u4*)p);
}
// Outputs from a quarter of the 256 MB last-level cache on are stored past it: kept there they only push out what the next launch reads, and leave it
// their write-back.
#define ROW_NT_BYTES (64ll << 20)

// A lane's piece of a run of columns: n of V elements from p on (none: n <= 0), V elements being 16 bytes.  Fetching and converting are apart, so that
// a lane can have several pieces in flight: `fetch` is one load that nothing waits for.  A piece that the run's end cuts (0 < n < V) is fetched as the
// V elements that END there; `settle` moves its elements down (zeros behind the n-th).  `tiny`: the run is shorter than V, elements come one by one.
template <typename T, int V>
struct row_piece {
  static_assert(sizeof(T) * V == 16, "a piece is 16 bytes");
  typedef typename ogl_vec<T, V>::type raw;
  static constexpr bool cuts = true;
  int n, back;
  bool tiny;
  __device__ __forceinline__ row_piece(int left, bool tiny_) : n(left), back(left > 0 && left < V && !tiny_ ? V - left : 0), tiny(tiny_) {}
  __device__ __forceinline__ raw fetch(const T* __restrict__ p) const {
    raw t = (raw)(T)0.f;
    if (!tiny) {
      if (n > 0) __builtin_memcpy(&t, p - back, 16);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < n) t[i] = p[i];
    }
    return t;
  }
  __device__ __forceinline__ void settle(raw& t) const {
    if (back) t = __builtin_bit_cast(raw, __builtin_bit_cast(unsigned __int128, t) >> (8 * (int)sizeof(T) * back));
  }
  __device__ __forceinline__ void expand(raw t, float (&v)[V]) const {
    settle(t);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)t[i];
  }
  __device__ __forceinline__ void load(const T* __restrict__ p, float (&v)[V]) const { expand(fetch(p), v); }
  __device__ __forceinline__ void store(T* __restrict__ p, const float (&v)[V], bool past) const {
    if (n >= V) {
      if (past) row_store_nt<T, V>(p, v);
      else row_store<T, V>(p, v);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < n) p[i] = (T)v[i];
    }
  }
};

// The same where every run is a multiple of V: a piece is whole or (n <= 0) not there.
template <typename T, int V>
struct row_even {
  typedef typename ogl_vec<T, V>::type raw;
  static constexpr bool cuts = false;
  static constexpr bool tiny = false;
  int n;
  __device__ __forceinline__ row_even(int left, bool) : n(left) {}
  __device__ __forceinline__ raw fetch(const T* __restrict__ p) const {
    raw t = (raw)(T)0.f;
    if (n > 0) __builtin_memcpy(&t, p, 16);
    return t;
  }
  __device__ __forceinline__ void expand(raw t, float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)t[i];
  }
  __device__ __forceinline__ void load(const T* __restrict__ p, float (&v)[V]) const { expand(fetch(p), v); }
  __device__ __forceinline__ void store(T* __restrict__ p, const float (&v)[V], bool past) const {
    if (n <= 0) return;
    if (past) row_store_nt<T, V>(p, v);
    else row_store<T, V>(p, v);
  }
};
// And where the caller has asked already: loads in a row have nothing between them.
template <typename T, int V>
struct row_whole : row_even<T, V> {
  static constexpr int n = V;
  __device__ __forceinline__ row_whole(int, bool) : row_even<T, V>(V, false) {}
};

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

// Reductions over teams of 2^k <= 64 neighbouring lanes; every lane of a team gets the same bits (each step adds two values that both lanes hold,
// and the mirrored steps pair lanes whose halves are already equal).  Steps inside 16 lanes are DPP moves (no LDS round trip).
template <int CTRL>
__device__ __forceinline__ int row_dpp(int v) {
  return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xF, 0xF, true);
}
template <typename F>
__device__ __forceinline__ int row_team(int v, int lanes, F f) {
  if (lanes > 1) v = f(v, row_dpp<0xB1>(v));                          // quad_perm 1 0 3 2
  if (lanes > 2) v = f(v, row_dpp<0x4E>(v));                          // quad_perm 2 3 0 1
  if (lanes > 4) v = f(v, row_dpp<0x141>(v));                         // row_half_mirror
  if (lanes > 8) v = f(v, row_dpp<0x140>(v));                         // row_mirror
  if (lanes > 16) v = f(v, __builtin_amdgcn_ds_swizzle(v, 0x401F));    // lane ^ 16
  if (lanes > 32) v = f(v, __shfl_xor(v, 32));
  return v;
}
__device__ __forceinline__ float row_team_sum(float v, int lanes) {
  return __builtin_bit_cast(float, row_team(__builtin_bit_cast(int, v), lanes, [](int a, int b) {
    return __builtin_bit_cast(int, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
  }));
}
__device__ __forceinline__ unsigned row_team_max(unsigned v, int lanes) {
  return (unsigned)row_team((int)v, lanes, [](int a, int b) { return (int)max((unsigned)a, (unsigned)b); });
}
