// Rows kept in 8 bits (gfx950): a cache of `n` rows whose groups of columns carry one float32 scale each, written by quantising float rows
// and read back by row ids.
//   group of x:  a = max(max |x|, 2^-80);  s = fl32(a / Q), Q = 127 (int8) or 448 (e4m3)
//   code = the value of the format nearest the exact quotient x / s, ties to even;   read back: fl32(code * s), rounded to the output type
// A group that holds an infinity or a NaN has no finite stand-in: s = NaN, codes 0, so that it reads back as NaN (and a product with it is NaN).
// The floor on a keeps every residual below clear of the subnormals; a group smaller than it reads back as zeros.
//
// Both directions move each byte once and are bound by memory.  The quotient is x * (1 / s), within four ulps of x / s: it can pick the wrong
// neighbour only that near a border between two codes.  Those elements (about 1 in 10 000 of random data) are found by their distance from the
// border and rounded again from the exact residual x - t s (one fma: t is within an ulp of the quotient, so the residual is representable), which
// keeps the common case at half a dozen operations an element and the result that of the exact quotient.
#include <algorithm>
#include "row_types.h"

#define QR_AMAX_FLOOR 0x1p-80f

enum { QR_SLOT_RANGE = 0, QR_SLOT_SCAN = 1, QR_SLOT_OWNER = 2 };
// Up to this many rows a repeated slot is found by comparing each row's slot with the later ones in LDS; above it by two small launches that
// leave each slot's last row in a workspace.
#define QR_SCAN_ROWS 256

struct qr_write_args {
  const void* x;
  int64_t ldx;
  int64_t m;
  int width;
  const int64_t* slots;
  int64_t start;
  unsigned char* codes;
  int64_t ldc;
  float* scales;
  int64_t n;
  int group, G, log_lanes;
  ogl_div by_g;
  const int32_t* owner;
  int mode;
};

// x / s rounded to odd: the 24-bit quotient with its last bit standing for everything behind it, so that one rounding to fewer bits (two or
// more fewer) is the rounding of the exact quotient.  inv = fl(1 / s): x inv is within an ulp of the quotient, its residual then exact, and one step
// with it correctly rounded (Markstein).
__device__ __forceinline__ float qr_quotient_odd(float x, float s, float inv) {
  float t = x * inv;
  t = __builtin_fmaf(__builtin_fmaf(-t, s, x), inv, t);
  const float r = __builtin_fmaf(-t, s, x);
  if (r == 0.f || t == 0.f) return t;
  const unsigned b = __builtin_bit_cast(unsigned, t);
  const bool beyond = (r > 0.f) == (t > 0.f);                       // the exact quotient lies further from zero than t
  return __builtin_bit_cast(float, (beyond ? b : b - 1u) | 1u);
}

// N quotients (N = 4 or 8) -> N codes in N / 4 dwords.  FMT 0: int8, 1: e4m3.  `near`: some quotient lies so near a border between two codes that
// its rounding may differ from the exact quotient's.
//   int8: t + 1.5 2^23 is rint(t) in the low byte (two's complement); near a border the distance of t from it (exact) is over 0.49995, half a step
//         less four ulps of 127 (3.1e-5).
//   e4m3: the 20 bits behind the kept three are within 32 ulps of 0x80000.  Quotients below 2^-6, where the grid is 2^-9 wide, count as near (zeros do not).
template <int FMT, int N>
__device__ __forceinline__ void qr_pack(const float (&t)[N], uint32_t (&out)[N / 4], bool& near) {
  if constexpr (FMT == 0) {
    const float magic = 12582912.f;
    float far = 0.f;
    uint32_t u[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float m = t[i] + magic;
      u[i] = __builtin_bit_cast(uint32_t, m);
      far = fmaxf(far, __builtin_fabsf(t[i] - (m - magic)));
    }
    near = far > 0.49995f;
#pragma unroll
    for (int d = 0; d < N / 4; ++d) {
      const uint32_t lo = __builtin_amdgcn_perm(u[4 * d + 1], u[4 * d], 0x0C0C0400u), hi = __builtin_amdgcn_perm(u[4 * d + 3], u[4 * d + 2], 0x0C0C0400u);
      out[d] = lo | (hi << 16);
    }
  } else {
    uint32_t border = ~0u, low = ~0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t b = __builtin_bit_cast(uint32_t, t[i]);
      border = min(border, ((b + 0x20u) ^ 0x80000u) & 0xFFFFFu);
      low = min(low, (b << 1) - 1u);
    }
    near = border <= 0x40u || low < (0x3C800000u << 1) - 1u;           // 0x3C800000: 2^-6
#pragma unroll
    for (int d = 0; d < N / 4; ++d) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * d], t[4 * d + 1], 0, false);
      out[d] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(t[4 * d + 2], t[4 * d + 3], w, true);
    }
  }
}

template <int FMT, int N>
__device__ __forceinline__ void qr_codes(const float (&v)[N], float s, float inv, uint32_t (&out)[N / 4]) {
  float t[N];
  bool near;
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = v[i] * inv;
  qr_pack<FMT, N>(t, out, near);
  if (near) {
    inv = 1.f / s;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = qr_quotient_odd(v[i], s, inv);
    qr_pack<FMT, N>(t, out, near);
  }
}

// The largest |x| of pieces, kept as bits: an infinity or NaN compares above every finite value.  16-bit types stay packed, two to a dword.
template <typename T>
struct qr_amax {
  typedef typename row_piece<T, 16 / sizeof(T)>::raw raw;
  uint32_t a = 0;
  __device__ __forceinline__ void add(raw t) {
    uint32_t d[4];
    __builtin_memcpy(d, &t, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        a = max(a, d[i] & 0x7FFFFFFFu);
      } else {
        typedef unsigned short us2 __attribute__((ext_vector_type(2)));
        a = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, a), __builtin_bit_cast(us2, d[i] & 0x7FFF7FFFu)));
      }
    }
  }
  __device__ __forceinline__ uint32_t bits() const {                  // of the value as a float32
    if constexpr (sizeof(T) == 4) return a;
    else return __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(T, (unsigned short)max(a & 0xFFFFu, a >> 16)));
  }
};
// N codes at e0 (a multiple of N: 4- or 8-byte aligned)
template <int N>
__device__ __forceinline__ void qr_store(unsigned char* cp, int e0, const uint32_t (&c)[N / 4]) {
  if constexpr (N == 4) *(uint32_t*)(cp + e0) = c[0];
  else *(uint2*)(cp + e0) = make_uint2(c[0], c[1]);
}

// s = fl(a / Q): a times fl(1 / Q), corrected by its exact residual (correctly rounded: fl(1 / Q) is, and nothing here is subnormal); inv: 1 / s to
// an ulp.
template <int FMT>
__device__ __forceinline__ void qr_scale(unsigned amax_bits, float& s, float& inv) {
  constexpr float Q = FMT == 0 ? 127.f : 448.f, R = 1.f / Q;
  const bool finite = amax_bits < 0x7F800000u;
  const float a = finite ? fmaxf(__builtin_bit_cast(float, amax_bits), QR_AMAX_FLOOR) : 1.f;
  const float t = a * R;
  s = __builtin_fmaf(__builtin_fmaf(-t, Q, a), R, t);
  inv = __builtin_amdgcn_rcpf(s);
  if (!finite) s = __builtin_nanf("");
}

// where row i goes: its slot, or -1 (padding, outside the cache, or a later row has the same slot).  `later` holds the slots in LDS (SCAN).
__device__ __forceinline__ int64_t qr_target(const qr_write_args& A, int64_t i, const int64_t* later, int lane, int lanes) {
  if (A.mode == QR_SLOT_RANGE) return A.start + i;
  if (A.mode == QR_SLOT_OWNER) {
    const int64_t slot = A.slots[i];
    return slot >= 0 && slot < A.n && A.owner[slot] == (int32_t)i ? slot : -1;
  }
  const int64_t slot = later[i];
  bool again = false;
  for (int j = (int)i + 1 + lane; j < (int)A.m; j += lanes) again |= later[j] == slot;
  return !row_team_max(again, lanes) && slot >= 0 && slot < A.n ? slot : -1;
}

// One team of 2^k lanes per (row, group), NC pieces of 16 bytes a lane held in registers between the maximum and the codes: the row is read once.
// What a team does once for its group (slot, addresses, scale) costs as much as 60 codes, and the vector units bound this kernel, not the memory, as
// soon as that is spread over few: a lane takes up to 40 elements, a team so few lanes as that gives (131072 rows of 8 x 128 bf16: 16 lanes of 8
// elements 113 us, 4 lanes of 32 99 us).
template <typename T, int FMT, int NC>
__global__ void __launch_bounds__(256) k_quant_rows(qr_write_args A) {
  __shared__ int64_t later[QR_SCAN_ROWS];
  if (A.mode == QR_SLOT_SCAN) {
    for (int j = threadIdx.x; j < (int)A.m; j += 256) later[j] = A.slots[j];
    __syncthreads();
  }
  constexpr int N = 16 / sizeof(T);
  const int lanes = 1 << A.log_lanes;
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t first = (int64_t)blockIdx.x * (256 >> A.log_lanes);   // the block's first (row, group), then 32-bit steps from there
  const int64_t row0 = first / A.G;
  const uint32_t k = (uint32_t)(first - row0 * A.G) + (threadIdx.x >> A.log_lanes), up = A.by_g.div(k);
  const bool live = up < (uint32_t)min(A.m - row0, (int64_t)INT32_MAX);   // (every lane stays for the shuffles)
  const uint32_t group = live ? k - up * (uint32_t)A.G : 0u;
  const int64_t slot = qr_target(A, row0 + (live ? up : 0u), later, lane, lanes);
  const int base = (int)group * A.group;
  const int end = live ? min(base + A.group, A.width) : 0;
  const T* xp = (const T*)A.x + row0 * A.ldx + (uint64_t)(live ? up : 0u) * (uint32_t)A.ldx;
  const bool tiny = A.width < N;
  typename row_piece<T, N>::raw raw[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e0 = base + ((c << A.log_lanes) + lane) * N;
    raw[c] = row_piece<T, N>(end - e0, tiny).fetch(xp + e0);
  }
  qr_amax<T> most;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    row_piece<T, N>(end - base - ((c << A.log_lanes) + lane) * N, tiny).settle(raw[c]);
    most.add(raw[c]);
  }
  const uint32_t amax = row_team_max(most.bits(), lanes);
  if (!live || slot < 0) return;
  float s, inv;
  qr_scale<FMT>(amax, s, inv);
  const bool bad = amax >= 0x7F800000u;
  unsigned char* cp = A.codes + (uint64_t)(uint32_t)slot * (uint32_t)A.ldc;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e0 = base + ((c << A.log_lanes) + lane) * N;
    if (e0 < end) {
      float v[N];
      uint32_t w[N / 4] = {};
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = (float)raw[c][i];
      if (!bad) qr_codes<FMT, N>(v, s, inv, w);
      qr_store<N>(cp, e0, w);
    }
  }
  if (lane == 0) A.scales[(uint64_t)(uint32_t)slot * (uint32_t)A.G + group] = s;
  if ((int)group == A.G - 1)                                          // zeros behind the last column: the products read whole 64-byte steps
    for (int e = ((end + N - 1) & -N) + lane * 4; e < (int)A.ldc; e += lanes * 4) *(uint32_t*)(cp + e) = 0u;
}

// A group wider than the registers of a wave: a block per (row, group), the row read twice (the second time from the L2).
template <typename T, int FMT>
__global__ void __launch_bounds__(256) k_quant_rows_wide(qr_write_args A) {
  __shared__ int64_t later[QR_SCAN_ROWS];
  __shared__ unsigned wave_max[4];
  if (A.mode == QR_SLOT_SCAN) {
    for (int j = threadIdx.x; j < (int)A.m; j += 256) later[j] = A.slots[j];
    __syncthreads();
  }
  constexpr int N = 16 / sizeof(T);
  const int64_t i = blockIdx.x / A.G;
  const int g = (int)(blockIdx.x - i * A.G);
  const int64_t slot = qr_target(A, i, later, threadIdx.x & 63, 64);
  if (slot < 0) return;                                              // (the same for the whole block: every wave compares all later rows)
  const T* xp = (const T*)A.x + i * A.ldx;
  const int base = g * A.group;
  const int end = min(base + A.group, A.width);
  qr_amax<T> most;
  for (int e0 = base + threadIdx.x * N; e0 < end; e0 += 256 * N) {
    const row_piece<T, N> P(end - e0, false);
    typename row_piece<T, N>::raw raw = P.fetch(xp + e0);
    P.settle(raw);
    most.add(raw);
  }
  uint32_t amax = row_team_max(most.bits(), 64);
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = amax;
  __syncthreads();
  amax = max(max(wave_max[0], wave_max[1]), max(wave_max[2], wave_max[3]));
  float s, inv;
  qr_scale<FMT>(amax, s, inv);
  const bool bad = amax >= 0x7F800000u;
  unsigned char* cp = A.codes + slot * A.ldc;
  for (int e0 = base + threadIdx.x * N; e0 < end; e0 += 256 * N) {
    float v[N];
    uint32_t w[N / 4] = {};
    row_piece<T, N>(end - e0, false).load(xp + e0, v);
    if (!bad) qr_codes<FMT, N>(v, s, inv, w);
    qr_store<N>(cp, e0, w);
  }
  if (threadIdx.x == 0) A.scales[slot * A.G + g] = s;
  if (g == A.G - 1)
    for (int e = ((end + N - 1) & -N) + threadIdx.x * 4; e < (int)A.ldc; e += 1024) *(uint32_t*)(cp + e) = 0u;
}

// Repeated slots: the last row stands.  owner[slot] is cleared at the slots of this call only, then takes the largest row index: no state is
// kept from one call to the next, and the maximum does not depend on the order of the atomics.
__global__ void __launch_bounds__(256) k_quant_owner_clear(const int64_t* __restrict__ slots, int64_t m, int64_t n, int32_t* __restrict__ owner) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= m) return;
  const int64_t s = slots[i];
  if (s >= 0 && s < n) owner[s] = -1;
}
__global__ void __launch_bounds__(256) k_quant_owner_max(const int64_t* __restrict__ slots, int64_t m, int64_t n, int32_t* __restrict__ owner) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= m) return;
  const int64_t s = slots[i];
  if (s >= 0 && s < n) atomicMax(owner + s, (int32_t)i);
}

// CH codes times their scale (keep = 0: zeros, whatever was loaded)
template <int FMT, int CH>
__device__ __forceinline__ void qr_expand(const uint32_t (&c)[CH / 4], uint32_t keep, float s, float (&v)[CH]) {
#pragma unroll
  for (int d = 0; d < CH / 4; ++d) {
    const int w = (int)(c[d] & keep);
    if constexpr (FMT == 0) {
#pragma unroll
      for (int b = 0; b < 4; ++b) v[4 * d + b] = (float)(int)(signed char)(w >> (8 * b)) * s;
    } else {
      v[4 * d] = __builtin_amdgcn_cvt_f32_fp8(w, 0) * s;
      v[4 * d + 1] = __builtin_amdgcn_cvt_f32_fp8(w, 1) * s;
      v[4 * d + 2] = __builtin_amdgcn_cvt_f32_fp8(w, 2) * s;
      v[4 * d + 3] = __builtin_amdgcn_cvt_f32_fp8(w, 3) * s;
    }
  }
  // The product is rounded to float32, then to the type.  Without this (it emits nothing) the compiler may make one v_fma_mixlo_f16 of both, which
  // rounds once.
#pragma unroll
  for (int e = 0; e < CH; ++e) asm("" : "+v"(v[e]));
}

// Read back, rows by id or in order: 16 bytes of output a thread and store (CH columns), REP of them 256 chunks apart with their loads issued
// together.  Every thread of the grid has chunks (ceil(width / CH) of them in a row), so narrow rows waste no lanes.
template <typename T, int FMT, int REP>
__global__ void __launch_bounds__(256) k_dequant_rows(const unsigned char* __restrict__ codes, int64_t ldc, const float* __restrict__ scales, int64_t n,
                                                      int width, int G, const int64_t* __restrict__ rows, int64_t m, ogl_div per_row, ogl_div per_group,
                                                      T* __restrict__ out, int64_t ldo, bool past) {
  constexpr int CH = 16 / sizeof(T);
  const int64_t first = (int64_t)blockIdx.x * (256 * REP);           // row and chunk of the block's first thread, then 32-bit steps from there
  const int64_t row0 = first / per_row.d;
  const uint32_t k0 = (uint32_t)(first - row0 * per_row.d) + threadIdx.x;
  uint32_t c[REP][CH / 4];
  float s[REP];
  int64_t at[REP];
  int e0[REP];
#pragma unroll
  for (int q = 0; q < REP; ++q) {
    const uint32_t k = k0 + q * 256, up = per_row.div(k);
    at[q] = row0 + up;
    const uint32_t chunk = k - up * per_row.d;
    e0[q] = (int)chunk * CH;
    const int64_t i = min(at[q], m - 1);
    const int64_t r = rows ? rows[i] : i;
    const bool ok = r >= 0 && r < n;
#pragma unroll
    for (int d = 0; d < CH / 4; ++d) c[q][d] = 0;
    s[q] = 0.f;
    if (ok) {
      __builtin_memcpy(c[q], codes + (uint64_t)(uint32_t)r * (uint32_t)ldc + e0[q], CH);
      s[q] = scales[(uint64_t)(uint32_t)r * (uint32_t)G + per_group.div(chunk)];
    }
  }
#pragma unroll
  for (int q = 0; q < REP; ++q) {
    if (at[q] >= m) continue;
    float v[CH];
    qr_expand<FMT, CH>(c[q], ~0u, s[q], v);
    T* op = out + at[q] * ldo + e0[q];
    if (e0[q] + CH <= width) {
      if (past) row_store_nt<T, CH>(op, v);
      else row_store<T, CH>(op, v);
    } else {
#pragma unroll
      for (int b = 0; b < CH; ++b)
        if (e0[q] + b < width) op[b] = (T)v[b];
    }
  }
}

// Many rows that are wide enough for a wave each: a wave takes R rows one below the other, so ids, row addresses and the scale of a whole row are
// scalars, and a chunk costs its loads, conversions and store.
template <typename T, int FMT, int R>
__global__ void __launch_bounds__(256) k_dequant_wide(const unsigned char* __restrict__ codes, int64_t ldc, const float* __restrict__ scales, int64_t n,
                                                      int width, int G, const int64_t* __restrict__ rows, int64_t m, int per_row, ogl_div per_group,
                                                      T* __restrict__ out, int64_t ldo, bool past) {
  constexpr int CH = 16 / sizeof(T);
  const int lane = threadIdx.x & 63;
  const int64_t row0 = ((int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * R;
  if (row0 >= m) return;
  const unsigned char* cp[R];
  const float* sp[R];
  uint32_t keep[R];                                                    // all ones: the row is there
  float whole[R];
#pragma unroll
  for (int q = 0; q < R; ++q) {
    const int64_t i = min(row0 + q, m - 1);
    const int64_t r = rows ? rows[i] : i;
    const bool ok = r >= 0 && r < n;
    cp[q] = codes + (ok ? r : 0) * ldc;
    sp[q] = scales + (ok ? r : 0) * G;
    keep[q] = ok ? ~0u : 0u;
    whole[q] = ok ? sp[q][0] : 0.f;
  }
  for (int chunk = lane; chunk < per_row; chunk += 64) {
    const int e0 = chunk * CH;
    uint32_t c[R][CH / 4];
    float s[R];
#pragma unroll
    for (int q = 0; q < R; ++q) __builtin_memcpy(c[q], cp[q] + e0, CH);
    if (G == 1) {
#pragma unroll
      for (int q = 0; q < R; ++q) s[q] = whole[q];
    } else {
      const int g = (int)per_group.div((uint32_t)chunk);
#pragma unroll
      for (int q = 0; q < R; ++q) s[q] = keep[q] ? sp[q][g] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < R; ++q) {
      if (row0 + q >= m) break;
      float v[CH];
      qr_expand<FMT, CH>(c[q], keep[q], s[q], v);
      T* op = out + (row0 + q) * ldo + e0;
      if (e0 + CH <= width) {
        if (past) row_store_nt<T, CH>(op, v);
        else row_store<T, CH>(op, v);
      } else {
#pragma unroll
        for (int b = 0; b < CH; ++b)
          if (e0 + b < width) op[b] = (T)v[b];
      }
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------------
static bool qr_cache_ok(const void* codes, int64_t ldc, int format, const void* scales, int64_t n, int width, int group) {
  if (n < 0 || n > UINT32_MAX || width < 1 || group < 1 || (format != OGL_ROWS_INT8 && format != OGL_ROWS_E4M3)) return false;
  if (ldc < width || ldc % 64 != 0 || ldc > INT32_MAX) return false;
  if (group < width && group % 8 != 0) return false;
  if (n > 0 && (!codes || !scales || ((uintptr_t)codes & 63) || ((uintptr_t)scales & 3))) return false;
  return true;
}

extern "C" int64_t ogl_quant_rows_workspace_bytes(int64_t m, int64_t n, int by_slots) {
  if (m < 0 || n < 0) return OGL_EINVAL;
  return by_slots && m > QR_SCAN_ROWS ? 4 * n : 0;
}

template <typename T, int FMT>
static int qr_launch_write(qr_write_args A, hipStream_t st) {
  const int pieces = (int)ogl_cdiv(std::min(A.group, A.width), 16 / (int)sizeof(T));   // of a group
  const int most = sizeof(T) == 4 ? 10 : 5;                           // a lane: 40 elements
  const int64_t teams = A.m * (int64_t)A.G;
  A.log_lanes = 0;                                                    // (four lanes at least: 64 bytes side by side)
  while ((1 << A.log_lanes) < pieces && ((1 << A.log_lanes) < 4 || (most << A.log_lanes) < pieces)) ++A.log_lanes;
  const bool wide = A.log_lanes > 6;
  if ((teams << (wide ? 8 : A.log_lanes)) > UINT32_MAX - 256) return OGL_EINVAL;   // the launch has at most 2^32 - 1 threads
  if (wide) {
    hipLaunchKernelGGL((k_quant_rows_wide<T, FMT>), dim3((unsigned)teams), dim3(256), 0, st, A);
    return OGL_OK;
  }
  const int nc = (int)ogl_cdiv(pieces, 1 << A.log_lanes);
  const dim3 grid((unsigned)ogl_cdiv(teams, 256 >> A.log_lanes));
#define QR_CASE(NC) hipLaunchKernelGGL((k_quant_rows<T, FMT, NC>), grid, dim3(256), 0, st, A)
  if (nc <= 1) QR_CASE(1);
  else if (nc <= 2) QR_CASE(2);
  else if (nc <= 3) QR_CASE(3);
  else if (nc <= 5) QR_CASE(5);
  else if constexpr (sizeof(T) == 4) {
    if (nc <= 8) QR_CASE(8);
    else QR_CASE(10);
  }
#undef QR_CASE
  return OGL_OK;
}

extern "C" int ogl_quant_rows_write(const void* x, int64_t ldx, int x_type, int64_t m, int width, const int64_t* slots, int64_t start, void* codes,
                                    int64_t ldc, int format, float* scales, int64_t n, int group, void* workspace, int64_t workspace_bytes,
                                    ogl_stream_t stream) {
  if (m < 0 || ldx < width || x_type < OGL_F32 || x_type > OGL_F16 || !qr_cache_ok(codes, ldc, format, scales, n, width, group)) return OGL_EINVAL;
  if (!slots && (start < 0 || start > n || m > n - start)) return OGL_EINVAL;
  if (m == 0 || n == 0) return OGL_OK;
  if (!x || m > INT32_MAX || (m > 1 && ldx > INT32_MAX) || ((uintptr_t)x & (x_type == OGL_F32 ? 3 : 1))) return OGL_EINVAL;
  qr_write_args A;
  A.x = x; A.ldx = ldx; A.m = m; A.width = width; A.slots = slots; A.start = start;
  A.codes = (unsigned char*)codes; A.ldc = ldc; A.scales = scales; A.n = n;
  A.group = std::min(group, (width + 7) & ~7);                       // (a group as wide as the row: base + group stays small)
  A.G = (int)ogl_cdiv(width, A.group);
  A.by_g = ogl_div::make((uint32_t)A.G);
  A.owner = (const int32_t*)workspace;
  A.mode = !slots ? QR_SLOT_RANGE : m <= QR_SCAN_ROWS ? QR_SLOT_SCAN : QR_SLOT_OWNER;
  if (m * (int64_t)A.G > INT32_MAX) return OGL_EINVAL;               // teams of the launch
  hipStream_t st = (hipStream_t)stream;
  if (A.mode == QR_SLOT_OWNER) {
    if (!workspace || workspace_bytes < 4 * n || ((uintptr_t)workspace & 3)) return OGL_EWORKSPACE;
    hipLaunchKernelGGL(k_quant_owner_clear, dim3((unsigned)ogl_cdiv(m, 256)), dim3(256), 0, st, slots, m, n, (int32_t*)workspace);
    hipLaunchKernelGGL(k_quant_owner_max, dim3((unsigned)ogl_cdiv(m, 256)), dim3(256), 0, st, slots, m, n, (int32_t*)workspace);
    OGL_CHECK_LAUNCH();
  }
  int rc;
  if (format == OGL_ROWS_INT8)
    rc = x_type == OGL_F32 ? qr_launch_write<float, 0>(A, st) : x_type == OGL_BF16 ? qr_launch_write<ogl_bf16, 0>(A, st) : qr_launch_write<ogl_f16, 0>(A, st);
  else
    rc = x_type == OGL_F32 ? qr_launch_write<float, 1>(A, st) : x_type == OGL_BF16 ? qr_launch_write<ogl_bf16, 1>(A, st) : qr_launch_write<ogl_f16, 1>(A, st);
  if (rc != OGL_OK) return rc;
  OGL_CHECK_LAUNCH();
  return OGL_OK;
}

extern "C" int ogl_quant_rows_read(const void* codes, int64_t ldc, int format, const float* scales, int64_t n, int width, int group,
                                   const int64_t* rows, int64_t m, void* out, int64_t ldo, int out_type, ogl_stream_t stream) {
  if (m < 0 || ldo < width || out_type < OGL_F32 || out_type > OGL_F16 || !qr_cache_ok(codes, ldc, format, scales, n, width, group)) return OGL_EINVAL;
  if (!rows && m > n) return OGL_EINVAL;
  if (m == 0) return OGL_OK;
  if (!out || ((uintptr_t)out & (out_type == OGL_F32 ? 3 : 1))) return OGL_EINVAL;
  const int ch = out_type == OGL_F32 ? 4 : 8;                         // columns a 16-byte store
  const int per_row = (int)ogl_cdiv(width, ch);
  const int64_t chunks = m * (int64_t)per_row;
  if (m > INT32_MAX || chunks > UINT32_MAX - 1024) return OGL_EINVAL;
  const int gw = std::min(group, (width + 7) & ~7);
  const int G = (int)ogl_cdiv(width, gw);
  const ogl_div dr = ogl_div::make((uint32_t)per_row), dg = ogl_div::make((uint32_t)((gw + ch - 1) / ch));
  hipStream_t st = (hipStream_t)stream;
  // Four chunks a thread where that still leaves eight blocks a CU: the chain id -> row -> store is long (232965 gathered rows of 602 to float32: 1
  // chunk 204 us, 2 186 us, 4 167 us, 8 157 us; with stores past the caches 192, -, 164, 166 us and the next launch's 158 us become 124 us).
  const bool many = chunks >= 4 * 2048 * 256;
  const bool past = chunks * 16 >= ROW_NT_BYTES;
  // A wave a row (four of them) where a row keeps half a wave busy: the same rows 166 -> 144 us (two rows 147, eight 149), 131072 rows of 1024 codes
  // to bfloat16 75 -> 69 us.  The other form spends its time on addresses: a division, two products of 64 bits and two loads for 16 bytes.
  const bool wide = many && per_row >= 32 && n > 0;
#define QR_REP(T, F, R) \
  hipLaunchKernelGGL((k_dequant_rows<T, F, R>), dim3((unsigned)ogl_cdiv(chunks, 256 * (R))), dim3(256), 0, st, (const unsigned char*)codes, ldc, scales, n, \
                     width, G, rows, m, dr, dg, (T*)out, ldo, past)
#define QR_WIDE(T, F) \
  hipLaunchKernelGGL((k_dequant_wide<T, F, 4>), dim3((unsigned)ogl_cdiv(m, 4 * 4)), dim3(256), 0, st, (const unsigned char*)codes, ldc, scales, n, \
                     width, G, rows, m, per_row, dg, (T*)out, ldo, past)
#define QR_READ(T, F) \
  do { \
    if (wide) QR_WIDE(T, F); \
    else if (many) QR_REP(T, F, 4); \
    else QR_REP(T, F, 1); \
  } while (0)
  if (format == OGL_ROWS_INT8) {
    if (out_type == OGL_F32) QR_READ(float, 0);
    else if (out_type == OGL_BF16) QR_READ(ogl_bf16, 0);
    else QR_READ(ogl_f16, 0);
  } else {
    if (out_type == OGL_F32) QR_READ(float, 1);
    else if (out_type == OGL_BF16) QR_READ(ogl_bf16, 1);
    else QR_READ(ogl_f16, 1);
  }
#undef QR_READ
#undef QR_WIDE
#undef QR_REP
  OGL_CHECK_LAUNCH();
  return OGL_OK;
}
