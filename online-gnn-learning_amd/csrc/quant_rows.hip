// Rows kept in 8 bits (gfx950): a cache of `n` rows whose groups of columns carry one float32 scale each, written by quantising float rows
// and read back by row ids.
//   group of x:  a = max(max |x|, 2^-80);  s = fl32(a / Q), Q = 127 (int8) or 448 (e4m3)
//   code = the value of the format nearest the exact quotient x / s, ties to even;   read back: fl32(code * s), rounded to the output type
// A group that holds an infinity or a NaN has no finite stand-in: s = NaN, codes 0, so that it reads back as NaN (and a product with it is NaN).
// The floor on a keeps every residual below clear of the subnormals; a group smaller than it reads back as zeros.
//
// Both directions move each byte once and are bound by memory.  The quotient is x * (1 / s), two roundings away from x / s: it can pick the wrong
// neighbour only within 2^-22 of a border between two codes.  Those elements (about 1 in 5 000 of random data) are found by their distance from
// the border and rounded again from the exact residual x - t s (one fma: t is within an ulp of the quotient, so the residual is representable),
// which keeps the common case at five operations an element and the result that of the exact quotient.
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
  int group, G;
  const int32_t* owner;
  int mode;
};

// x / s rounded to odd: the 24-bit quotient with its last bit standing for everything behind it, so that one rounding to fewer bits (two or
// more fewer) is the rounding of the exact quotient.  inv = fl(1 / s).
__device__ __forceinline__ float qr_quotient_odd(float x, float s, float inv) {
  float t = x * inv;
  t = __builtin_fmaf(__builtin_fmaf(-t, s, x), inv, t);             // correctly rounded (inv is, and the residual is exact)
  const float r = __builtin_fmaf(-t, s, x);
  if (r == 0.f || t == 0.f) return t;
  const unsigned b = __builtin_bit_cast(unsigned, t);
  const bool beyond = (r > 0.f) == (t > 0.f);                       // the exact quotient lies further from zero than t
  return __builtin_bit_cast(float, (beyond ? b : b - 1u) | 1u);
}

// four floats -> four codes in a dword.  FMT 0: int8, 1: e4m3
template <int FMT>
__device__ __forceinline__ unsigned qr_pack4(float a, float b, float c, float d) {
  if constexpr (FMT == 0) {
    const float magic = 12582912.f;                                  // 1.5 * 2^23: the low byte of t + magic is rint(t) in two's complement
    const unsigned p = __builtin_bit_cast(unsigned, a + magic), q = __builtin_bit_cast(unsigned, b + magic);
    const unsigned u = __builtin_bit_cast(unsigned, c + magic), v = __builtin_bit_cast(unsigned, d + magic);
    return (p & 0xFFu) | ((q & 0xFFu) << 8) | ((u & 0xFFu) << 16) | (v << 24);
  } else {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return (unsigned)w;
  }
}

// distance-from-a-border test: true where x * inv is so near a border between two codes that its rounding may differ from the exact quotient's
template <int FMT>
__device__ __forceinline__ bool qr_near_border(float t) {
  if constexpr (FMT == 0) {
    return __builtin_fabsf(t - __builtin_rintf(t)) > 0.4999f;        // t - rint(t) is exact; the error of t is below 127 * 2^-22
  } else {
    const unsigned b = __builtin_bit_cast(unsigned, t);
    const float v = t * 512.f;                                       // below 2^-6 the grid is 2^-9 wide
    const bool low = __builtin_fabsf(v - __builtin_rintf(v)) > 0.4999f && __builtin_fabsf(t) < 0.0156252f;
    return low || ((b & 0xFFFFFu) - 0x7FFF0u) <= 0x20u;              // 20 bits behind the kept three: half a step is 0x80000
  }
}

template <int FMT>
__device__ __forceinline__ uint2 qr_codes8(const float (&v)[8], float s, float inv) {
  float t[8];
  bool near = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    t[i] = v[i] * inv;
    near |= qr_near_border<FMT>(t[i]);
  }
  if (near) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = qr_quotient_odd(v[i], s, inv);
  }
  return make_uint2(qr_pack4<FMT>(t[0], t[1], t[2], t[3]), qr_pack4<FMT>(t[4], t[5], t[6], t[7]));
}

// up to 8 elements at e0 of a row of `width` (zeros behind it), and the largest |x| as bits (an infinity or NaN compares above every finite value)
template <typename T>
__device__ __forceinline__ unsigned qr_load8(const T* __restrict__ xp, int e0, int end, float (&v)[8]) {
  if (e0 + 8 <= end) {
    row_load<T, 8>(xp + e0, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e0 + i < end ? (float)xp[e0 + i] : 0.f;
  }
  unsigned a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, __builtin_bit_cast(unsigned, v[i]) & 0x7FFFFFFFu);
  return a;
}

template <int FMT>
__device__ __forceinline__ void qr_scale(unsigned amax_bits, float& s, float& inv) {
  const float a = __builtin_bit_cast(float, amax_bits);
  const bool finite = amax_bits < 0x7F800000u;
  s = fmaxf(finite ? a : 1.f, QR_AMAX_FLOOR) / (FMT == 0 ? 127.f : 448.f);
  inv = 1.f / s;
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
  int any = again;
  for (int o = 1; o < lanes; o <<= 1) any |= __shfl_xor(any, o);
  return !any && slot >= 0 && slot < A.n ? slot : -1;
}

// One team of LANES lanes per (row, group), 8 * NC columns a lane held in registers between the maximum and the codes: the row is read once.
// A wave's loads are contiguous (teams follow each other along the row).
template <typename T, int FMT, int LANES, int NC>
__global__ void __launch_bounds__(256) k_quant_rows(qr_write_args A) {
  __shared__ int64_t later[QR_SCAN_ROWS];
  if (A.mode == QR_SLOT_SCAN) {
    for (int j = threadIdx.x; j < (int)A.m; j += 256) later[j] = A.slots[j];
    __syncthreads();
  }
  const int lane = threadIdx.x % LANES;
  const int64_t team = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const bool live = team < A.m * (int64_t)A.G;                       // (every lane stays for the shuffles)
  const int64_t i = live ? team / A.G : 0;
  const int g = live ? (int)(team - i * A.G) : 0;
  const int64_t slot = qr_target(A, i, later, lane, LANES);
  const T* xp = (const T*)A.x + i * A.ldx;
  const int base = g * A.group;
  const int end = min(base + A.group, A.width);
  float v[NC][8];
  unsigned amax = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) amax = max(amax, qr_load8(xp, base + (c * LANES + lane) * 8, end, v[c]));
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) amax = max(amax, (unsigned)__shfl_xor((int)amax, o));
  if (!live || slot < 0) return;
  float s, inv;
  qr_scale<FMT>(amax, s, inv);
  const bool bad = amax >= 0x7F800000u;
  unsigned char* cp = A.codes + slot * A.ldc;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e0 = base + (c * LANES + lane) * 8;
    if (e0 < end) *(uint2*)(cp + e0) = bad ? make_uint2(0u, 0u) : qr_codes8<FMT>(v[c], s, inv);
  }
  if (lane == 0) A.scales[slot * A.G + g] = s;
  if (g == A.G - 1)                                                  // zeros behind the last column: the products read whole 64-byte steps
    for (int e = ((end + 7) & ~7) + lane * 8; e < (int)A.ldc; e += LANES * 8) *(uint2*)(cp + e) = make_uint2(0u, 0u);
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
  const int64_t i = blockIdx.x / A.G;
  const int g = (int)(blockIdx.x - i * A.G);
  const int64_t slot = qr_target(A, i, later, threadIdx.x & 63, 64);
  if (slot < 0) return;                                              // (the same for the whole block: every wave compares all later rows)
  const T* xp = (const T*)A.x + i * A.ldx;
  const int base = g * A.group;
  const int end = min(base + A.group, A.width);
  unsigned amax = 0;
  float v[8];
  for (int e0 = base + threadIdx.x * 8; e0 < end; e0 += 2048) amax = max(amax, qr_load8(xp, e0, end, v));
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) amax = max(amax, (unsigned)__shfl_xor((int)amax, o));
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = amax;
  __syncthreads();
  amax = max(max(wave_max[0], wave_max[1]), max(wave_max[2], wave_max[3]));
  float s, inv;
  qr_scale<FMT>(amax, s, inv);
  const bool bad = amax >= 0x7F800000u;
  unsigned char* cp = A.codes + slot * A.ldc;
  for (int e0 = base + threadIdx.x * 8; e0 < end; e0 += 2048) {
    qr_load8(xp, e0, end, v);
    *(uint2*)(cp + e0) = bad ? make_uint2(0u, 0u) : qr_codes8<FMT>(v, s, inv);
  }
  if (threadIdx.x == 0) A.scales[slot * A.G + g] = s;
  if (g == A.G - 1)
    for (int e = ((end + 7) & ~7) + threadIdx.x * 8; e < (int)A.ldc; e += 2048) *(uint2*)(cp + e) = make_uint2(0u, 0u);
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

// Read back: 8 columns a thread (8 bytes in, 16 or 32 out), rows by id or in order; ids outside the cache yield zero rows.
// Every thread of the grid has a chunk (m * ceil(width / 8) of them in a row), so narrow rows waste no lanes.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) k_dequant_rows(const unsigned char* __restrict__ codes, int64_t ldc, const float* __restrict__ scales, int64_t n,
                                                      int width, int G, const int64_t* __restrict__ rows, int64_t m, ogl_div per_row, ogl_div per_group,
                                                      T* __restrict__ out, int64_t ldo) {
  const int64_t first = (int64_t)blockIdx.x * 256;                   // row and chunk of the block's first thread, then 32-bit steps from there
  const int64_t row0 = first / per_row.d;
  const uint32_t k = (uint32_t)(first - row0 * per_row.d) + threadIdx.x;
  const uint32_t up = per_row.div(k);
  const int64_t i = row0 + up;
  if (i >= m) return;
  const uint32_t chunk = k - up * per_row.d;
  const int e0 = (int)chunk * 8;
  const int64_t r = rows ? rows[i] : i;
  const bool ok = r >= 0 && r < n;
  float v[8];
  if (ok) {
    const uint2 c = *(const uint2*)(codes + r * ldc + e0);
    const float s = scales[r * G + per_group.div(chunk)];
    if constexpr (FMT == 0) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        v[b] = (float)(int)(signed char)(c.x >> (8 * b)) * s;
        v[4 + b] = (float)(int)(signed char)(c.y >> (8 * b)) * s;
      }
    } else {
      v[0] = __builtin_amdgcn_cvt_f32_fp8((int)c.x, 0) * s;
      v[1] = __builtin_amdgcn_cvt_f32_fp8((int)c.x, 1) * s;
      v[2] = __builtin_amdgcn_cvt_f32_fp8((int)c.x, 2) * s;
      v[3] = __builtin_amdgcn_cvt_f32_fp8((int)c.x, 3) * s;
      v[4] = __builtin_amdgcn_cvt_f32_fp8((int)c.y, 0) * s;
      v[5] = __builtin_amdgcn_cvt_f32_fp8((int)c.y, 1) * s;
      v[6] = __builtin_amdgcn_cvt_f32_fp8((int)c.y, 2) * s;
      v[7] = __builtin_amdgcn_cvt_f32_fp8((int)c.y, 3) * s;
    }
  } else {
#pragma unroll
    for (int b = 0; b < 8; ++b) v[b] = 0.f;
  }
  T* op = out + i * ldo + e0;
  if (e0 + 8 <= width) {
    row_store<T, 8>(op, v);
  } else {
#pragma unroll
    for (int b = 0; b < 8; ++b)
      if (e0 + b < width) op[b] = (T)v[b];
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------------
static bool qr_cache_ok(const void* codes, int64_t ldc, int format, const void* scales, int64_t n, int width, int group) {
  if (n < 0 || width < 1 || group < 1 || (format != OGL_ROWS_INT8 && format != OGL_ROWS_E4M3)) return false;
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
static int qr_launch_write(const qr_write_args& A, hipStream_t st) {
  const int chunks = (int)ogl_cdiv(std::min(A.group, A.width), 8);   // 8-column chunks of a group
  const int64_t teams = A.m * (int64_t)A.G;
  int64_t lanes = 1;                                                 // of a team; the launch has at most 2^32 - 1 threads
  while (lanes < 64 && lanes < chunks) lanes *= 2;
  if (teams * (chunks > 256 ? 256 : lanes) > UINT32_MAX - 256) return OGL_EINVAL;
#define QR_CASE(L, NC) \
  hipLaunchKernelGGL((k_quant_rows<T, FMT, L, NC>), dim3((unsigned)ogl_cdiv(teams, 256 / (L))), dim3(256), 0, st, A)
  if (chunks <= 1) QR_CASE(1, 1);
  else if (chunks <= 2) QR_CASE(2, 1);
  else if (chunks <= 4) QR_CASE(4, 1);
  else if (chunks <= 8) QR_CASE(8, 1);
  else if (chunks <= 16) QR_CASE(16, 1);
  else if (chunks <= 32) QR_CASE(32, 1);
  else if (chunks <= 64) QR_CASE(64, 1);
  else if (chunks <= 128) QR_CASE(64, 2);
  else if (chunks <= 256) QR_CASE(64, 4);
  else hipLaunchKernelGGL((k_quant_rows_wide<T, FMT>), dim3((unsigned)teams), dim3(256), 0, st, A);
#undef QR_CASE
  return OGL_OK;
}

extern "C" int ogl_quant_rows_write(const void* x, int64_t ldx, int x_type, int64_t m, int width, const int64_t* slots, int64_t start, void* codes,
                                    int64_t ldc, int format, float* scales, int64_t n, int group, void* workspace, int64_t workspace_bytes,
                                    ogl_stream_t stream) {
  if (m < 0 || ldx < width || x_type < OGL_F32 || x_type > OGL_F16 || !qr_cache_ok(codes, ldc, format, scales, n, width, group)) return OGL_EINVAL;
  if (!slots && (start < 0 || start > n || m > n - start)) return OGL_EINVAL;
  if (m == 0 || n == 0) return OGL_OK;
  if (!x || m > INT32_MAX || ((uintptr_t)x & (x_type == OGL_F32 ? 3 : 1))) return OGL_EINVAL;
  qr_write_args A;
  A.x = x; A.ldx = ldx; A.m = m; A.width = width; A.slots = slots; A.start = start;
  A.codes = (unsigned char*)codes; A.ldc = ldc; A.scales = scales; A.n = n;
  A.group = std::min(group, (width + 7) & ~7);                       // (a group as wide as the row: base + group stays small)
  A.G = (int)ogl_cdiv(width, A.group);
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
  const int per_row = (width + 7) / 8;
  const int64_t blocks = ogl_cdiv(m * (int64_t)per_row, 256);
  if (m > INT32_MAX || blocks > UINT32_MAX / 256) return OGL_EINVAL;
  const int gw = std::min(group, per_row * 8);
  const int G = (int)ogl_cdiv(width, gw);
  const ogl_div dr = ogl_div::make((uint32_t)per_row), dg = ogl_div::make((uint32_t)((gw + 7) / 8));
  hipStream_t st = (hipStream_t)stream;
#define QR_READ(T, F) \
  hipLaunchKernelGGL((k_dequant_rows<T, F>), dim3((unsigned)blocks), dim3(256), 0, st, (const unsigned char*)codes, ldc, scales, n, width, G, rows, m, \
                     dr, dg, (T*)out, ldo)
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
  OGL_CHECK_LAUNCH();
  return OGL_OK;
}
