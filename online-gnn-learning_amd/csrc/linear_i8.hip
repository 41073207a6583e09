// Products of rows kept in 8 bits (gfx950):  y[m, n] = act((sx[m] sw[n]) * sum_k x[m, k] w[n, k] + bias[n]),  x and w int8 with one float32 scale a row.
//
// The sum is exact (int32 accumulators of v_mfma_i32_16x16x64_i8; |sum| <= 128^2 K < 2^31 for K < 131072, whatever
// the bytes hold), so its order is free: waves may split K and partial sums may be joined in any order with the same result.  Rounded to float32: the
// sum once (above 2^24), sx sw, their product, and the addition of the bias.
//
// Both operands lie K-contiguous (a weight's rows are its output channels), which is what the matrix instruction reads: 16 bytes of one row a lane.
// Rows are a multiple of 64 bytes with zeros behind the last column, so there is no tail in K beyond a missing half step.  The weight rows are the
// instruction's first operand: a lane then holds 4 consecutive output columns of one row of y, a 16-byte store.
#include <algorithm>
#include "row_types.h"

typedef int v4i32 __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(1))) void* i8_gptr;
typedef __attribute__((address_space(3))) void* i8_lptr;

struct i8_args {
  const signed char* x;
  int64_t ldx;
  const float* sx;
  const int64_t* rows;   // nullable: row of x for each row of y
  int64_t nrows;         // rows of x
  const signed char* w;
  int64_t ldw;
  const float* sw;
  const float* bias;     // nullable
  void* y;
  int64_t ldy;
  int64_t M;
  int N, K64, relu;      // K64: 64-byte steps of a row
};

// the row of x behind row m of y, and whether there is one (rows outside the table count as zero rows: row 0 is read, with scale 0)
__device__ __forceinline__ int64_t i8_row(const i8_args& A, int64_t m, bool& ok) {
  const int64_t r = A.rows ? A.rows[m] : m;
  ok = r >= 0 && r < A.nrows;
  return ok ? r : 0;
}

// 4 consecutive outputs of a row from n on
template <typename T>
__device__ __forceinline__ void i8_out(const i8_args& A, int64_t m, int n, v4i32 acc, float sx, const float (&sw)[4], const float (&b)[4]) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = (float)acc[i] * (sx * sw[i]) + b[i];
    if (A.relu) v[i] = v[i] < 0.f ? 0.f : v[i];                     // (a NaN stays)
  }
  T* yp = (T*)A.y + m * A.ldy + n;
  if (n + 4 <= A.N) {
    row_store<T, 4>(yp, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < A.N) yp[i] = (T)v[i];
  }
}

// ---- few rows: every wave of a block takes a slice of K for the block's 16 output columns, straight from memory to the matrix unit ----------------
// 16 weight rows x K a block, so N / 16 blocks; the weight is read once per MT * 16 rows of x and bounds the time.
template <typename T, int MT>
__global__ void __launch_bounds__(512) k_i8_few(i8_args A) {
  constexpr int WAVES = 8;
  __shared__ v4i32 part[WAVES][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, c = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  const signed char* wp = A.w + (int64_t)min(n0 + r, A.N - 1) * A.ldw + c * 16;
  const signed char* xp[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    bool ok;
    xp[t] = A.x + i8_row(A, min(m0 + t * 16 + r, A.M - 1), ok) * A.ldx + c * 16;
  }
  v4i32 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = v4i32{0, 0, 0, 0};
#pragma unroll 4
  for (int k = wave; k < A.K64; k += WAVES) {
    const v4i32 a = *(const v4i32*)(wp + (int64_t)k * 64);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const v4i32 b = *(const v4i32*)(xp[t] + (int64_t)k * 64);
      acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc[t], 0, 0, 0);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  for (int t = wave; t < MT; t += WAVES) {
    v4i32 s = part[0][t][lane];
#pragma unroll
    for (int q = 1; q < WAVES; ++q) s += part[q][t][lane];
    const int64_t m = m0 + t * 16 + r;
    const int n = n0 + c * 4;
    if (m < A.M && n < A.N) {
      float sw[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int nn = min(n + i, A.N - 1);
        sw[i] = A.sw[nn];
        b[i] = A.bias ? A.bias[nn] : 0.f;
      }
      bool ok;
      const int64_t row = i8_row(A, m, ok);
      i8_out<T>(A, m, n, s, ok ? A.sx[row] : 0.f, sw, b);
    }
  }
}

// ---- many rows: BM x BN tiles through LDS ---------------------------------------------------------------------------------------------------------
// A stage holds 128 bytes of each row, moved by LDS-DMA (16 bytes a lane, 8 lanes a row: whole 128-byte lines).  16-byte piece p of row r holds the
// row's bytes 16 (p ^ ((r >> 1) & 7)): the 16 rows a fragment load reads side by side then touch every bank once.
#define I8_BK 128

template <typename T, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64) k_i8_tile(i8_args A, int tiles_m, int tiles_n) {
  constexpr int THREADS = WM * WN * 64;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;                 // 16 x 16 tiles of a wave
  constexpr int NA = BM * 8 / THREADS, NB = BN * 8 / THREADS;
  __shared__ __align__(128) signed char sx0[BM * I8_BK], sx1[BM * I8_BK], sw0[BN * I8_BK], sw1[BN * I8_BK];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // tiles by XCD: consecutive blocks go to different XCDs, each of which takes a contiguous run of tiles, 8 row tiles wide, so that its L2 holds them
  const int tiles = tiles_m * tiles_n;
  const int per = tiles / 8, rest = tiles % 8, xcd = blockIdx.x % 8, nth = blockIdx.x / 8;
  const int lin = xcd * per + min(xcd, rest) + nth;
  const int group = lin / (8 * tiles_n), in = lin - group * 8 * tiles_n;
  const int wide = min(8, tiles_m - group * 8);
  const int64_t m0 = (int64_t)(group * 8 + in % wide) * BM;
  const int n0 = in / wide * BN;

  // where this thread's pieces come from: its lane's byte inside a step (the same for all its rows: they lie 16 apart or more) and the rows' offsets
  // in units of 64 bytes (32 bits reach 256 GB)
  uint32_t xrow[NA], wrow[NB];
  const int piece = (tid & 7) ^ ((tid >> 4) & 7);
  const signed char *xl = A.x + piece * 16, *wl = A.w + piece * 16;
#pragma unroll
  for (int u = 0; u < NA; ++u) {
    bool ok;
    xrow[u] = (uint32_t)((uint64_t)i8_row(A, min(m0 + ((u * THREADS + tid) >> 3), A.M - 1), ok) * (uint64_t)(A.ldx >> 6));
  }
#pragma unroll
  for (int u = 0; u < NB; ++u) wrow[u] = (uint32_t)min(n0 + ((u * THREADS + tid) >> 3), A.N - 1) * (uint32_t)(A.ldw >> 6);
  const int steps = (A.K64 + 1) >> 1;
  const bool half = A.K64 & 1;                                        // the last step has 64 bytes only: its second half is read from the first again
  auto fetch = [&](int k, signed char* dx, signed char* dw) {
    const int64_t off = (int64_t)k * I8_BK - (half && k == steps - 1 && (piece & 4) ? 64 : 0);
    const signed char *xk = xl + off, *wk = wl + off;
#pragma unroll
    for (int u = 0; u < NA; ++u)
      __builtin_amdgcn_global_load_lds((i8_gptr)(xk + (uint64_t)xrow[u] * 64u), (i8_lptr)(dx + (u * THREADS + wave * 64) * 16), 16, 0, 0);
#pragma unroll
    for (int u = 0; u < NB; ++u)
      __builtin_amdgcn_global_load_lds((i8_gptr)(wk + (uint64_t)wrow[u] * 64u), (i8_lptr)(dw + (u * THREADS + wave * 64) * 16), 16, 0, 0);
  };
  const int r = lane & 15, c = lane >> 4;
  const int sw = (r >> 1) & 7;                                        // (tiles start at multiples of 16 rows: the swizzle is the lane's)
  const int xoff = (wm * TM * 16 + r) * I8_BK, woff = (wn * TN * 16 + r) * I8_BK;
  const int p0 = ((c ^ sw) * 16), p1 = (((4 + c) ^ sw) * 16);

  v4i32 acc[TN][TM];
#pragma unroll
  for (int a = 0; a < TN; ++a)
#pragma unroll
    for (int b = 0; b < TM; ++b) acc[a][b] = v4i32{0, 0, 0, 0};
  v4i32 fw[2][TN], fx[2][TM];
  auto read = [&](int h, const signed char* bx, const signed char* bw, int p) {
#pragma unroll
    for (int a = 0; a < TN; ++a) fw[h][a] = *(const v4i32*)(bw + woff + a * 16 * I8_BK + p);
#pragma unroll
    for (int b = 0; b < TM; ++b) fx[h][b] = *(const v4i32*)(bx + xoff + b * 16 * I8_BK + p);
  };
  auto multiply = [&](int h) {
#pragma unroll
    for (int b = 0; b < TM; ++b)
#pragma unroll
      for (int a = 0; a < TN; ++a) acc[a][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[h][a], fx[h][b], acc[a][b], 0, 0, 0);
  };
  // one step: the fragments of its first half are in registers (0); its second half (1) is read while they multiply, then every wave is done with
  // the stage and the next one has landed: it is refilled for the step after next while the next stage's first half is read.  (The waits are
  // builtins: the compiler then knows that the stage it reads has landed, and waits for no younger DMA.)
  auto step = [&](int k, signed char* cx, signed char* cw, const signed char* nx, const signed char* nw) {
    __builtin_amdgcn_s_waitcnt(0xC07F);                               // lgkmcnt(0): the first half, read during the last multiplication
    read(1, cx, cw, p1);
    multiply(0);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070);                               // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (k + 2 < steps) fetch(k + 2, cx, cw);
    read(0, nx, nw, p0);                                              // (behind the last step: an old stage, never multiplied)
    if (!(half && k == steps - 1)) multiply(1);
  };
  fetch(0, sx0, sw0);
  __builtin_amdgcn_s_waitcnt(0x0070);
  __builtin_amdgcn_s_barrier();
  if (steps > 1) fetch(1, sx1, sw1);
  read(0, sx0, sw0, p0);
  for (int k = 0; k < steps; k += 2) {
    step(k, sx0, sw0, sx1, sw1);
    if (k + 1 < steps) step(k + 1, sx1, sw1, sx0, sw0);
  }

#pragma unroll
  for (int a = 0; a < TN; ++a) {
    const int n = n0 + (wn * TN + a) * 16 + c * 4;
    if (n >= A.N) continue;
    float s[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int nn = min(n + i, A.N - 1);
      s[i] = A.sw[nn];
      b[i] = A.bias ? A.bias[nn] : 0.f;
    }
#pragma unroll
    for (int t = 0; t < TM; ++t) {
      const int64_t m = m0 + (wm * TM + t) * 16 + r;
      if (m >= A.M) continue;
      bool ok;
      const int64_t row = i8_row(A, m, ok);
      i8_out<T>(A, m, n, acc[a][t], ok ? A.sx[row] : 0.f, s, b);
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------------------
template <typename T, int BM, int BN, int WM, int WN>
static int i8_launch_tile(const i8_args& A, hipStream_t st) {
  const int64_t tm = ogl_cdiv(A.M, BM), tn = ogl_cdiv(A.N, BN);
  if (tm * tn * WM * WN * 64 > UINT32_MAX || tm * tn > INT32_MAX) return OGL_EINVAL;
  hipLaunchKernelGGL((k_i8_tile<T, BM, BN, WM, WN>), dim3((unsigned)(tm * tn)), dim3(WM * WN * 64), 0, st, A, (int)tm, (int)tn);
  return OGL_OK;
}

template <typename T>
static int i8_launch(const i8_args& A, hipStream_t st) {
  const unsigned nb = (unsigned)ogl_cdiv(A.N, 16);
  if (A.M <= 16) {
    hipLaunchKernelGGL((k_i8_few<T, 1>), dim3(nb, 1), dim3(512), 0, st, A);
    return OGL_OK;
  }
  if (A.M <= 64) {
    hipLaunchKernelGGL((k_i8_few<T, 4>), dim3(nb, 1), dim3(512), 0, st, A);
    return OGL_OK;
  }
  if (ogl_cdiv(A.M, 256) * ogl_cdiv(A.N, 256) >= 256) return i8_launch_tile<T, 256, 256, 2, 4>(A, st);
  return i8_launch_tile<T, 64, 64, 2, 2>(A, st);
}

extern "C" int ogl_linear_i8(const void* x, int64_t ldx, const float* sx, const int64_t* rows, int64_t nrows, int64_t M, int K, const void* w, int64_t ldw,
                             const float* sw, int N, const float* bias, int relu, void* y, int64_t ldy, int y_type, ogl_stream_t stream) {
  if (M < 0 || N < 0 || K < 1 || K > 131071 || nrows < 0 || ldx < K || ldw < K || ldx % 64 || ldw % 64 || ldy < N || y_type < OGL_F32 || y_type > OGL_F16)
    return OGL_EINVAL;
  if (!rows && M > nrows) return OGL_EINVAL;
  if (M == 0 || N == 0) return OGL_OK;
  if (!w || !sw || !y || ((uintptr_t)w & 63) || ((uintptr_t)y & (y_type == OGL_F32 ? 3 : 1)) || nrows == 0 || !x || !sx || ((uintptr_t)x & 63))
    return OGL_EINVAL;
  i8_args A;
  A.x = (const signed char*)x; A.ldx = ldx; A.sx = sx; A.rows = rows; A.nrows = nrows;
  A.w = (const signed char*)w; A.ldw = ldw; A.sw = sw; A.bias = bias;
  A.y = y; A.ldy = ldy; A.M = M; A.N = N; A.K64 = (K + 63) / 64; A.relu = relu;
  hipStream_t st = (hipStream_t)stream;
  const int rc = y_type == OGL_F32 ? i8_launch<float>(A, st) : y_type == OGL_BF16 ? i8_launch<ogl_bf16>(A, st) : i8_launch<ogl_f16>(A, st);
  if (rc != OGL_OK) return rc;
  OGL_CHECK_LAUNCH();
  return OGL_OK;
}
