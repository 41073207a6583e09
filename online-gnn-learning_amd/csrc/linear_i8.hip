// Products of rows kept in 8 bits (gfx950):  y[m, n] = act((sx[m] sw[n]) * sum_k x[m, k] w[n, k] + bias[n]),  x and w int8 with one float32 scale a row.
//
// The sum is exact (int32 accumulators of v_mfma_i32_32x32x32_i8 and 16x16x64; |sum| <= 128^2 K < 2^31 for K < 131072, whatever the bytes hold), so its
// order is free: waves may split K and partial sums may be joined in any order with the same result.  Rounded to float32: the sum once (above 2^24),
// sx sw, and, in one fused step, their product with the bias added; every form does the same, so a row's bits do not depend on the form.
//
// Both operands lie K-contiguous (a weight's rows are its output channels), which is what the matrix instruction reads: 16 bytes of one row a lane.
// Rows are a multiple of 64 bytes with zeros behind the last column, so there is no tail in K.  The weight rows are the
// instruction's first operand: a lane then holds 4 consecutive output columns of one row of y, a 16-byte store.
#include <algorithm>
#include "row_types.h"

typedef int v4i32 __attribute__((ext_vector_type(4)));
typedef int v16i32 __attribute__((ext_vector_type(16)));
typedef int i8_piece __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes of y, wherever they lie
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

// scales and bias of 4 columns (behind the last one: anything)
__device__ __forceinline__ void i8_columns(const i8_args& A, int n, float (&sw)[4], float (&b)[4]) {
  if (n + 4 <= A.N) {
    __builtin_memcpy(sw, A.sw + n, 16);
    if (A.bias) __builtin_memcpy(b, A.bias + n, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int nn = min(n + i, A.N - 1);
      sw[i] = A.sw[nn];
      if (A.bias) b[i] = A.bias[nn];
    }
  }
  if (!A.bias) b[0] = b[1] = b[2] = b[3] = 0.f;
}
// 4 outputs of a row
__device__ __forceinline__ void i8_values(const i8_args& A, v4i32 acc, float sx, const float (&sw)[4], const float (&b)[4], float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = __builtin_fmaf((float)acc[i], sx * sw[i], b[i]);
    if (A.relu) v[i] = v[i] < 0.f ? 0.f : v[i];                     // (a NaN stays)
  }
}
template <typename T>
__device__ __forceinline__ void i8_out(const i8_args& A, int64_t m, int n, v4i32 acc, float sx, const float (&sw)[4], const float (&b)[4]) {
  float v[4];
  i8_values(A, acc, sx, sw, b, v);
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
// 16 weight rows x K a block, so N / 16 blocks; the weight is read once per MT * 16 rows of x.  16 x 12288, K = 4096 takes 14.5 us, 3.5 TB/s of a weight
// that no cache holds.  A step of a wave is its loads (the weight's and those of x), a wait for them and MT products: the loop is not unrolled, and the
// waves of a CU have eight steps a block in flight between them.  Two steps at a time, 4 or 16 waves a block and loads past the caches took the same or
// longer; more steps of a wave in flight have not been tried.
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
      i8_columns(A, n, sw, b);
      bool ok;
      const int64_t row = i8_row(A, m, ok);
      i8_out<T>(A, m, n, s, ok ? A.sx[row] : 0.f, sw, b);
    }
  }
}

// ---- many rows: BM x BN tiles through LDS ---------------------------------------------------------------------------------------------------------
// A stage holds 64 bytes of each row, moved by LDS-DMA (16 bytes a lane, 4 lanes a row); four stages are a ring.  16-byte piece p of row r holds the
// row's bytes 16 (p ^ ((r >> 2) & 3)): the 16 rows a fragment load reads side by side then touch every bank once.
// A block stays on its CU and takes every blocks-th tile.  Its steps are one sequence over all its tiles, so the first ones of the next tile are on
// their way while the last ones of a tile multiply.
template <typename T, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64) k_i8_tile(i8_args A, int tiles_m, int tiles_n, int blocks) {
  constexpr int THREADS = WM * WN * 64;
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32;                 // 32 x 32 tiles of a wave
  constexpr int NA = BM * 4 / THREADS, NB = BN * 4 / THREADS;
  constexpr bool PAST = BM * BN >= 65536;
  // what a wave turns over at a time: AT of its tiles side by side (128 bytes of a row, or what there is of them), ROWS rows
  constexpr int AT = TN * 32 * (int)sizeof(T) <= 128 ? TN : 1;
  constexpr int LINE = AT * 32 * (int)sizeof(T), UNITS = LINE / 16;    // a row's run of columns: bytes, 16-byte units
  constexpr int ROWS = AT == 1 ? 32 : 16;
  constexpr int WAVE_LDS = AT == 1 ? std::max(ROWS * LINE, 256) : ROWS * LINE + AT * 32 * 8;
  static_assert(TN <= 2 && WAVE_LDS <= 4096, "a lane holds one column's scale; the stages leave each wave 4 KB");
  // (arrays of their own: the compiler then knows which stage a DMA writes, and a read of another one waits for none)
  __shared__ __align__(128) signed char x0[BM * 64], x1[BM * 64], x2[BM * 64], x3[BM * 64], w0[BN * 64], w1[BN * 64], w2[BN * 64], w3[BN * 64];
  __shared__ __align__(128) signed char turned[WM * WN * WAVE_LDS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int tiles = tiles_m * tiles_n, steps = A.K64;

  // Tiles by XCD: consecutive blocks run on different XCDs.  Each XCD has a contiguous run of tiles, 8 row tiles wide, so that its L2 holds what its
  // CUs read at a time.
  auto place = [&](int t, int64_t& m0, int& n0) {
    const int per = tiles / 8, rest = tiles % 8, xcd = t % 8, nth = t / 8;
    const int lin = xcd * per + min(xcd, rest) + nth;
    const int group = lin / (8 * tiles_n), in = lin - group * 8 * tiles_n;
    const int wide = min(8, tiles_m - group * 8);
    m0 = (int64_t)(group * 8 + in % wide) * BM;
    n0 = in / wide * BN;
  };

  // what is fetched next: step fk of tile ft (behind the last tile: the last one again, so that every step fetches the same number of pieces).  A
  // thread's pieces: its lane's bytes inside a step (the same for all its rows: they lie 16 apart or more) and the rows' offsets in units of 64 bytes
  // (32 bits reach 256 GB)
  int ft = blockIdx.x, fk = 0;
  uint32_t xrow[NA], wrow[NB];
  const int piece = ((tid & 3) ^ ((tid >> 4) & 3)) * 16;
  const signed char *xk = A.x + piece, *wk = A.w + piece;
  auto aim = [&]() {
    int64_t m0;
    int n0;
    place(ft, m0, n0);
#pragma unroll
    for (int u = 0; u < NA; ++u) {
      bool ok;
      xrow[u] = (uint32_t)((uint64_t)i8_row(A, min(m0 + ((u * THREADS + tid) >> 2), A.M - 1), ok) * (uint64_t)(A.ldx >> 6));
    }
#pragma unroll
    for (int u = 0; u < NB; ++u) wrow[u] = (uint32_t)min(n0 + ((u * THREADS + tid) >> 2), A.N - 1) * (uint32_t)(A.ldw >> 6);
  };
  auto advance = [&]() {
    if (++fk == steps) {
      fk = 0;
      if (ft + blocks < tiles) ft += blocks;
      aim();
    }
  };
  auto fetch = [&](int u, signed char* dx, signed char* dw) {          // piece u of NA + NB
    const uint64_t off = (uint64_t)fk * 64u;
    if (u < NA)
      __builtin_amdgcn_global_load_lds((i8_gptr)(xk + off + (uint64_t)xrow[u < NA ? u : 0] * 64u), (i8_lptr)(dx + (u * THREADS + wave * 64) * 16), 16, 0, 0);
    else
      __builtin_amdgcn_global_load_lds((i8_gptr)(wk + off + (uint64_t)wrow[u < NA ? 0 : u - NA] * 64u), (i8_lptr)(dw + ((u - NA) * THREADS + wave * 64) * 16),
                                       16, 0, 0);
  };
  const int r = lane & 31, c = lane >> 5;
  const int swz = (r >> 2) & 3;                                       // (tiles start at multiples of 32 rows: the swizzle is the lane's)
  const int xoff = (wm * TM * 32 + r) * 64, woff = (wn * TN * 32 + r) * 64;

  v16i32 acc[TN][TM];
  auto clear = [&]() {
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
      for (int b = 0; b < TM; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[a][b][i] = 0;
  };
  v4i32 fw[2][TN], fx[2][TM];
  auto read = [&](int s, int i, const signed char* bx, const signed char* bw) {        // of the 32 bytes s of a stage the i-th fragment, 16 bytes a lane,
    const int p = ((2 * s + c) ^ swz) * 16;                                            // in the order that the products take them
    if (i == 0 || (i > 1 && i <= TN)) {
      const int a = i == 0 ? 0 : i - 1;
      fw[s][a] = *(const v4i32*)(bw + woff + a * 32 * 64 + p);
    } else {
      const int b = i == 1 ? 0 : i - TN;
      fx[s][b] = *(const v4i32*)(bx + xoff + b * 32 * 64 + p);
    }
  };
  auto multiply = [&](int s, int i) {                                                  // the i-th of the wave's TM TN tiles
    acc[i % TN][i / TN] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[s][i % TN], fx[s][i / TN], acc[i % TN][i / TN], 0, 0, 0);
  };
  // A lane holds one row of y for each b, and of each 32 columns the quads 8 q + 4 c .. + 3.  Stored from there an instruction would write 32 bytes of
  // each of 32 rows: each wave turns its rows over in LDS and stores runs of 128 bytes (62500 x 600 float32, K = 602: 89 us without).  32 rows at a
  // time where a tile's row is 128 bytes: with longer runs of fewer rows only some lanes write, and the LDS is what the epilogue waits for (68 us so,
  // 58 us with all lanes writing).
  // PAST: the tiles of large products are stored past the caches, whose write-back of 33 MB or more otherwise meets the next tiles' reads (4096 x 4096
  // bfloat16, K = 512 20.9 -> 18.4 us; 8192 x 8192, K = 4096 293 -> 276 us).
  // Scales and bias are loaded before the first store: a load behind it would wait for it (one counter for both, in order).
  signed char* turn = turned + wave * WAVE_LDS;
  auto finish = [&](int t) {
    constexpr int E = 16 / (int)sizeof(T);
    int64_t m0;
    int n0;
    place(t, m0, n0);
    m0 += wm * TM * 32;
    n0 += wn * TN * 32;
    float sx[TM], sw = 0.f, bias = 0.f;
    if (lane < TN * 32) {
      const int n = min(n0 + lane, A.N - 1);
      sw = A.sw[n];
      if (A.bias) bias = A.bias[n];
    }
#pragma unroll
    for (int b = 0; b < TM; ++b) {
      bool ok;
      const int64_t row = i8_row(A, min(m0 + b * 32 + r, A.M - 1), ok);
      sx[b] = ok ? A.sx[row] : 0.f;
    }
    const bool full = m0 + TM * 32 <= A.M && n0 + TN * 32 <= A.N;
#pragma unroll
    for (int a = 0; a < TN; a += AT) {
      // scales [AT 32] and biases [AT 32]: behind the rows, or (one tile at a time) in their place, from where each lane takes its own first
      float* cols = (float*)(turn + (AT == 1 ? 0 : ROWS * LINE));
      const int mine = lane - a * 32;
      __builtin_amdgcn_wave_barrier();
      if (mine >= 0 && mine < AT * 32) {
        cols[mine] = sw;
        cols[AT * 32 + mine] = bias;
      }
      __builtin_amdgcn_wave_barrier();
      float w[AT == 1 ? 4 : 1][4], d[AT == 1 ? 4 : 1][4];
      if constexpr (AT == 1) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          *(float4*)w[u] = *(const float4*)(cols + u * 8 + c * 4);
          *(float4*)d[u] = *(const float4*)(cols + 32 + u * 8 + c * 4);
        }
        __builtin_amdgcn_wave_barrier();
      }
#pragma unroll
      for (int b = 0; b < TM; ++b) {
        float v[AT * 4][4];
#pragma unroll
        for (int u = 0; u < AT * 4; ++u) {
          if constexpr (AT > 1) {
            *(float4*)w[0] = *(const float4*)(cols + u * 8 + c * 4);
            *(float4*)d[0] = *(const float4*)(cols + AT * 32 + u * 8 + c * 4);
          }
          const v16i32& s = acc[a + (u >> 2)][b];
          const int q = (u & 3) * 4;
          i8_values(A, v4i32{s[q], s[q + 1], s[q + 2], s[q + 3]}, sx[b], w[AT == 1 ? u : 0], d[AT == 1 ? u : 0], v[u]);
        }
#pragma unroll
        for (int h = 0; h < 32 / ROWS; ++h) {
          const int rr = r & (ROWS - 1);
          if (ROWS == 32 || r / ROWS == h) {
#pragma unroll
            for (int u = 0; u < AT * 4; ++u) {
              const int at = (u * 8 + c * 4) * (int)sizeof(T);
              row_store<T, 4>((T*)(turn + rr * LINE + ((at >> 4) ^ (rr & (UNITS - 1))) * 16 + (at & 15)), v[u]);
            }
          }
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int it = 0; it < ROWS * UNITS / 64; ++it) {
            const int line = it * (64 / UNITS) + lane / UNITS, unit = lane % UNITS;
            const int64_t m = m0 + b * 32 + h * ROWS + line;
            const int n = n0 + a * 32 + unit * E;
            const T* from = (const T*)(turn + line * LINE + (unit ^ (line & (UNITS - 1))) * 16);
            T* yp = (T*)A.y + m * A.ldy + n;
            if (full) {
              if constexpr (PAST) __builtin_nontemporal_store(*(const i8_piece*)from, (i8_piece*)yp);
              else __builtin_memcpy(yp, from, 16);
            } else if (m < A.M && n < A.N) {
              if (n + E <= A.N) {
                __builtin_memcpy(yp, from, 16);
              } else {
                for (int i = 0; i < E; ++i)
                  if (n + i < A.N) yp[i] = from[i];
              }
            }
          }
          __builtin_amdgcn_wave_barrier();
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };
  // One step: the fragments of a stage's first 32 bytes are in registers; those of its second 32 are read while the first multiply.  Then every wave
  // has read the stage, and the next one (fetched three steps ago; two younger ones may be on their way) has landed: its first fragments are read, and
  // the stage is refilled for four steps on, while the second ones multiply.  Reads and fetches go between the products one by one: issued in one go,
  // those of all waves queue for the LDS and hold up the products behind them.  (The waits are builtins: the compiler then waits for no younger DMA.)
  constexpr int PIECES = NA + NB, TILES = TM * TN, FRAGS = TM + TN, SLOTS = TILES > FRAGS ? TILES : FRAGS;
  auto step = [&](signed char* cx, signed char* cw, const signed char* nx, const signed char* nw) {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      if (i < TILES) multiply(0, i);
      if (i < FRAGS) read(1, i, cx, cw);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_waitcnt((2 * PIECES & 15) | (2 * PIECES >> 4 << 14) | 0x0070);   // vmcnt(2 PIECES) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < (SLOTS > PIECES ? SLOTS : PIECES); ++i) {
      if (i < TILES) multiply(1, i);
      if (i < FRAGS) read(0, i, nx, nw);                              // (behind the last step: a stage that is never multiplied)
      if (i < PIECES) fetch(i, cx, cw);
      __builtin_amdgcn_sched_barrier(0);
    }
    advance();
  };
  aim();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
#pragma unroll
    for (int u = 0; u < PIECES; ++u) fetch(u, q == 0 ? x0 : q == 1 ? x1 : q == 2 ? x2 : x3, q == 0 ? w0 : q == 1 ? w1 : q == 2 ? w2 : w3);
    advance();
  }
  __builtin_amdgcn_s_waitcnt(0x0070);                                 // (all of them: no path into the loop then has a stage on its way)
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int i = 0; i < FRAGS; ++i) read(0, i, x0, w0);
  int at = 0;                                                          // the stage that the sequence of steps has come to
  for (int t = blockIdx.x; t < tiles; t += blocks) {
    clear();
    for (int k = 0;;) {
      if (at == 0) {
        step(x0, w0, x1, w1);
        at = 1;
        if (++k == steps) break;
      }
      if (at == 1) {
        step(x1, w1, x2, w2);
        at = 2;
        if (++k == steps) break;
      }
      if (at == 2) {
        step(x2, w2, x3, w3);
        at = 3;
        if (++k == steps) break;
      }
      step(x3, w3, x0, w0);
      at = 0;
      if (++k == steps) break;
    }
    finish(t);
  }
  __builtin_amdgcn_s_waitcnt(0x0070);                                 // what was fetched behind the last step
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------------------
template <typename T, int BM, int BN, int WM, int WN>
static int i8_launch_tile(const i8_args& A, int blocks, hipStream_t st) {
  const int64_t tm = ogl_cdiv(A.M, BM), tn = ogl_cdiv(A.N, BN);
  if (tm * tn > INT32_MAX) return OGL_EINVAL;
  blocks = (int)std::min<int64_t>(tm * tn, blocks);
  hipLaunchKernelGGL((k_i8_tile<T, BM, BN, WM, WN>), dim3((unsigned)blocks), dim3(WM * WN * 64), 0, st, A, (int)tm, (int)tn, blocks);
  return OGL_OK;
}

template <typename T>
static int i8_launch(const i8_args& A, hipStream_t st) {
  const unsigned nb = (unsigned)ogl_cdiv(A.N, 16);
  if (A.M <= 16) {
    if ((int64_t)nb * 512 > (int64_t)UINT32_MAX) return OGL_EINVAL;   // the launch has at most 2^32 - 1 threads
    hipLaunchKernelGGL((k_i8_few<T, 1>), dim3(nb, 1), dim3(512), 0, st, A);
    return OGL_OK;
  }
  // Up to 64 rows while the blocks of 16 columns fit one a CU: behind that they read x as often as w.  32 x 4096, K = 4096: 11.7 us, in tiles 12.5 us;
  // 32 x 6144 16.2 us, 12.6 us; 64 x 12288 30.7 us, 14.4 us; 64 x 600, K = 602 4.4 us, 5.4 us.
  if (A.M <= 64 && nb <= 256) {
    hipLaunchKernelGGL((k_i8_few<T, 4>), dim3(nb, 1), dim3(512), 0, st, A);
    return OGL_OK;
  }
  // Large tiles read each operand less often, small ones fill the card.  256 x 256 (one block a CU) from a tile a CU on: 4096 x 4096, K = 4096 70 us,
  // in 128 x 128 tiles 101 us, in 64 x 64 ones 145 us.  128 x 128 (two blocks a CU) from 3 tiles for 4 CUs on, 1024 x 4096, K = 4096: 26 us, 64 x 64
  // 39 us, 256 x 256 46 us; 512 x 4096 (128 tiles) 22.6 us, 64 x 64 21.2 us; with few steps the epilogue weighs more, 16000 x 600, K = 602 (625 tiles):
  // 25 us, 64 x 64 23 us.
  if (ogl_cdiv(A.M, 256) * ogl_cdiv(A.N, 256) >= 256) return i8_launch_tile<T, 256, 256, 2, 4>(A, 256, st);
  if (ogl_cdiv(A.M, 128) * ogl_cdiv(A.N, 128) >= 192 && A.K64 >= 16) return i8_launch_tile<T, 128, 128, 2, 2>(A, 512, st);
  return i8_launch_tile<T, 64, 64, 2, 2>(A, 768, st);
}

extern "C" int ogl_linear_i8(const void* x, int64_t ldx, const float* sx, const int64_t* rows, int64_t nrows, int64_t M, int K, const void* w, int64_t ldw,
                             const float* sw, int N, const float* bias, int relu, void* y, int64_t ldy, int y_type, ogl_stream_t stream) {
  if (M < 0 || N < 0 || K < 1 || K > 131071 || nrows < 0 || ldx < K || ldw < K || ldx % 64 || ldw % 64 || ldy < N || y_type < OGL_F32 || y_type > OGL_F16)
    return OGL_EINVAL;
  if (!rows && M > nrows) return OGL_EINVAL;
  if (N > INT32_MAX - 256) return OGL_EINVAL;                           // (columns of a whole tile are counted in 31 bits)
  const double most = 4294967296.;                                    // offsets count 64 bytes in 32 bits
  if ((double)nrows * (double)(ldx / 64) >= most || (double)N * (double)(ldw / 64) >= most) return OGL_EINVAL;
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
