// Group norm with an activation, channels last (gfx950): x [B, L, C] (strides for B and L, channels contiguous), G groups of Cg = C / G channels,
// m = L Cg values a group.
//   mean = sum x / m;  var = sum (x - mean)^2 / m;  rstd = 1 / sqrt(var + eps);  h = (x - mean) rstd;  z = h w + b;  y = act(z)
//   dz = dy act'(z);  db = sum dz;  dw = sum dz h;  s1 = sum_group dz w;  s2 = sum_group dz w h;  dx = rstd (dz w - (s1 + h s2) / m)
//
// Bound by memory: a forward pass has to read x and write y, a backward pass to read x and dy and write dx.  Two forms:
//   rows  (L = 1, a matrix of vertices)  a team of lanes holds one group in registers: one pass over memory, the variance from the differences.
//         The backward's teams keep their channels from row to row, so that dw and db stay in registers until the end.
//   maps  (L > 1, or groups too wide for a team)  a thread keeps its 16 bytes of channels and walks the positions.  Samples enough to fill the
//         card: a block a sample (a window of whole groups of it), which reads it twice, the second time from the caches.  Few samples: tiles of
//         positions with partial sums, joined by the next launch.
// Statistics, sums and everything between load and store are float32.  Partial means and squared deviations are joined as such (count, mean, M2),
// the squares taken around each thread's first value, so a mean far from zero costs no digits.  Sums run in an order fixed by the sizes: no atomics.
#include <algorithm>
#include "row_types.h"

#pragma clang fp contract(off)   // products that have to cancel exactly (a group of one value) round where they are written; fma where it is meant

enum { GN_THREADS = 256 };

struct gn_args {
  const void *x, *dy;
  void* y;                       // or dx
  int64_t xb, xl, gb, gl, yb, yl; // strides of x, dy, y in elements
  const void *w, *b;
  int p_type;                    // of w, b: 0 float32, otherwise the type of x
  float *mean, *rstd;            // [B, G]
  float* part;                   // workspace
  float* sums;                   // [B, G, 2] behind it (tiled backward)
  int64_t B;
  int L, C, G, Cg, act, write_dx;
  float eps;
  // maps: windows of gw groups, nvec 16-byte pieces wide; rp positions side by side; tiles of tile_rows positions
  int gw, nw, nvec, rp, tiles, tile_rows, grid_b;
  // rows: lanes of a team; the backward's tg groups x tr rows a block
  int lanes, tg, tr, chunks;
  ogl_div by_g;
};

__device__ __forceinline__ float gn_act(float z, int act) {
  if (act == OGL_ACT_RELU) return z < 0.f ? 0.f : z;
  if (act == OGL_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
  if (act == OGL_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  return z;
}
__device__ __forceinline__ float gn_slope(float z, int act) {
  if (act == OGL_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (act == OGL_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
    return s * __builtin_fmaf(z, 1.f - s, 1.f);
  }
  if (act == OGL_ACT_GELU) return __builtin_fmaf(z * 0.39894228040143268f, __expf(-0.5f * z * z), 0.5f * (1.f + erff(z * 0.70710678118654752f)));
  return 1.f;
}

// n of V elements from p (the others 0) / to p
template <typename T, int V>
__device__ __forceinline__ void gn_load(const T* __restrict__ p, int n, float (&v)[V]) {
  if (n >= V) {
    row_load<T, V>(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = e < n ? (float)p[e] : 0.f;
  }
}
template <typename T, int V>
__device__ __forceinline__ void gn_store(T* __restrict__ p, int n, const float (&v)[V]) {
  if (n >= V) {
    row_store<T, V>(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < n) p[e] = (T)v[e];
  }
}
// channel parameters c .. c + n - 1 (`none` where there are none)
template <typename T, int V>
__device__ __forceinline__ void gn_param(const void* p, int p_type, int c, int n, float none, float (&v)[V]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = none;
  } else if (p_type == OGL_F32) {
    gn_load<float, V>((const float*)p + c, n, v);
  } else {
    gn_load<T, V>((const T*)p + c, n, v);
  }
}

__device__ __forceinline__ float gn_team_sum(float v, int lanes) {
  for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
// over the whole block, the same order for every thread
__device__ __forceinline__ float gn_block_sum(float v, float* lds) {
  v = gn_team_sum(v, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// ================================================================ rows ========================================================================
// One team per (row, group); BLOCK: the team is the block.  NV pieces of V channels a lane.
template <typename T, int V, int NV, bool BLOCK>
__global__ void __launch_bounds__(GN_THREADS) k_gn_rows_fwd(gn_args A) {
  __shared__ float lds[4];
  const int lanes = BLOCK ? GN_THREADS : A.lanes;
  const int lane = threadIdx.x & (lanes - 1);
  const int teams = GN_THREADS / lanes;
  const int64_t first = (int64_t)blockIdx.x * teams;                 // the block's first team, then 32-bit steps from there
  const int64_t b0 = first / A.G;
  const uint32_t k = (uint32_t)(first - b0 * A.G) + threadIdx.x / lanes;
  const uint32_t up = A.by_g.div(k);
  const int64_t b = b0 + up;
  const int g = (int)(k - up * A.G);
  const bool live = b < A.B;                                          // (every lane stays for the shuffles)
  const int c0 = g * A.Cg;
  const T* xp = (const T*)A.x + (live ? b : 0) * A.xb + c0;
  float v[NV][V], s = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e0 = (j * lanes + lane) * V;
    gn_load<T, V>(xp + e0, live ? A.Cg - e0 : 0, v[j]);
#pragma unroll
    for (int e = 0; e < V; ++e) s += v[j][e];
  }
  const float inv = 1.f / (float)A.Cg;
  const float mean = (BLOCK ? gn_block_sum(s, lds) : gn_team_sum(s, lanes)) * inv;
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int n = A.Cg - (j * lanes + lane) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[j][e] -= mean;
      q = e < n ? __builtin_fmaf(v[j][e], v[j][e], q) : q;
    }
  }
  const float var = (BLOCK ? gn_block_sum(q, lds) : gn_team_sum(q, lanes)) * inv;
  const float rstd = 1.f / sqrtf(var + A.eps);
  if (!live) return;
  if (lane == 0 && A.mean) {
    A.mean[b * A.G + g] = mean;
    A.rstd[b * A.G + g] = rstd;
  }
  T* yp = (T*)A.y + b * A.yb + c0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e0 = (j * lanes + lane) * V, n = A.Cg - e0;
    if (n <= 0) continue;
    float w[V], bb[V];
    gn_param<T, V>(A.w, A.p_type, c0 + e0, n, 1.f, w);
    gn_param<T, V>(A.b, A.p_type, c0 + e0, n, 0.f, bb);
#pragma unroll
    for (int e = 0; e < V; ++e) v[j][e] = gn_act(__builtin_fmaf(v[j][e] * rstd, w[e], bb[e]), A.act);
    gn_store<T, V>(yp + e0, n, v[j]);
  }
}

// tg groups side by side x tr rows a block; block x of `chunks` takes every chunks-th set of rows, block y the next groups.  The sums over its rows
// go to part[x][0: dz, 1: dz h][C].
template <typename T, int V, int NV, bool BLOCK>
__global__ void __launch_bounds__(GN_THREADS) k_gn_rows_bwd(gn_args A) {
  __shared__ float lds[2 * GN_THREADS];
  const int lanes = BLOCK ? GN_THREADS : A.lanes;
  const int lane = threadIdx.x & (lanes - 1), team = threadIdx.x / lanes;
  const int gi = team % A.tg, ri = team / A.tg;
  const int g = blockIdx.y * A.tg + gi;
  const bool mine = g < A.G;
  const int c0 = (mine ? g : 0) * A.Cg;
  const float inv = 1.f / (float)A.Cg;
  float w[NV][V], bb[NV][V], sz[NV][V], sh[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e0 = (j * lanes + lane) * V, n = mine ? A.Cg - e0 : 0;
    gn_param<T, V>(A.w, A.p_type, c0 + e0, n, 1.f, w[j]);
    gn_param<T, V>(A.b, A.p_type, c0 + e0, n, 0.f, bb[j]);
#pragma unroll
    for (int e = 0; e < V; ++e) sz[j][e] = sh[j][e] = 0.f;
  }
  // every team runs the same number of rounds: the shuffles (and the block's barriers) see all of it
  const int64_t step = (int64_t)A.chunks * A.tr;
  for (int64_t r0 = (int64_t)blockIdx.x * A.tr; r0 < A.B; r0 += step) {
    const int64_t b = r0 + ri;
    const bool live = mine && b < A.B;
    const int64_t at = live ? b : 0;
    const T* xp = (const T*)A.x + at * A.xb + c0;
    const T* gp = (const T*)A.dy + at * A.gb + c0;
    const float mean = live ? A.mean[at * A.G + g] : 0.f, rstd = live ? A.rstd[at * A.G + g] : 0.f;
    float h[NV][V], dz[NV][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e0 = (j * lanes + lane) * V, n = live ? A.Cg - e0 : 0;
      gn_load<T, V>(xp + e0, n, h[j]);
      gn_load<T, V>(gp + e0, n, dz[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int n = live ? A.Cg - (j * lanes + lane) * V : 0;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (e < n) {
          h[j][e] = (h[j][e] - mean) * rstd;
          dz[j][e] *= gn_slope(__builtin_fmaf(h[j][e], w[j][e], bb[j][e]), A.act);
          sz[j][e] += dz[j][e];
          sh[j][e] = __builtin_fmaf(dz[j][e], h[j][e], sh[j][e]);
          dz[j][e] *= w[j][e];
          s1 += dz[j][e];
          s2 = __builtin_fmaf(dz[j][e], h[j][e], s2);
        }
      }
    }
    if (A.write_dx) {
      s1 = (BLOCK ? gn_block_sum(s1, lds) : gn_team_sum(s1, lanes)) * inv;
      s2 = (BLOCK ? gn_block_sum(s2, lds) : gn_team_sum(s2, lanes)) * inv;
      T* dp = (T*)A.y + at * A.yb + c0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e0 = (j * lanes + lane) * V, n = live ? A.Cg - e0 : 0;
        if (n <= 0) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) dz[j][e] = rstd * (dz[j][e] - __builtin_fmaf(h[j][e], s2, s1));
        gn_store<T, V>(dp + e0, n, dz[j]);
      }
    }
  }
  if (!A.part) return;
  float* out = A.part + (int64_t)blockIdx.x * 2 * A.C + c0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e0 = (j * lanes + lane) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float a = sz[j][e], c = sh[j][e];
      if (A.tr > 1) {                                                  // the rows of the block, in order
        __syncthreads();
        lds[threadIdx.x] = a;
        lds[GN_THREADS + threadIdx.x] = c;
        __syncthreads();
        a = c = 0.f;
        if (ri == 0)
          for (int q = 0; q < A.tr; ++q) {
            a += lds[q * A.tg * lanes + threadIdx.x];
            c += lds[GN_THREADS + q * A.tg * lanes + threadIdx.x];
          }
      }
      if (ri == 0 && mine && e0 + e < A.Cg) {
        out[e0 + e] = a;
        out[A.C + e0 + e] = c;
      }
    }
  }
}

// ================================================================ maps ========================================================================
// A block works on a window of gw whole groups (W channels) of one sample.  NARROW: a thread has one 16-byte piece of channels j and every rp-th
// position from ri on.  WIDE (one group of more than 256 pieces): a thread has every 256th piece, at every position.
struct gn_place {
  int64_t b;
  int win, tile, g0, groups, c0, W, j, ri;
  bool on;
};
__device__ __forceinline__ gn_place gn_where(const gn_args& A, int64_t b, int win, int tile) {
  gn_place P;
  P.b = b;
  P.win = win;
  P.tile = tile;
  P.g0 = win * A.gw;
  P.groups = min(A.gw, A.G - P.g0);
  P.c0 = P.g0 * A.Cg;
  P.W = P.groups * A.Cg;
  P.j = threadIdx.x % A.nvec;
  P.ri = threadIdx.x / A.nvec;
  P.on = P.ri < A.rp;
  return P;
}

struct gn_stats_lds {
  float mean[GN_THREADS * 8], m2[GN_THREADS * 8];                      // [rp][W]; WIDE: of a thread's values
  int count[GN_THREADS];                                               // rows of ri; WIDE: values of the thread
};

// lanes of a wave that work on one of `groups` groups together
__device__ __forceinline__ int gn_group_lanes(int groups) {
  int t = 64;
  while (t > 1 && t * groups > GN_THREADS) t >>= 1;
  return t;
}

// (mean, M2) of each of the block's groups over positions r0 .. r1, handed to `done(group of the window, mean, M2)` by one lane a group
template <typename T, int V, bool WIDE, typename F>
__device__ __forceinline__ void gn_block_stats(const gn_args& A, const gn_place& P, int r0, int r1, gn_stats_lds& S, F done) {
  const T* xp = (const T*)A.x + P.b * A.xb + P.c0;
  if constexpr (!WIDE) {
    float k[V], s[V], q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) k[e] = s[e] = q[e] = 0.f;
    int n = 0;
    const int have = P.on ? P.W - P.j * V : 0;
    if (have > 0) {
      for (int r = r0 + P.ri; r < r1; r += A.rp) {
        float v[V];
        gn_load<T, V>(xp + (int64_t)r * A.xl + P.j * V, have, v);
        if (n == 0) {
#pragma unroll
          for (int e = 0; e < V; ++e) k[e] = v[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = v[e] - k[e];
          s[e] += d;
          q[e] = __builtin_fmaf(d, d, q[e]);
        }
        ++n;
      }
      const float in = n ? 1.f / (float)n : 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < have) {
          const float d = s[e] * in;
          S.mean[P.ri * P.W + P.j * V + e] = k[e] + d;
          S.m2[P.ri * P.W + P.j * V + e] = fmaxf(__builtin_fmaf(-d, s[e], q[e]), 0.f);
        }
    }
    if (P.on && P.j == 0) S.count[P.ri] = n;
  } else {
    float k = 0.f, s = 0.f, q = 0.f;
    int n = 0;
    for (int j = threadIdx.x; j < A.nvec; j += GN_THREADS) {
      const int have = P.W - j * V;
      for (int r = r0; r < r1; ++r) {
        float v[V];
        gn_load<T, V>(xp + (int64_t)r * A.xl + j * V, have, v);
        if (n == 0) k = v[0];
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e < have) {
            const float d = v[e] - k;
            s += d;
            q = __builtin_fmaf(d, d, q);
            ++n;
          }
      }
    }
    const float d = n ? s / (float)n : 0.f;
    S.mean[threadIdx.x] = k + d;
    S.m2[threadIdx.x] = fmaxf(__builtin_fmaf(-d, s, q), 0.f);
    S.count[threadIdx.x] = n;
  }
  __syncthreads();
  const int lanes = WIDE ? 64 : gn_group_lanes(P.groups);
  const int lane = threadIdx.x & (lanes - 1), per = GN_THREADS / lanes;
  for (int q0 = 0; q0 < P.groups; q0 += per) {
    const int g = q0 + threadIdx.x / lanes;
    const bool live = g < P.groups;
    const int entries = live ? (WIDE ? GN_THREADS : A.rp * A.Cg) : 0;
    const float total = (float)A.Cg * (float)(r1 - r0);
    float mean = 0.f, m2 = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      float a = 0.f;
      for (int t = lane; t < entries; t += lanes) {
        const int ri = WIDE ? t : t / A.Cg, at = WIDE ? t : ri * P.W + g * A.Cg + (t - ri * A.Cg);
        const int n = S.count[ri];
        if (n) {
          const float d = S.mean[at] - mean;
          a += pass == 0 ? (float)n * d : __builtin_fmaf((float)n * d, d, S.m2[at]);
        }
      }
      a = gn_team_sum(a, lanes);
      if (pass == 0) mean = a / total;
      else m2 = a;
    }
    if (live && lane == 0) done(g, mean, m2);
  }
  __syncthreads();
}

// y of positions r0 .. r1 from the window's statistics in LDS
template <typename T, int V, bool WIDE>
__device__ __forceinline__ void gn_apply_rows(const gn_args& A, const gn_place& P, int r0, int r1, const float* mean, const float* rstd) {
  const T* xp = (const T*)A.x + P.b * A.xb + P.c0;
  T* yp = (T*)A.y + P.b * A.yb + P.c0;
  for (int j = WIDE ? (int)threadIdx.x : P.j; j < A.nvec; j += WIDE ? GN_THREADS : A.nvec) {
    const int have = WIDE || P.on ? P.W - j * V : 0;
    if (have <= 0) return;
    float mu[V], a[V], bb[V];
    gn_param<T, V>(A.w, A.p_type, P.c0 + j * V, have, 1.f, a);
    gn_param<T, V>(A.b, A.p_type, P.c0 + j * V, have, 0.f, bb);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int g = WIDE ? 0 : min(j * V + e, P.W - 1) / A.Cg;
      mu[e] = mean[g];
      a[e] *= rstd[g];
    }
#pragma unroll 4
    for (int r = r0 + (WIDE ? 0 : P.ri); r < r1; r += WIDE ? 1 : A.rp) {
      float v[V];
      gn_load<T, V>(xp + (int64_t)r * A.xl + j * V, have, v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = gn_act(__builtin_fmaf(v[e] - mu[e], a[e], bb[e]), A.act);
      gn_store<T, V>(yp + (int64_t)r * A.yl + j * V, have, v);
    }
  }
}

// a block a sample window
template <typename T, int V, bool WIDE>
__global__ void __launch_bounds__(GN_THREADS) k_gn_sample_fwd(gn_args A) {
  __shared__ gn_stats_lds S;
  __shared__ float mean[GN_THREADS], rstd[GN_THREADS];
  const int64_t b = blockIdx.x / A.nw;
  const gn_place P = gn_where(A, b, (int)(blockIdx.x - b * A.nw), 0);
  const float inv = 1.f / ((float)A.Cg * (float)A.L);
  gn_block_stats<T, V, WIDE>(A, P, 0, A.L, S, [&](int g, float mu, float m2) {
    const float r = 1.f / sqrtf(m2 * inv + A.eps);
    mean[g] = mu;
    rstd[g] = r;
    if (A.mean) {
      A.mean[b * A.G + P.g0 + g] = mu;
      A.rstd[b * A.G + P.g0 + g] = r;
    }
  });
  gn_apply_rows<T, V, WIDE>(A, P, 0, A.L, mean, rstd);
}

// tiles of positions: part[(b, group), tile] = (mean, M2)
template <typename T, int V, bool WIDE>
__global__ void __launch_bounds__(GN_THREADS) k_gn_stats(gn_args A) {
  __shared__ gn_stats_lds S;
  const int64_t u = blockIdx.x / A.tiles;
  const int tile = (int)(blockIdx.x - u * A.tiles);
  const int64_t b = u / A.nw;
  const gn_place P = gn_where(A, b, (int)(u - b * A.nw), tile);
  const int r0 = tile * A.tile_rows, r1 = min(A.L, r0 + A.tile_rows);
  gn_block_stats<T, V, WIDE>(A, P, r0, r1, S, [&](int g, float mu, float m2) {
    float2* o = (float2*)A.part + (b * A.G + P.g0 + g) * A.tiles + tile;
    *o = make_float2(mu, m2);
  });
}
template <typename T, int V, bool WIDE>
__global__ void __launch_bounds__(GN_THREADS) k_gn_apply(gn_args A) {
  __shared__ float mean[GN_THREADS], rstd[GN_THREADS];
  const int64_t u = blockIdx.x / A.tiles;
  const int tile = (int)(blockIdx.x - u * A.tiles);
  const int64_t b = u / A.nw;
  const gn_place P = gn_where(A, b, (int)(u - b * A.nw), tile);
  const int lanes = gn_group_lanes(P.groups);
  const int lane = threadIdx.x & (lanes - 1), per = GN_THREADS / lanes;
  const float total = (float)A.Cg * (float)A.L;
  for (int q0 = 0; q0 < P.groups; q0 += per) {
    const int g = q0 + threadIdx.x / lanes;
    const bool live = g < P.groups;
    const float2* o = (const float2*)A.part + (b * A.G + P.g0 + (live ? g : 0)) * A.tiles;
    float mu = 0.f, m2 = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      float a = 0.f;
      for (int t = lane; t < A.tiles; t += lanes) {
        const float2 v = o[t];
        const float n = (float)A.Cg * (float)min(A.tile_rows, A.L - t * A.tile_rows), d = v.x - mu;
        a += pass == 0 ? n * d : __builtin_fmaf(n * d, d, v.y);
      }
      a = gn_team_sum(a, lanes);
      if (pass == 0) mu = a / total;
      else m2 = a;
    }
    if (live && lane == 0) {
      const float r = 1.f / sqrtf(m2 / total + A.eps);
      mean[g] = mu;
      rstd[g] = r;
      if (A.mean && tile == 0) {
        A.mean[b * A.G + P.g0 + g] = mu;
        A.rstd[b * A.G + P.g0 + g] = r;
      }
    }
  }
  __syncthreads();
  const int r0 = tile * A.tile_rows;
  gn_apply_rows<T, V, WIDE>(A, P, r0, min(A.L, r0 + A.tile_rows), mean, rstd);
}

// what the backward keeps of a thread's channels
template <int V>
struct gn_cols {
  float mu[V], rs[V], w[V], b[V];
};
template <typename T, int V>
__device__ __forceinline__ void gn_columns(const gn_args& A, int64_t b, int c0, int have, gn_cols<V>& K) {
  gn_param<T, V>(A.w, A.p_type, c0, have, 1.f, K.w);
  gn_param<T, V>(A.b, A.p_type, c0, have, 0.f, K.b);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int64_t g = b * A.G + min(c0 + e, A.C - 1) / A.Cg;
    K.mu[e] = A.mean[g];
    K.rs[e] = A.rstd[g];
  }
}
// sums of dz and dz h over positions r0, r0 + step, .. < r1
template <typename T, int V>
__device__ __forceinline__ void gn_channel_sums(const gn_args& A, const T* xp, const T* gp, int have, int r0, int r1, int step, const gn_cols<V>& K,
                                                float (&sz)[V], float (&sh)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) sz[e] = sh[e] = 0.f;
#pragma unroll 2
  for (int r = r0; r < r1; r += step) {
    float v[V], d[V];
    gn_load<T, V>(xp + (int64_t)r * A.xl, have, v);
    gn_load<T, V>(gp + (int64_t)r * A.gl, have, d);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float h = (v[e] - K.mu[e]) * K.rs[e];
      const float dz = d[e] * gn_slope(__builtin_fmaf(h, K.w[e], K.b[e]), A.act);
      sz[e] += dz;
      sh[e] = __builtin_fmaf(dz, h, sh[e]);
    }
  }
}
// dx of those positions; s1, s2: of each channel's group, divided by m
template <typename T, int V>
__device__ __forceinline__ void gn_dx_rows(const gn_args& A, const T* xp, const T* gp, T* dp, int have, int r0, int r1, int step, const gn_cols<V>& K,
                                           const float (&s1)[V], const float (&s2)[V]) {
#pragma unroll 2
  for (int r = r0; r < r1; r += step) {
    float v[V], d[V];
    gn_load<T, V>(xp + (int64_t)r * A.xl, have, v);
    gn_load<T, V>(gp + (int64_t)r * A.gl, have, d);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float h = (v[e] - K.mu[e]) * K.rs[e];
      const float t = d[e] * gn_slope(__builtin_fmaf(h, K.w[e], K.b[e]), A.act) * K.w[e];
      v[e] = K.rs[e] * (t - __builtin_fmaf(h, s2[e], s1[e]));
    }
    gn_store<T, V>(dp + (int64_t)r * A.yl, have, v);
  }
}

// a block a sample window, block x of grid_b taking every grid_b-th sample: part[x][0: dz, 1: dz h][C] holds the sums over its samples
template <typename T, int V, bool WIDE>
__global__ void __launch_bounds__(GN_THREADS) k_gn_sample_bwd(gn_args A) {
  __shared__ float cz[GN_THREADS * V], ch[GN_THREADS * V];             // [rp][W]; WIDE: s1, s2 of a thread
  __shared__ float g1[GN_THREADS], g2[GN_THREADS];
  const int64_t x = blockIdx.x / A.nw;
  const gn_place P = gn_where(A, x, (int)(blockIdx.x - x * A.nw), 0);
  const float inv = 1.f / ((float)A.Cg * (float)A.L);
  float* out = A.part ? A.part + x * 2 * A.C + P.c0 : nullptr;
  float tz[V], th[V];
#pragma unroll
  for (int e = 0; e < V; ++e) tz[e] = th[e] = 0.f;
  for (int64_t b = x; b < A.B; b += A.grid_b) {
    const T* xp = (const T*)A.x + b * A.xb + P.c0;
    const T* gp = (const T*)A.dy + b * A.gb + P.c0;
    T* dp = (T*)A.y + b * A.yb + P.c0;
    gn_cols<V> K;
    if constexpr (!WIDE) {
      const int have = P.on ? P.W - P.j * V : 0;
      if (have > 0) {
        float sz[V], sh[V];
        gn_columns<T, V>(A, b, P.c0 + P.j * V, have, K);
        gn_channel_sums<T, V>(A, xp + P.j * V, gp + P.j * V, have, P.ri, A.L, A.rp, K, sz, sh);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          tz[e] += sz[e];
          th[e] += sh[e];
          if (e < have) {
            cz[P.ri * P.W + P.j * V + e] = sz[e] * K.w[e];
            ch[P.ri * P.W + P.j * V + e] = sh[e] * K.w[e];
          }
        }
      }
    } else {
      float s1 = 0.f, s2 = 0.f;
      for (int j = threadIdx.x; j < A.nvec; j += GN_THREADS) {
        const int have = P.W - j * V;
        float sz[V], sh[V];
        gn_columns<T, V>(A, b, P.c0 + j * V, have, K);
        gn_channel_sums<T, V>(A, xp + j * V, gp + j * V, have, 0, A.L, 1, K, sz, sh);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e < have) {
            s1 += sz[e] * K.w[e];
            s2 += sh[e] * K.w[e];
            if (out) {                                                  // this thread's own entries
              out[j * V + e] = b == x ? sz[e] : out[j * V + e] + sz[e];
              out[A.C + j * V + e] = b == x ? sh[e] : out[A.C + j * V + e] + sh[e];
            }
          }
      }
      cz[threadIdx.x] = s1;
      ch[threadIdx.x] = s2;
    }
    if (A.write_dx) {                                                   // (the same for the whole grid)
      __syncthreads();
      const int lanes = WIDE ? 64 : gn_group_lanes(P.groups);
      const int lane = threadIdx.x & (lanes - 1), per = GN_THREADS / lanes;
      for (int q0 = 0; q0 < P.groups; q0 += per) {
        const int g = q0 + threadIdx.x / lanes;
        const bool live = g < P.groups;
        const int entries = live ? (WIDE ? GN_THREADS : A.rp * A.Cg) : 0;
        float s1 = 0.f, s2 = 0.f;
        for (int t = lane; t < entries; t += lanes) {
          const int ri = WIDE ? 0 : t / A.Cg, at = WIDE ? t : ri * P.W + g * A.Cg + (t - ri * A.Cg);
          s1 += cz[at];
          s2 += ch[at];
        }
        s1 = gn_team_sum(s1, lanes);
        s2 = gn_team_sum(s2, lanes);
        if (live && lane == 0) {
          g1[g] = s1 * inv;
          g2[g] = s2 * inv;
        }
      }
      __syncthreads();
      float s1[V], s2[V];
      for (int j = WIDE ? (int)threadIdx.x : P.j; j < A.nvec; j += WIDE ? GN_THREADS : A.nvec) {
        const int have = WIDE || P.on ? P.W - j * V : 0;
        if (have <= 0) break;
        if (WIDE) gn_columns<T, V>(A, b, P.c0 + j * V, have, K);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int g = WIDE ? 0 : min(j * V + e, P.W - 1) / A.Cg;
          s1[e] = g1[g];
          s2[e] = g2[g];
        }
        gn_dx_rows<T, V>(A, xp + j * V, gp + j * V, dp + j * V, have, WIDE ? 0 : P.ri, A.L, WIDE ? 1 : A.rp, K, s1, s2);
      }
    }
    __syncthreads();                                                    // cz, ch, g1, g2 are free again
  }
  if (WIDE || !out) return;
  const int have = P.on ? P.W - P.j * V : 0;
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (e < have) {
      cz[P.ri * P.W + P.j * V + e] = tz[e];
      ch[P.ri * P.W + P.j * V + e] = th[e];
    }
  __syncthreads();
  for (int c = threadIdx.x; c < P.W; c += GN_THREADS) {
    float a = 0.f, d = 0.f;
    for (int q = 0; q < A.rp; ++q) {
      a += cz[q * P.W + c];
      d += ch[q * P.W + c];
    }
    out[c] = a;
    out[A.C + c] = d;
  }
}

// tiles of positions: part[b, tile][0: dz, 1: dz h][C]
template <typename T, int V, bool WIDE>
__global__ void __launch_bounds__(GN_THREADS) k_gn_bwd_sums(gn_args A) {
  __shared__ float cz[GN_THREADS * V], ch[GN_THREADS * V];
  const int64_t u = blockIdx.x / A.tiles;
  const int tile = (int)(blockIdx.x - u * A.tiles);
  const int64_t b = u / A.nw;
  const gn_place P = gn_where(A, b, (int)(u - b * A.nw), tile);
  const int r0 = tile * A.tile_rows, r1 = min(A.L, r0 + A.tile_rows);
  const T* xp = (const T*)A.x + b * A.xb + P.c0;
  const T* gp = (const T*)A.dy + b * A.gb + P.c0;
  float* out = A.part + (b * A.tiles + tile) * 2 * A.C + P.c0;
  gn_cols<V> K;
  float sz[V], sh[V];
  if constexpr (WIDE) {
    for (int j = threadIdx.x; j < A.nvec; j += GN_THREADS) {
      const int have = P.W - j * V;
      gn_columns<T, V>(A, b, P.c0 + j * V, have, K);
      gn_channel_sums<T, V>(A, xp + j * V, gp + j * V, have, r0, r1, 1, K, sz, sh);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < have) {
          out[j * V + e] = sz[e];
          out[A.C + j * V + e] = sh[e];
        }
    }
  } else {
    const int have = P.on ? P.W - P.j * V : 0;
    if (have > 0) {
      gn_columns<T, V>(A, b, P.c0 + P.j * V, have, K);
      gn_channel_sums<T, V>(A, xp + P.j * V, gp + P.j * V, have, r0 + P.ri, r1, A.rp, K, sz, sh);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < have) {
          cz[P.ri * P.W + P.j * V + e] = sz[e];
          ch[P.ri * P.W + P.j * V + e] = sh[e];
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < P.W; c += GN_THREADS) {
      float a = 0.f, d = 0.f;
      for (int q = 0; q < A.rp; ++q) {
        a += cz[q * P.W + c];
        d += ch[q * P.W + c];
      }
      out[c] = a;
      out[A.C + c] = d;
    }
  }
}

// Two sums over the partials in one launch.  Blocks below `groups` (B G, or 0): s1, s2 of one (sample, group), over its tiles and channels, divided
// by m.  The others: 16 of the 2 C columns over all `rows` partials -> db, dw.
template <typename T>
__global__ void __launch_bounds__(1024) k_gn_fold(gn_args A, int64_t groups, int64_t rows, void* dw, void* db) {
  __shared__ float lds[2 * 1024];
  const int tid = threadIdx.x;
  if ((int64_t)blockIdx.x < groups) {
    const int64_t b = blockIdx.x / A.G;
    const int g = (int)(blockIdx.x - b * A.G);
    float s1 = 0.f, s2 = 0.f;
    const float* p = A.part + b * A.tiles * 2 * A.C + (int64_t)g * A.Cg;
    for (int i = tid; i < A.tiles * A.Cg; i += 1024) {
      const int t = i / A.Cg, c = i - t * A.Cg;
      float w[1];
      gn_param<T, 1>(A.w, A.p_type, g * A.Cg + c, 1, 1.f, w);
      s1 += p[(int64_t)t * 2 * A.C + c] * w[0];
      s2 += p[(int64_t)t * 2 * A.C + A.C + c] * w[0];
    }
    s1 = gn_team_sum(s1, 64);
    s2 = gn_team_sum(s2, 64);
    if ((tid & 63) == 0) {
      lds[tid >> 6] = s1;
      lds[16 + (tid >> 6)] = s2;
    }
    __syncthreads();
    if (tid < 2) {
      float a = 0.f;
      for (int q = 0; q < 16; ++q) a += lds[tid * 16 + q];
      A.sums[(b * A.G + g) * 2 + tid] = a / ((float)A.Cg * (float)A.L);
    }
    return;
  }
  const int64_t col = ((int64_t)blockIdx.x - groups) * 16 + (tid & 15);
  const int slice = tid >> 4;
  float a = 0.f;
  if (col < 2 * (int64_t)A.C)
    for (int64_t r = slice; r < rows; r += 64) a += A.part[r * 2 * A.C + col];
  lds[tid] = a;
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if (slice < o) lds[tid] += lds[tid + o * 16];
    __syncthreads();
  }
  if (slice == 0 && col < 2 * (int64_t)A.C) {
    void* d = col < A.C ? db : dw;
    const int64_t c = col < A.C ? col : col - A.C;
    if (d) {
      if (A.p_type == OGL_F32) ((float*)d)[c] = lds[tid];
      else ((T*)d)[c] = (T)lds[tid];
    }
  }
}

template <typename T, int V, bool WIDE>
__global__ void __launch_bounds__(GN_THREADS) k_gn_bwd_apply(gn_args A) {
  const int64_t u = blockIdx.x / A.tiles;
  const int tile = (int)(blockIdx.x - u * A.tiles);
  const int64_t b = u / A.nw;
  const gn_place P = gn_where(A, b, (int)(u - b * A.nw), tile);
  const int r0 = tile * A.tile_rows, r1 = min(A.L, r0 + A.tile_rows);
  const T* xp = (const T*)A.x + b * A.xb + P.c0;
  const T* gp = (const T*)A.dy + b * A.gb + P.c0;
  T* dp = (T*)A.y + b * A.yb + P.c0;
  for (int j = WIDE ? (int)threadIdx.x : P.j; j < A.nvec; j += WIDE ? GN_THREADS : A.nvec) {
    const int have = WIDE || P.on ? P.W - j * V : 0;
    if (have <= 0) return;
    gn_cols<V> K;
    gn_columns<T, V>(A, b, P.c0 + j * V, have, K);
    float s1[V], s2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float* s = A.sums + (b * A.G + P.g0 + min(j * V + e, P.W - 1) / A.Cg) * 2;
      s1[e] = s[0];
      s2[e] = s[1];
    }
    gn_dx_rows<T, V>(A, xp + j * V, gp + j * V, dp + j * V, have, r0 + (WIDE ? 0 : P.ri), r1, WIDE ? 1 : A.rp, K, s1, s2);
  }
}

// ================================================================ host ========================================================================
struct gn_plan {
  bool rows, block, wide;
  int nv;                      // rows: pieces a lane
  int64_t part, sums;          // floats of workspace
};

static gn_plan gn_make(gn_args& A, int x_type, bool backward) {
  gn_plan P = {};
  const int V = x_type == OGL_F32 ? 4 : 8;
  const int pieces = (int)ogl_cdiv(A.Cg, V);
  P.rows = A.L == 1 && pieces <= 4 * GN_THREADS;
  if (P.rows) {
    // up to 256 pieces a group: teams inside a wave (1, 2 or 4 pieces a lane); above, the block is the team
    P.block = pieces > 256;
    A.lanes = P.block ? GN_THREADS : 1;
    while (!P.block && A.lanes < 64 && A.lanes < pieces) A.lanes *= 2;
    const int per = (int)ogl_cdiv(pieces, A.lanes);
    P.nv = per <= 1 ? 1 : per <= 2 ? 2 : 4;
    const int teams = GN_THREADS / A.lanes;
    A.tg = 1;
    while (A.tg < teams && A.tg < A.G) A.tg *= 2;
    A.tr = teams / A.tg;
    // about four blocks a CU at most: each leaves 2 C partial sums
    A.chunks = (int)std::min<int64_t>(ogl_cdiv(A.B, A.tr), std::max<int64_t>(1, 1024 / ogl_cdiv(A.G, A.tg)));
    P.part = backward ? (int64_t)A.chunks * 2 * A.C : 0;
    A.by_g = ogl_div::make((uint32_t)A.G);
    return P;
  }
  // Windows of whole groups, at most 256 pieces wide, that keep most threads busy (pieces x positions side by side of 256) and waste least at the
  // last window; of equals the widest.  One group wider than that: WIDE.
  P.wide = pieces > GN_THREADS;
  A.gw = 1;
  if (!P.wide) {
    double best = -1;
    for (int gw = std::min(A.G, 256); gw >= 1; --gw) {
      const int nvec = (int)ogl_cdiv((int64_t)gw * A.Cg, V);
      if (nvec > GN_THREADS) continue;
      if (gw < A.G && (int64_t)gw * A.Cg * (16 / V) < 128) break;      // windows of less than a line
      const double busy = (double)(GN_THREADS / nvec * nvec) / GN_THREADS * ((double)gw * A.Cg / ((double)nvec * V)) *
                          ((double)A.G / (double)(ogl_cdiv(A.G, gw) * gw));
      if (busy > best + 0.02) best = busy, A.gw = gw;
    }
  }
  A.nw = (int)ogl_cdiv(A.G, A.gw);
  A.nvec = (int)ogl_cdiv((int64_t)A.gw * A.Cg, V);
  A.rp = P.wide ? 1 : GN_THREADS / A.nvec;
  // a block a sample window where there are enough of them to fill the card or little to do in each; else tiles of 8 positions a thread or more
  const int64_t blocks = A.B * A.nw;
  int64_t tiles = 1;
  if (blocks < 1024 && A.L > A.rp * 16) tiles = std::min<int64_t>(std::min<int64_t>(ogl_cdiv(A.L, A.rp * 8), ogl_cdiv(2048, blocks)), 256);
  A.tile_rows = (int)ogl_cdiv(A.L, tiles);
  A.tiles = (int)ogl_cdiv(A.L, A.tile_rows);
  A.grid_b = (int)std::min<int64_t>(A.B, std::max<int64_t>(1, 2048 / A.nw));
  if (backward) {
    P.part = (A.tiles == 1 ? (int64_t)A.grid_b : A.B * A.tiles) * 2 * A.C;
    P.sums = A.tiles == 1 ? 0 : A.B * A.G * 2;
  } else {
    P.part = A.tiles == 1 ? 0 : A.B * A.G * A.tiles * 2;
  }
  return P;
}

static bool gn_sizes_ok(int64_t B, int64_t L, int C, int G, int x_type) {
  return B >= 0 && L >= 0 && L <= (1 << 30) && C >= 1 && G >= 1 && C % G == 0 && C <= (1 << 22) && x_type >= OGL_F32 && x_type <= OGL_F16 &&
         (B == 0 || L == 0 || B <= (int64_t)1 << 40);
}

extern "C" int64_t ogl_group_norm_workspace_bytes(int64_t B, int64_t L, int C, int G, int x_type, int backward) {
  if (!gn_sizes_ok(B, L, C, G, x_type)) return OGL_EINVAL;
  if (B == 0 || L == 0) return 0;
  gn_args A = {};
  A.B = B; A.L = (int)L; A.C = C; A.G = G; A.Cg = C / G;
  const gn_plan P = gn_make(A, x_type, backward != 0);
  return 4 * (P.part + P.sums);
}

#define GN_LAUNCH(K, GRID, ...)                                                                   \
  do {                                                                                            \
    const int64_t grid_ = (GRID);                                                                 \
    if (grid_ * GN_THREADS > (int64_t)UINT32_MAX) return OGL_EINVAL;                               \
    hipLaunchKernelGGL(HIP_KERNEL_NAME(K), dim3((unsigned)grid_), dim3(GN_THREADS), 0, st, A);    \
  } while (0)

template <typename T, int V>
static int gn_forward(const gn_args& A, const gn_plan& P, hipStream_t st) {
  if (P.rows) {
    const int64_t grid = ogl_cdiv(A.B * A.G, GN_THREADS / A.lanes);
    if (P.block) {
      if (P.nv == 1) GN_LAUNCH((k_gn_rows_fwd<T, V, 1, true>), grid);
      else if (P.nv == 2) GN_LAUNCH((k_gn_rows_fwd<T, V, 2, true>), grid);
      else GN_LAUNCH((k_gn_rows_fwd<T, V, 4, true>), grid);
    } else {
      if (P.nv == 1) GN_LAUNCH((k_gn_rows_fwd<T, V, 1, false>), grid);
      else if (P.nv == 2) GN_LAUNCH((k_gn_rows_fwd<T, V, 2, false>), grid);
      else GN_LAUNCH((k_gn_rows_fwd<T, V, 4, false>), grid);
    }
    return OGL_OK;
  }
  if (A.tiles == 1) {
    if (P.wide) GN_LAUNCH((k_gn_sample_fwd<T, V, true>), A.B * A.nw);
    else GN_LAUNCH((k_gn_sample_fwd<T, V, false>), A.B * A.nw);
    return OGL_OK;
  }
  const int64_t grid = A.B * A.nw * A.tiles;
  if (P.wide) {
    GN_LAUNCH((k_gn_stats<T, V, true>), grid);
    GN_LAUNCH((k_gn_apply<T, V, true>), grid);
  } else {
    GN_LAUNCH((k_gn_stats<T, V, false>), grid);
    GN_LAUNCH((k_gn_apply<T, V, false>), grid);
  }
  return OGL_OK;
}

template <typename T, int V>
static int gn_backward(const gn_args& A, const gn_plan& P, void* dw, void* db, hipStream_t st) {
  int64_t rows = 0, groups = 0;
  if (P.rows) {
    const dim3 grid((unsigned)A.chunks, (unsigned)ogl_cdiv(A.G, A.tg));
    if (grid.y > 65535) return OGL_EINVAL;
#define GN_ROWS(NV, BLOCK) hipLaunchKernelGGL((k_gn_rows_bwd<T, V, NV, BLOCK>), grid, dim3(GN_THREADS), 0, st, A)
    if (P.block) {
      if (P.nv == 1) GN_ROWS(1, true);
      else if (P.nv == 2) GN_ROWS(2, true);
      else GN_ROWS(4, true);
    } else {
      if (P.nv == 1) GN_ROWS(1, false);
      else if (P.nv == 2) GN_ROWS(2, false);
      else GN_ROWS(4, false);
    }
#undef GN_ROWS
    rows = A.chunks;
  } else if (A.tiles == 1) {
    if (P.wide) GN_LAUNCH((k_gn_sample_bwd<T, V, true>), (int64_t)A.grid_b * A.nw);
    else GN_LAUNCH((k_gn_sample_bwd<T, V, false>), (int64_t)A.grid_b * A.nw);
    rows = A.grid_b;
  } else {
    if (P.wide) GN_LAUNCH((k_gn_bwd_sums<T, V, true>), A.B * A.nw * A.tiles);
    else GN_LAUNCH((k_gn_bwd_sums<T, V, false>), A.B * A.nw * A.tiles);
    rows = A.B * A.tiles;
    groups = A.write_dx ? A.B * A.G : 0;
  }
  const int64_t folds = dw || db ? ogl_cdiv(2 * (int64_t)A.C, 16) : 0;
  if ((groups + folds) * 1024 > (int64_t)UINT32_MAX) return OGL_EINVAL;
  if (groups + folds > 0)
    hipLaunchKernelGGL(k_gn_fold<T>, dim3((unsigned)(groups + folds)), dim3(1024), 0, st, A, groups, rows, dw, db);
  if (groups > 0) {
    if (P.wide) GN_LAUNCH((k_gn_bwd_apply<T, V, true>), A.B * A.nw * A.tiles);
    else GN_LAUNCH((k_gn_bwd_apply<T, V, false>), A.B * A.nw * A.tiles);
  }
  return OGL_OK;
}

static bool gn_aligned(const void* p, int type) { return p == nullptr || ((uintptr_t)p & (type == OGL_F32 ? 3 : 1)) == 0; }

extern "C" int ogl_group_norm_fwd(const void* x, int64_t xb, int64_t xl, int x_type, int64_t B, int64_t L, int C, int G, const void* w, const void* b,
                                  int p_type, float eps, int act, void* y, int64_t yb, int64_t yl, float* mean, float* rstd, void* workspace,
                                  int64_t workspace_bytes, ogl_stream_t stream) {
  if (!gn_sizes_ok(B, L, C, G, x_type) || (p_type != OGL_F32 && p_type != x_type) || act < OGL_ACT_NONE || act > OGL_ACT_GELU || !(eps >= 0.f))
    return OGL_EINVAL;
  if (B == 0 || L == 0) return OGL_OK;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr) || (L > 1 && (xl < C || yl < C)) || (B > 1 && (xb < C || yb < C))) return OGL_EINVAL;
  if (!gn_aligned(x, x_type) || !gn_aligned(y, x_type) || !gn_aligned(w, p_type) || !gn_aligned(b, p_type)) return OGL_EINVAL;
  gn_args A = {};
  A.x = x; A.y = y; A.xb = xb; A.xl = xl; A.yb = yb; A.yl = yl; A.w = w; A.b = b; A.p_type = p_type; A.mean = mean; A.rstd = rstd;
  A.B = B; A.L = (int)L; A.C = C; A.G = G; A.Cg = C / G; A.eps = eps; A.act = act;
  const gn_plan P = gn_make(A, x_type, false);
  if (P.part > 0 && (!workspace || workspace_bytes < 4 * P.part || ((uintptr_t)workspace & 7))) return OGL_EWORKSPACE;
  A.part = (float*)workspace;
  hipStream_t st = (hipStream_t)stream;
  const int rc = x_type == OGL_F32 ? gn_forward<float, 4>(A, P, st) : x_type == OGL_BF16 ? gn_forward<ogl_bf16, 8>(A, P, st) : gn_forward<ogl_f16, 8>(A, P, st);
  if (rc != OGL_OK) return rc;
  OGL_CHECK_LAUNCH();
  return OGL_OK;
}

extern "C" int ogl_group_norm_bwd(const void* dy, int64_t gb, int64_t gl, const void* x, int64_t xb, int64_t xl, int x_type, int64_t B, int64_t L, int C,
                                  int G, const void* w, const void* b, int p_type, int act, const float* mean, const float* rstd, void* dx, int64_t db_,
                                  int64_t dl, void* dw, void* db, void* workspace, int64_t workspace_bytes, ogl_stream_t stream) {
  if (!gn_sizes_ok(B, L, C, G, x_type) || (p_type != OGL_F32 && p_type != x_type) || act < OGL_ACT_NONE || act > OGL_ACT_GELU) return OGL_EINVAL;
  if (B == 0 || L == 0) return OGL_EINVAL;                              // (no sums to write: the caller's gradients are zeros)
  if (!dy || !x || !mean || !rstd || (L > 1 && (xl < C || gl < C || (dx && dl < C))) || (B > 1 && (xb < C || gb < C || (dx && db_ < C)))) return OGL_EINVAL;
  if (!gn_aligned(x, x_type) || !gn_aligned(dy, x_type) || !gn_aligned(dx, x_type) || !gn_aligned(w, p_type) || !gn_aligned(b, p_type) ||
      !gn_aligned(dw, p_type) || !gn_aligned(db, p_type))
    return OGL_EINVAL;
  if (!dx && !dw && !db) return OGL_OK;
  gn_args A = {};
  A.x = x; A.dy = dy; A.y = dx; A.xb = xb; A.xl = xl; A.gb = gb; A.gl = gl; A.yb = db_; A.yl = dl; A.w = w; A.b = b; A.p_type = p_type;
  A.mean = (float*)mean; A.rstd = (float*)rstd; A.write_dx = dx != nullptr;
  A.B = B; A.L = (int)L; A.C = C; A.G = G; A.Cg = C / G; A.act = act;
  const gn_plan P = gn_make(A, x_type, true);
  if (!workspace || workspace_bytes < 4 * (P.part + P.sums) || ((uintptr_t)workspace & 7)) return OGL_EWORKSPACE;
  A.part = (float*)workspace;
  A.sums = A.part + P.part;
  hipStream_t st = (hipStream_t)stream;
  const int rc = x_type == OGL_F32    ? gn_backward<float, 4>(A, P, dw, db, st)
                 : x_type == OGL_BF16 ? gn_backward<ogl_bf16, 8>(A, P, dw, db, st)
                                      : gn_backward<ogl_f16, 8>(A, P, dw, db, st);
  if (rc != OGL_OK) return rc;
  OGL_CHECK_LAUNCH();
  return OGL_OK;
}
