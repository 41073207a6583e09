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
#pragma once
#include "group_norm.h"

#pragma clang fp contract(off)   // products that have to cancel exactly (a group of one value) round where they are written; fma where it is meant

// A lane's team in the rows kernels: `lanes` neighbours (any number up to 64, so that few lanes of a wave are left over), tw of them a wave.
struct gn_team {
  int team, pos;
  bool on;
  __device__ __forceinline__ gn_team(const gn_args& A, int lane) {
    team = (int)A.by_lanes.div((uint32_t)lane);
    pos = lane - team * A.lanes;
    on = team < A.tw;
  }
};
// over a team, the same bits in every lane; every lane of the wave takes part
__device__ __forceinline__ float gn_span_sum(float v, const gn_args& A, const gn_team& t) {
  if ((A.lanes & (A.lanes - 1)) == 0) return row_team_sum(v, A.lanes);
  const int at = (threadIdx.x & 63) * 4;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1)
    if (o < A.lanes) {
      const float u = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(at + o * 4, __builtin_bit_cast(int, v)));
      v += t.pos + o < A.lanes ? u : 0.f;
    }
  return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(at - t.pos * 4, __builtin_bit_cast(int, v)));
}

// The normal distribution function at z, and e^(-z^2 / 2): Phi(-|z|) = erfc(x) / 2 at x = |z| / sqrt 2 by the polynomial of Abramowitz and Stegun
// 7.1.26 in 1 / (1 + 0.3275911 x), off by at most 7.5e-8; the exponential is the one that the density needs too.  The library's erff takes both of
// its branches in most waves: the gelu cases were bound by it.  The error is absolute: with the roundings z Phi(z) is off by up to 2.8e-7 |z|, 5e-7 of the
// value at z near 0, 3e-6 at -2, 5e-4 at -4, 4e-3 at -6.  0.5 z (1 + erff(z / sqrt 2)) cancels there and is off by 5e-4 at -4, all of the value at -6.
__device__ __forceinline__ float gn_phi(float z, float& e) {
  e = __expf(-0.5f * z * z);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(__builtin_fabsf(z), 0.3275911f * 0.70710678f, 1.f));
  float p = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
  p = __builtin_fmaf(t, p, 1.421413741f);
  p = __builtin_fmaf(t, p, -0.284496736f);
  p = __builtin_fmaf(t, p, 0.254829592f);
  const float q = 0.5f * t * p * e;
  return z < 0.f ? q : 1.f - q;
}
template <int ACT>
__device__ __forceinline__ float gn_act(float z) {
  float e;
  if constexpr (ACT == OGL_ACT_RELU) return z < 0.f ? 0.f : z;
  else if constexpr (ACT == OGL_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
  else if constexpr (ACT == OGL_ACT_GELU) return z * gn_phi(z, e);
  else return z;
}
template <int ACT>
__device__ __forceinline__ float gn_slope(float z) {
  if constexpr (ACT == OGL_ACT_RELU) {
    return z > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == OGL_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
    return s * __builtin_fmaf(z, 1.f - s, 1.f);
  } else if constexpr (ACT == OGL_ACT_GELU) {
    float e;
    const float phi = gn_phi(z, e);
    return __builtin_fmaf(z * 0.39894228040143268f, e, phi);
  } else {
    return 1.f;
  }
}
// f with the activation as a constant: one branch around a loop over many values instead of one at each of them
template <typename F>
__device__ __forceinline__ void gn_by_act(int act, F f) {
  if (act == OGL_ACT_SILU) f(std::integral_constant<int, OGL_ACT_SILU>());
  else if (act == OGL_ACT_GELU) f(std::integral_constant<int, OGL_ACT_GELU>());
  else if (act == OGL_ACT_RELU) f(std::integral_constant<int, OGL_ACT_RELU>());
  else f(std::integral_constant<int, OGL_ACT_NONE>());
}

// channel parameters c .. of a piece (`none` where there are none)
template <typename T, int V, typename PIECE>
__device__ __forceinline__ void gn_param(const void* p, int p_type, int c, const PIECE& P, float none, float (&v)[V]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = none;
  } else if (p_type == OGL_F32) {
    if constexpr (V == 4) {
      row_piece<float, 4>(P.n, P.tiny).load((const float*)p + c, v);
    } else {                                                            // eight channels of 32 bits: two pieces
      const row_piece<float, 4> lo(P.n, P.tiny || P.n < 4), hi(P.n - 4, P.tiny);
      float a[4], b[4];
      lo.load((const float*)p + c, a);
      hi.load((const float*)p + c + 4, b);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        v[4 + e] = b[e];
      }
    }
  } else {
    P.load((const T*)p + c, v);
  }
}

// a squared deviation that rounding took below zero; a NaN stays one
__device__ __forceinline__ float gn_not_negative(float v) { return v < 0.f ? 0.f : v; }
// over the whole block, the same order for every thread
__device__ __forceinline__ float gn_block_sum(float v, float* lds) {
  v = row_team_sum(v, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// ================================================================ rows ========================================================================
// One team per group and R rows one below the other; BLOCK: the team is the block.  NV pieces of V channels a lane and row.  R: a team's loads are
// issued together; one piece a lane in flight leaves the memory waiting.
template <typename T, int V, int NV, int R, bool BLOCK, typename PIECE>
__global__ void __launch_bounds__(GN_THREADS) k_gn_rows_fwd(gn_args A) {
  __shared__ float lds[4];
  const gn_team t(A, threadIdx.x & 63);
  const int lanes = BLOCK ? GN_THREADS : A.lanes, lane = BLOCK ? (int)threadIdx.x : t.pos;
  const int64_t first = (int64_t)blockIdx.x * (BLOCK ? 1 : 4 * A.tw);  // the block's first team, then 32-bit steps from there
  const int64_t b0 = first / A.G;
  const uint32_t k = (uint32_t)(first - b0 * A.G) + (BLOCK ? 0u : (threadIdx.x >> 6) * A.tw + t.team);
  const uint32_t up = A.by_g.div(k);
  const int64_t b = (b0 + up) * R;
  const int g = (int)(k - up * A.G);
  const int rows = BLOCK || t.on ? (int)min((int64_t)R, max((int64_t)0, A.B - b)) : 0;   // (every lane stays for the shuffles)
  const int c0 = g * A.Cg;
  const T* xp = (const T*)A.x + (rows ? b : 0) * A.xb + c0;
  const bool tiny = A.Cg < V;
  typename PIECE::raw raw[R][NV];
  float v[R][NV][V], mean[R], rstd[R];
#pragma unroll
  for (int q = 0; q < R; ++q)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e0 = (j * lanes + lane) * V;
      raw[q][j] = PIECE(q < rows ? A.Cg - e0 : 0, tiny).fetch(xp + q * A.xb + e0);
    }
#pragma unroll
  for (int q = 0; q < R; ++q)
#pragma unroll
    for (int j = 0; j < NV; ++j) PIECE(q < rows ? A.Cg - (j * lanes + lane) * V : 0, tiny).expand(raw[q][j], v[q][j]);
  const float inv = 1.f / (float)A.Cg;
#pragma unroll
  for (int q = 0; q < R; ++q) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) s += v[q][j][e];
    mean[q] = (BLOCK ? gn_block_sum(s, lds) : gn_span_sum(s, A, t)) * inv;
  }
#pragma unroll
  for (int q = 0; q < R; ++q) {
    float d = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int n = A.Cg - (j * lanes + lane) * V;
      if (n >= V) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          v[q][j][e] -= mean[q];
          d = __builtin_fmaf(v[q][j][e], v[q][j][e], d);
        }
      } else if (PIECE::cuts && n > 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          v[q][j][e] -= mean[q];
          d = e < n ? __builtin_fmaf(v[q][j][e], v[q][j][e], d) : d;
        }
      }
    }
    rstd[q] = 1.f / sqrtf((BLOCK ? gn_block_sum(d, lds) : gn_span_sum(d, A, t)) * inv + A.eps);
  }
  if (lane == 0 && A.mean) {
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (q < rows) {
        A.mean[(b + q) * A.G + g] = mean[q];
        A.rstd[(b + q) * A.G + g] = rstd[q];
      }
  }
  T* yp = (T*)A.y + b * A.yb + c0;
  gn_by_act(A.act, [&](auto act) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e0 = (j * lanes + lane) * V;
      const PIECE P(rows ? A.Cg - e0 : 0, tiny);
      if (P.n <= 0) continue;
      float w[V], bb[V];                                               // (loaded ahead of the reductions they cost registers and time: 64 -> 70 us)
      gn_param<T, V, PIECE>(A.w, A.p_type, c0 + e0, P, 1.f, w);
      gn_param<T, V, PIECE>(A.b, A.p_type, c0 + e0, P, 0.f, bb);
#pragma unroll
      for (int q = 0; q < R; ++q) {
        if (q >= rows) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) v[q][j][e] = gn_act<decltype(act)::value>(__builtin_fmaf(v[q][j][e] * rstd[q], w[e], bb[e]));
        P.store(yp + q * A.yb + e0, v[q][j], A.past);
      }
    }
  });
}

// A wave has tg groups side by side and rpw rows, a block its four waves' rows; block x of `chunks` takes every chunks-th set of rows, blocks (y, z) the
// next groups.  The sums over its rows go to part[x][0: dz, 1: dz h][C].
template <typename T, int V, int NV, int R, bool BLOCK, typename PIECE>
__global__ void __launch_bounds__(GN_THREADS) k_gn_rows_bwd(gn_args A) {
  __shared__ float lds[2 * GN_THREADS];
  const gn_team t(A, threadIdx.x & 63);
  const int lanes = BLOCK ? GN_THREADS : A.lanes, lane = BLOCK ? (int)threadIdx.x : t.pos;
  const int rw = BLOCK ? 0 : (int)A.by_tg.div((uint32_t)t.team), gi = BLOCK ? 0 : t.team - rw * A.tg;
  const int ri = BLOCK ? 0 : (int)(threadIdx.x >> 6) * A.rpw + rw, block_rows = BLOCK ? 1 : 4 * A.rpw;
  const int g = (blockIdx.z * gridDim.y + blockIdx.y) * A.tg + gi;
  const bool mine = g < A.G && (BLOCK || (t.on && rw < A.rpw));
  const int c0 = (mine ? g : 0) * A.Cg;
  const float inv = 1.f / (float)A.Cg;
  const bool tiny = A.Cg < V;
  float w[NV][V], bb[NV][V], sz[NV][V], sh[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e0 = (j * lanes + lane) * V;
    const PIECE P(mine ? A.Cg - e0 : 0, tiny);
    gn_param<T, V, PIECE>(A.w, A.p_type, c0 + e0, P, 1.f, w[j]);
    gn_param<T, V, PIECE>(A.b, A.p_type, c0 + e0, P, 0.f, bb[j]);
#pragma unroll
    for (int e = 0; e < V; ++e) sz[j][e] = sh[j][e] = 0.f;
  }
  // every team runs the same number of rounds: the shuffles (and the block's barriers) see all of it
  const int64_t step = (int64_t)A.chunks * block_rows * R;
  for (int64_t r0 = (int64_t)blockIdx.x * block_rows * R; r0 < A.B; r0 += step) {
    const int64_t b = r0 + ri * R;
    const int rows = mine ? (int)min((int64_t)R, max((int64_t)0, A.B - b)) : 0;
    const int64_t at = rows ? b : 0;
    const T* xp = (const T*)A.x + at * A.xb + c0;
    const T* gp = (const T*)A.dy + at * A.gb + c0;
    typename PIECE::raw rx[R][NV], rg[R][NV];
    float h[R][NV][V], dz[R][NV][V], mean[R], rstd[R], s1[R], s2[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mean[q] = q < rows ? A.mean[(at + q) * A.G + g] : 0.f;
      rstd[q] = q < rows ? A.rstd[(at + q) * A.G + g] : 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e0 = (j * lanes + lane) * V;
        const PIECE P(q < rows ? A.Cg - e0 : 0, tiny);
        rx[q][j] = P.fetch(xp + q * A.xb + e0);
        rg[q][j] = P.fetch(gp + q * A.gb + e0);
      }
    }
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const PIECE P(q < rows ? A.Cg - (j * lanes + lane) * V : 0, tiny);
        P.expand(rx[q][j], h[q][j]);
        P.expand(rg[q][j], dz[q][j]);
      }
    gn_by_act(A.act, [&](auto act) {
#pragma unroll
      for (int q = 0; q < R; ++q) {
        s1[q] = s2[q] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)                                  // (behind a run's end dy is 0, and so is every term)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            h[q][j][e] = (h[q][j][e] - mean[q]) * rstd[q];
            dz[q][j][e] *= gn_slope<decltype(act)::value>(__builtin_fmaf(h[q][j][e], w[j][e], bb[j][e]));
            sz[j][e] += dz[q][j][e];
            sh[j][e] = __builtin_fmaf(dz[q][j][e], h[q][j][e], sh[j][e]);
            dz[q][j][e] *= w[j][e];
            s1[q] += dz[q][j][e];
            s2[q] = __builtin_fmaf(dz[q][j][e], h[q][j][e], s2[q]);
          }
      }
    });
    if (A.write_dx) {
#pragma unroll
      for (int q = 0; q < R; ++q) {
        if (A.Cg == 1) rstd[q] = 0.f;                                   // a group of one value: dx is 0, not the rounding of what cancels
        s1[q] = -(BLOCK ? gn_block_sum(s1[q], lds) : gn_span_sum(s1[q], A, t)) * inv * rstd[q];
        s2[q] = -(BLOCK ? gn_block_sum(s2[q], lds) : gn_span_sum(s2[q], A, t)) * inv * rstd[q];
      }
      T* dp = (T*)A.y + at * A.yb + c0;
#pragma unroll
      for (int q = 0; q < R; ++q)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int e0 = (j * lanes + lane) * V;
          const PIECE P(q < rows ? A.Cg - e0 : 0, tiny);
          if (P.n <= 0) continue;
#pragma unroll
          for (int e = 0; e < V; ++e) dz[q][j][e] = __builtin_fmaf(dz[q][j][e], rstd[q], __builtin_fmaf(h[q][j][e], s2[q], s1[q]));
          P.store(dp + q * A.yb + e0, dz[q][j], A.past);
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
      if (!BLOCK) {                                                    // the rows of the block, in order
        __syncthreads();
        lds[threadIdx.x] = a;
        lds[GN_THREADS + threadIdx.x] = c;
        __syncthreads();
        a = c = 0.f;
        if (ri == 0 && mine)
          for (int wave = 0; wave < 4; ++wave)
            for (int q = 0; q < A.rpw; ++q) {
              const int at = wave * 64 + q * A.tg * lanes + threadIdx.x;
              a += lds[at];
              c += lds[GN_THREADS + at];
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
template <int NT>
__device__ __forceinline__ gn_place gn_where(const gn_args& A, int64_t b, int win, int tile) {
  gn_place P;
  P.b = b;
  P.win = win;
  P.tile = tile;
  P.g0 = win * A.gw;
  P.groups = min(A.gw, A.G - P.g0);
  P.c0 = P.g0 * A.Cg;
  P.W = P.groups * A.Cg;
  P.ri = (int)A.by_nvec.div(threadIdx.x);
  P.j = threadIdx.x - P.ri * A.nvec;
  P.on = P.ri < A.rp;
  return P;
}

template <int NT>
struct __align__(16) gn_stats_lds {
  float a[NT * 8], q[NT * 8];                          // [rp][nvec V] sums around a pivot, then (mean, M2) of a channel; WIDE: of a thread
  int count[NT];                                               // WIDE: values of the thread
};
template <int V>
__device__ __forceinline__ void gn_lds_put(float* p, const float (&v)[V]) {
#pragma unroll
  for (int e = 0; e < V; e += 4) *(float4*)(p + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
}

// lanes of a wave that work on one of `groups` groups (or channels) together
template <int NT>
__device__ __forceinline__ int gn_group_lanes(int groups) {
  int t = 64;
  while (t > 1 && t * groups > NT) t >>= 1;
  return t;
}

// (mean, M2) of each of the block's groups over positions r0 .. r1, handed to `done(group of the window, mean, M2)` by one lane a group.
// NARROW: a thread's sums and squares around its first value, from them its (mean, M2); those of a channel's threads joined around the first one's mean,
// then those of a group's channels likewise.
template <typename T, int V, bool WIDE, typename PIECE, int NT, typename F>
__device__ __forceinline__ void gn_block_stats(const gn_args& A, const gn_place& P, int r0, int r1, gn_stats_lds<NT>& S, F done) {
  const T* xp = (const T*)A.x + P.b * A.xb + P.c0 + (int64_t)r0 * A.xl;
  const int rows = r1 - r0;
  const float in = 1.f / (float)rows;
  if constexpr (!WIDE) {
    const int have = P.on ? P.W - P.j * V : 0;
    if (have > 0) {
      float k[V], s[V], q[V];
      const PIECE C(have, P.W < V);
      const int64_t step = (int64_t)A.rp * A.xl;
      const T* p = xp + P.j * V + P.ri * A.xl;
      int r = P.ri;
      auto take = [&](auto count, auto first) {                        // that many loads in flight
        constexpr int U = decltype(count)::value;
        typename PIECE::raw raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = C.fetch(p + u * step);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float v[V];
          C.expand(raw[u], v);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (decltype(first)::value && u == 0) {
              k[e] = v[e];
              s[e] = q[e] = 0.f;
            } else {
              const float d = v[e] - k[e];
              s[e] += d;
              q[e] = __builtin_fmaf(d, d, q[e]);
            }
          }
        }
        r += U * A.rp;
        p += U * step;
      };
      const std::integral_constant<int, 1> one;
      const std::integral_constant<int, 8> eight;
      if (r < rows) {
        if (r + 7 * A.rp < rows) take(eight, std::true_type());
        else take(one, std::true_type());
        while (r + 7 * A.rp < rows) take(eight, std::false_type());
        if (r + 3 * A.rp < rows) take(std::integral_constant<int, 4>(), std::false_type());
        while (r < rows) take(one, std::false_type());
        const float n = (float)((r - P.ri) / A.rp), by = 1.f / n;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = s[e] * by;
          k[e] += d;
          q[e] = gn_not_negative(__builtin_fmaf(-d, s[e], q[e]));
        }
        gn_lds_put<V>(S.a + (P.ri * A.nvec + P.j) * V, k);
        gn_lds_put<V>(S.q + (P.ri * A.nvec + P.j) * V, q);
      }
    }
    __syncthreads();
    const int lanes = gn_group_lanes<NT>(P.W), lane = threadIdx.x & (lanes - 1);
    const int most = min(A.rp, rows), whole = rows / A.rp, rest = rows - whole * A.rp;
    for (int c0 = 0; c0 < P.W; c0 += NT / lanes) {
      const int c = c0 + threadIdx.x / lanes;                          // (its entry of position 0 is this team's from here on)
      const bool live = c < P.W;
      const float first = live ? S.a[c] : 0.f;
      float s = 0.f, q = 0.f;
      if (live)
        for (int ri = lane; ri < most; ri += lanes) {
          const float n = (float)(whole + (ri < rest)), d = S.a[ri * A.nvec * V + c] - first;
          s = __builtin_fmaf(n, d, s);
          q += __builtin_fmaf(n * d, d, S.q[ri * A.nvec * V + c]);
        }
      s = row_team_sum(s, lanes);
      q = row_team_sum(q, lanes);
      const float d = s * in;
      if (live && lane == 0) {
        S.a[c] = first + d;
        S.q[c] = gn_not_negative(__builtin_fmaf(-d, s, q));
      }
    }
  } else {
    float k = 0.f, s = 0.f, q = 0.f;
    int n = 0;
    for (int j = threadIdx.x; j < A.nvec; j += NT) {
      const int have = P.W - j * V;
      for (int r = 0; r < rows; ++r) {
        float v[V];
        PIECE(have, false).load(xp + (int64_t)r * A.xl + j * V, v);
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
    S.a[threadIdx.x] = k + d;
    S.q[threadIdx.x] = gn_not_negative(__builtin_fmaf(-d, s, q));
    S.count[threadIdx.x] = n;
  }
  __syncthreads();
  const int lanes = WIDE ? 64 : gn_group_lanes<NT>(P.groups);
  const int lane = threadIdx.x & (lanes - 1), per = NT / lanes;
  for (int q0 = 0; q0 < P.groups; q0 += per) {
    const int g = q0 + threadIdx.x / lanes;
    const bool live = g < P.groups;
    const int at = WIDE ? 0 : g * A.Cg;
    const float total = (float)A.Cg * (float)rows, first = live ? S.a[at] : 0.f;
    float a = 0.f, m2 = 0.f;
    if (live)
      for (int c = lane; c < (WIDE ? NT : A.Cg); c += lanes) {
        const float n = WIDE ? (float)S.count[c] : (float)rows, d = S.a[at + c] - first;
        if (n > 0.f) {
          a = __builtin_fmaf(n, d, a);
          m2 += __builtin_fmaf(n * d, d, S.q[at + c]);
        }
      }
    a = row_team_sum(a, lanes);
    m2 = row_team_sum(m2, lanes);
    const float mean = first + a / total;
    m2 = gn_not_negative(__builtin_fmaf(-a / total, a, m2));
    if (live && lane == 0) done(g, mean, m2);
  }
  __syncthreads();
}

// y of positions r0 .. r1 from the window's statistics, which `stats` (called once by every thread) puts into LDS while the first loads are on their way
template <typename T, int V, bool WIDE, typename PIECE, int NT, typename F>
__device__ __forceinline__ void gn_apply_rows(const gn_args& A, const gn_place& P, int r0, int r1, const float* mean, const float* rstd, F stats) {
  constexpr int U = 2;
  typedef typename PIECE::raw raw_t;
  const int step = WIDE ? 1 : A.rp, first = r0 + (WIDE ? 0 : P.ri);
  raw_t ahead[U];
  if constexpr (!WIDE) {
    const int have = P.on ? P.W - P.j * V : 0;
    const PIECE C(have, P.W < V);
    const T* xp = (const T*)A.x + P.b * A.xb + P.c0 + P.j * V;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (have > 0 && first + u * step < r1) ahead[u] = C.fetch(xp + (int64_t)(first + u * step) * A.xl);
  }
  stats();
  for (int j = WIDE ? (int)threadIdx.x : P.j; j < A.nvec; j += WIDE ? NT : A.nvec) {
    const int have = WIDE || P.on ? P.W - j * V : 0;
    if (have <= 0) return;
    const PIECE C(have, P.W < V);
    const T* xp = (const T*)A.x + P.b * A.xb + P.c0 + j * V;
    T* yp = (T*)A.y + P.b * A.yb + P.c0 + j * V;
    float mu[V], a[V], bb[V];
    gn_param<T, V, PIECE>(A.w, A.p_type, P.c0 + j * V, C, 1.f, a);
    gn_param<T, V, PIECE>(A.b, A.p_type, P.c0 + j * V, C, 0.f, bb);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int g = WIDE ? 0 : (int)A.by_cg.div(min(j * V + e, P.W - 1));
      mu[e] = mean[g];
      a[e] *= rstd[g];
    }
    gn_by_act(A.act, [&](auto act) {
      for (int r = first; r < r1; r += U * step) {
        raw_t raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (!WIDE && r == first) raw[u] = ahead[u];
          else if (r + u * step < r1) raw[u] = C.fetch(xp + (int64_t)(r + u * step) * A.xl);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (r + u * step >= r1) break;
          float v[V];
          C.expand(raw[u], v);
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] = gn_act<decltype(act)::value>(__builtin_fmaf(v[e] - mu[e], a[e], bb[e]));
          C.store(yp + (int64_t)(r + u * step) * A.yl, v, A.past);
        }
      }
    });
  }
}

// a block a sample window, block x of grid_b taking every grid_b-th sample
template <typename T, int V, bool WIDE, typename PIECE, int NT>
__global__ void __launch_bounds__(NT) k_gn_sample_fwd(gn_args A) {
  __shared__ gn_stats_lds<NT> S;
  __shared__ float mean[NT], rstd[NT];
  const int64_t x = A.by_nw.div(blockIdx.x);
  gn_place P = gn_where<NT>(A, x, (int)(blockIdx.x - (uint32_t)x * A.nw), 0);
  const float inv = 1.f / ((float)A.Cg * (float)A.L);
  for (int64_t b = x; b < A.B; b += A.grid_b) {                        // (the statistics' barriers keep the rounds apart)
    P.b = b;
    gn_apply_rows<T, V, WIDE, PIECE, NT>(A, P, 0, A.L, mean, rstd, [&]() {
      gn_block_stats<T, V, WIDE, PIECE, NT>(A, P, 0, A.L, S, [&](int g, float mu, float m2) {
        const float r = 1.f / sqrtf(m2 * inv + A.eps);
        mean[g] = mu;
        rstd[g] = r;
        if (A.mean) {
          A.mean[b * A.G + P.g0 + g] = mu;
          A.rstd[b * A.G + P.g0 + g] = r;
        }
      });
    });
  }
}

// tiles of positions: part[(b, group), tile] = (mean, M2)
template <typename T, int V, bool WIDE, typename PIECE, int NT>
__global__ void __launch_bounds__(NT) k_gn_stats(gn_args A) {
  __shared__ gn_stats_lds<NT> S;
  const uint32_t u = A.by_tiles.div(blockIdx.x);
  const int tile = (int)(blockIdx.x - u * A.tiles);
  const int64_t b = A.by_nw.div(u);
  const gn_place P = gn_where<NT>(A, b, (int)(u - (uint32_t)b * A.nw), tile);
  const int r0 = tile * A.tile_rows, r1 = min(A.L, r0 + A.tile_rows);
  gn_block_stats<T, V, WIDE, PIECE, NT>(A, P, r0, r1, S, [&](int g, float mu, float m2) {
    float2* o = (float2*)A.part + (b * A.G + P.g0 + g) * A.tiles + tile;
    *o = make_float2(mu, m2);
  });
}
template <typename T, int V, bool WIDE, typename PIECE, int NT>
__global__ void __launch_bounds__(NT) k_gn_apply(gn_args A) {
  __shared__ float mean[NT], rstd[NT];
  const uint32_t u = A.by_tiles.div(blockIdx.x);
  const int tile = (int)(blockIdx.x - u * A.tiles);
  const int64_t b = A.by_nw.div(u);
  const gn_place P = gn_where<NT>(A, b, (int)(u - (uint32_t)b * A.nw), tile);
  const int r0 = tile * A.tile_rows;
  gn_apply_rows<T, V, WIDE, PIECE, NT>(A, P, r0, min(A.L, r0 + A.tile_rows), mean, rstd, [&]() {
    const int lanes = gn_group_lanes<NT>(P.groups);
    const int lane = threadIdx.x & (lanes - 1), per = NT / lanes;
    const float total = (float)A.Cg * (float)A.L;
    for (int q0 = 0; q0 < P.groups; q0 += per) {
      const int g = q0 + threadIdx.x / lanes;
      const bool live = g < P.groups;
      const float2* o = (const float2*)A.part + (b * A.G + P.g0 + (live ? g : 0)) * A.tiles;
      const float first = o[0].x;                                        // (the tiles' means lie near each other: sums around the first one's)
      float a = 0.f, m2 = 0.f;
#pragma unroll 4
      for (int t = lane; t < A.tiles; t += lanes) {
        const float2 v = o[t];
        const float n = (float)A.Cg * (float)min(A.tile_rows, A.L - t * A.tile_rows), d = v.x - first;
        a = __builtin_fmaf(n, d, a);
        m2 += __builtin_fmaf(n * d, d, v.y);
      }
      a = row_team_sum(a, lanes);
      m2 = row_team_sum(m2, lanes);
      const float mu = first + a / total;
      m2 = gn_not_negative(__builtin_fmaf(-a / total, a, m2));
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
  });
}

// what the backward keeps of a thread's channels
template <int V>
struct gn_cols {
  float mu[V], rs[V], w[V], a[V], b[V];                                // a = rs w: z = (x - mu) a + b
};
template <typename T, int V, typename PIECE>
__device__ __forceinline__ void gn_columns(const gn_args& A, int64_t b, int c0, const PIECE& C, gn_cols<V>& K) {
  gn_param<T, V, PIECE>(A.w, A.p_type, c0, C, 1.f, K.w);
  gn_param<T, V, PIECE>(A.b, A.p_type, c0, C, 0.f, K.b);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int64_t g = b * A.G + A.by_cg.div(min(c0 + e, A.C - 1));
    K.mu[e] = A.mean[g];
    K.rs[e] = A.rstd[g];
    K.a[e] = K.rs[e] * K.w[e];
  }
}
// sums of dz and dz h over positions r0, r0 + step, .. < r1
template <typename T, int V, typename PIECE>
__device__ __forceinline__ void gn_channel_sums(const gn_args& A, const T* xp, const T* gp, const PIECE& C, int r0, int r1, int step,
                                                const gn_cols<V>& K, float (&sz)[V], float (&sh)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) sz[e] = sh[e] = 0.f;
  int r = r0;
  auto rows = [&](auto count, auto act) {
    constexpr int U = decltype(count)::value;
    typename PIECE::raw rx[U], rg[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      rx[u] = C.fetch(xp + (int64_t)(r + u * step) * A.xl);
      rg[u] = C.fetch(gp + (int64_t)(r + u * step) * A.gl);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[V], d[V];
      C.expand(rx[u], v);
      C.expand(rg[u], d);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xm = v[e] - K.mu[e];
        const float dz = d[e] * gn_slope<decltype(act)::value>(__builtin_fmaf(xm, K.a[e], K.b[e]));
        sz[e] += dz;
        sh[e] = __builtin_fmaf(dz, xm, sh[e]);
      }
    }
    r += U * step;
  };
  gn_by_act(A.act, [&](auto act) {
    while (r + step < r1) rows(std::integral_constant<int, 2>(), act);
    while (r < r1) rows(std::integral_constant<int, 1>(), act);
  });
#pragma unroll
  for (int e = 0; e < V; ++e) sh[e] *= K.rs[e];
}
// dx of those positions; s1, s2: of each channel's group, divided by m
template <typename T, int V, typename PIECE>
__device__ __forceinline__ void gn_dx_rows(const gn_args& A, const T* xp, const T* gp, T* dp, const PIECE& C, int r0, int r1, int step,
                                           const gn_cols<V>& K, const float (&s1)[V], const float (&s2)[V]) {
  float k1[V], k2[V];                                                  // dx = dz a - rs s1 - (x - mu) rs^2 s2
#pragma unroll
  for (int e = 0; e < V; ++e) {
    k1[e] = -K.rs[e] * s1[e];
    k2[e] = -K.rs[e] * K.rs[e] * s2[e];
  }
  int r = r0;
  auto rows = [&](auto count, auto act) {
    constexpr int U = decltype(count)::value;
    typename PIECE::raw rx[U], rg[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      rx[u] = C.fetch(xp + (int64_t)(r + u * step) * A.xl);
      rg[u] = C.fetch(gp + (int64_t)(r + u * step) * A.gl);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[V], d[V];
      C.expand(rx[u], v);
      C.expand(rg[u], d);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xm = v[e] - K.mu[e];
        const float dz = d[e] * gn_slope<decltype(act)::value>(__builtin_fmaf(xm, K.a[e], K.b[e]));
        v[e] = __builtin_fmaf(dz, K.a[e], __builtin_fmaf(xm, k2[e], k1[e]));
      }
      C.store(dp + (int64_t)(r + u * step) * A.yl, v, A.past);
    }
    r += U * step;
  };
  gn_by_act(A.act, [&](auto act) {
    while (r + step < r1) rows(std::integral_constant<int, 2>(), act);
    while (r < r1) rows(std::integral_constant<int, 1>(), act);
  });
}

// the window's channel sums over the block's positions -> out[0: dz, 1: dz h][C]; every thread takes part
template <int V, int NT>
__device__ __forceinline__ void gn_fold_window(const gn_args& A, const gn_place& P, const float* cz, const float* ch, float* out) {
  const int lanes = gn_group_lanes<NT>(P.W), lane = threadIdx.x & (lanes - 1);
  for (int c0 = 0; c0 < P.W; c0 += NT / lanes) {
    const int c = c0 + threadIdx.x / lanes;
    float a = 0.f, d = 0.f;
    if (c < P.W)
      for (int q = lane; q < A.rp; q += lanes) {
        a += cz[q * A.nvec * V + c];
        d += ch[q * A.nvec * V + c];
      }
    a = row_team_sum(a, lanes);
    d = row_team_sum(d, lanes);
    if (c < P.W && lane == 0) {
      out[c] = a;
      out[A.C + c] = d;
    }
  }
}

// a block a sample window, block x of grid_b taking every grid_b-th sample: part[x][0: dz, 1: dz h][C] holds the sums over its samples
template <typename T, int V, bool WIDE, typename PIECE, int NT>
__global__ void __launch_bounds__(NT) k_gn_sample_bwd(gn_args A) {
  __shared__ __align__(16) float cz[NT * V], ch[NT * V];   // [rp][nvec V]; WIDE: s1, s2 of a thread
  __shared__ float g1[NT], g2[NT];
  const int64_t x = A.by_nw.div(blockIdx.x);
  const gn_place P = gn_where<NT>(A, x, (int)(blockIdx.x - (uint32_t)x * A.nw), 0);
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
        const PIECE C(have, P.W < V);
        gn_columns<T, V, PIECE>(A, b, P.c0 + P.j * V, C, K);
        gn_channel_sums<T, V, PIECE>(A, xp + P.j * V, gp + P.j * V, C, P.ri, A.L, A.rp, K, sz, sh);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          tz[e] += sz[e];
          th[e] += sh[e];
          sz[e] *= K.w[e];
          sh[e] *= K.w[e];
        }
        gn_lds_put<V>(cz + (P.ri * A.nvec + P.j) * V, sz);
        gn_lds_put<V>(ch + (P.ri * A.nvec + P.j) * V, sh);
      }
    } else {
      float s1 = 0.f, s2 = 0.f;
      for (int j = threadIdx.x; j < A.nvec; j += NT) {
        const int have = P.W - j * V;
        float sz[V], sh[V];
        const PIECE C(have, false);
        gn_columns<T, V, PIECE>(A, b, P.c0 + j * V, C, K);
        gn_channel_sums<T, V, PIECE>(A, xp + j * V, gp + j * V, C, 0, A.L, 1, K, sz, sh);
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
      const int lanes = WIDE ? 64 : gn_group_lanes<NT>(P.groups);
      const int lane = threadIdx.x & (lanes - 1), per = NT / lanes;
      for (int q0 = 0; q0 < P.groups; q0 += per) {
        const int g = q0 + threadIdx.x / lanes;
        const bool live = g < P.groups;
        float s1 = 0.f, s2 = 0.f;
        if (live) {
          for (int i = lane; i < (WIDE ? NT : A.rp * A.Cg); i += lanes) {
            const int ri = WIDE ? 0 : (int)A.by_cg.div((uint32_t)i);
            const int at = WIDE ? i : ri * A.nvec * V + g * A.Cg + i - ri * A.Cg;
            s1 += cz[at];
            s2 += ch[at];
          }
        }
        s1 = row_team_sum(s1, lanes);
        s2 = row_team_sum(s2, lanes);
        if (live && lane == 0) {
          g1[g] = s1 * inv;
          g2[g] = s2 * inv;
        }
      }
      __syncthreads();
      float s1[V], s2[V];
      for (int j = WIDE ? (int)threadIdx.x : P.j; j < A.nvec; j += WIDE ? NT : A.nvec) {
        const int have = WIDE || P.on ? P.W - j * V : 0;
        if (have <= 0) break;
        const PIECE C(have, P.W < V);
        if (WIDE) gn_columns<T, V, PIECE>(A, b, P.c0 + j * V, C, K);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int g = WIDE ? 0 : (int)A.by_cg.div(min(j * V + e, P.W - 1));
          s1[e] = g1[g];
          s2[e] = g2[g];
        }
        gn_dx_rows<T, V, PIECE>(A, xp + j * V, gp + j * V, dp + j * V, C, WIDE ? 0 : P.ri, A.L, WIDE ? 1 : A.rp, K, s1, s2);
      }
    }
    __syncthreads();                                                    // cz, ch, g1, g2 are free again
  }
  if (WIDE || !out) return;
  const int have = P.on ? P.W - P.j * V : 0;
  if (have > 0) {
    gn_lds_put<V>(cz + (P.ri * A.nvec + P.j) * V, tz);
    gn_lds_put<V>(ch + (P.ri * A.nvec + P.j) * V, th);
  }
  __syncthreads();
  gn_fold_window<V, NT>(A, P, cz, ch, out);
}

// tiles of positions: part[b, tile][0: dz, 1: dz h][C]
template <typename T, int V, bool WIDE, typename PIECE, int NT>
__global__ void __launch_bounds__(NT) k_gn_bwd_sums(gn_args A) {
  __shared__ __align__(16) float cz[NT * V], ch[NT * V];
  const uint32_t u = A.by_tiles.div(blockIdx.x);
  const int tile = (int)(blockIdx.x - u * A.tiles);
  const int64_t b = A.by_nw.div(u);
  const gn_place P = gn_where<NT>(A, b, (int)(u - (uint32_t)b * A.nw), tile);
  const int r0 = tile * A.tile_rows, r1 = min(A.L, r0 + A.tile_rows);
  const T* xp = (const T*)A.x + b * A.xb + P.c0;
  const T* gp = (const T*)A.dy + b * A.gb + P.c0;
  float* out = A.part + (b * A.tiles + tile) * 2 * A.C + P.c0;
  gn_cols<V> K;
  float sz[V], sh[V];
  if constexpr (WIDE) {
    for (int j = threadIdx.x; j < A.nvec; j += NT) {
      const int have = P.W - j * V;
      const PIECE C(have, false);
      gn_columns<T, V, PIECE>(A, b, P.c0 + j * V, C, K);
      gn_channel_sums<T, V, PIECE>(A, xp + j * V, gp + j * V, C, r0, r1, 1, K, sz, sh);
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
      const PIECE C(have, P.W < V);
      gn_columns<T, V, PIECE>(A, b, P.c0 + P.j * V, C, K);
      gn_channel_sums<T, V, PIECE>(A, xp + P.j * V, gp + P.j * V, C, r0 + P.ri, r1, A.rp, K, sz, sh);
      gn_lds_put<V>(cz + (P.ri * A.nvec + P.j) * V, sz);
      gn_lds_put<V>(ch + (P.ri * A.nvec + P.j) * V, sh);
    }
    __syncthreads();
    gn_fold_window<V, NT>(A, P, cz, ch, out);
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
      const int cc = g * A.Cg + c;
      const float w = !A.w ? 1.f : A.p_type == OGL_F32 ? ((const float*)A.w)[cc] : (float)((const T*)A.w)[cc];
      s1 += p[(int64_t)t * 2 * A.C + c] * w;
      s2 += p[(int64_t)t * 2 * A.C + A.C + c] * w;
    }
    s1 = row_team_sum(s1, 64);
    s2 = row_team_sum(s2, 64);
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
  if (col < 2 * (int64_t)A.C) {
#pragma unroll 8
    for (int64_t r = slice; r < rows; r += 64) a += A.part[r * 2 * A.C + col];
  }
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

template <typename T, int V, bool WIDE, typename PIECE, int NT>
__global__ void __launch_bounds__(NT) k_gn_bwd_apply(gn_args A) {
  const uint32_t u = A.by_tiles.div(blockIdx.x);
  const int tile = (int)(blockIdx.x - u * A.tiles);
  const int64_t b = A.by_nw.div(u);
  const gn_place P = gn_where<NT>(A, b, (int)(u - (uint32_t)b * A.nw), tile);
  const int r0 = tile * A.tile_rows, r1 = min(A.L, r0 + A.tile_rows);
  const T* xp = (const T*)A.x + b * A.xb + P.c0;
  const T* gp = (const T*)A.dy + b * A.gb + P.c0;
  T* dp = (T*)A.y + b * A.yb + P.c0;
  for (int j = WIDE ? (int)threadIdx.x : P.j; j < A.nvec; j += WIDE ? NT : A.nvec) {
    const int have = WIDE || P.on ? P.W - j * V : 0;
    if (have <= 0) return;
    const PIECE C(have, P.W < V);
    gn_cols<V> K;
    gn_columns<T, V, PIECE>(A, b, P.c0 + j * V, C, K);
    float s1[V], s2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float* s = A.sums + (b * A.G + P.g0 + (int)A.by_cg.div(min(j * V + e, P.W - 1))) * 2;
      s1[e] = s[0];
      s2[e] = s[1];
    }
    gn_dx_rows<T, V, PIECE>(A, xp + j * V, gp + j * V, dp + j * V, C, r0 + (WIDE ? 0 : P.ri), r1, WIDE ? 1 : A.rp, K, s1, s2);
  }
}

// ================================================================ launches ====================================================================
#define GN_LAUNCH_N(THREADS, K, GRID)                                                          \
  do {                                                                                         \
    const int64_t grid_ = (GRID);                                                              \
    if (grid_ * (THREADS) > (int64_t)UINT32_MAX) return OGL_EINVAL;                            \
    hipLaunchKernelGGL(HIP_KERNEL_NAME(K), dim3((unsigned)grid_), dim3(THREADS), 0, st, A);    \
  } while (0)
#define GN_LAUNCH(K, GRID) GN_LAUNCH_N(GN_THREADS, K, GRID)

template <typename T, int V>
int gn_forward(const gn_args& A, const gn_plan& P, hipStream_t st) {
  typedef row_piece<T, V> cut;
  typedef row_even<T, V> even;
  typedef row_whole<T, V> whole;
  if (P.rows) {
    const int64_t grid = ogl_cdiv(ogl_cdiv(A.B, P.r) * A.G, P.block ? 1 : 4 * A.tw);
#define GN_ROWS(NV, R, BLOCK)                                                  \
  do {                                                                         \
    if (P.even) GN_LAUNCH((k_gn_rows_fwd<T, V, NV, R, BLOCK, even>), grid);    \
    else GN_LAUNCH((k_gn_rows_fwd<T, V, NV, R, BLOCK, cut>), grid);            \
  } while (0)
    if (P.block) {                                                     // (more than 320 pieces: two a lane at least)
      if (P.nv == 2) GN_ROWS(2, 1, true);
      else GN_ROWS(4, 1, true);
    } else {
      if (P.nv == 1 && P.r == 4) GN_ROWS(1, 4, false);
      else if (P.nv == 1) GN_ROWS(1, 1, false);
      else if (P.nv == 2 && P.r == 2) GN_ROWS(2, 2, false);
      else if (P.nv == 2) GN_ROWS(2, 1, false);
      else if (P.nv == 3) GN_ROWS(3, 1, false);
      else GN_ROWS(5, 1, false);
    }
#undef GN_ROWS
    return OGL_OK;
  }
  if (A.tiles == 1) {
    const int64_t grid = (int64_t)A.grid_b * A.nw;
    if (P.wide) GN_LAUNCH((k_gn_sample_fwd<T, V, true, cut, GN_THREADS>), grid);
    else if (P.threads == 64 && P.even) GN_LAUNCH_N(64, (k_gn_sample_fwd<T, V, false, whole, 64>), grid);
    else if (P.threads == 64) GN_LAUNCH_N(64, (k_gn_sample_fwd<T, V, false, cut, 64>), grid);
    else if (P.even) GN_LAUNCH((k_gn_sample_fwd<T, V, false, whole, GN_THREADS>), grid);
    else GN_LAUNCH((k_gn_sample_fwd<T, V, false, cut, GN_THREADS>), grid);
    return OGL_OK;
  }
  const int64_t grid = A.B * A.nw * A.tiles;
  if (P.wide) {
    GN_LAUNCH((k_gn_stats<T, V, true, cut, GN_THREADS>), grid);
    GN_LAUNCH((k_gn_apply<T, V, true, cut, GN_THREADS>), grid);
  } else {
    if (P.even) GN_LAUNCH((k_gn_stats<T, V, false, whole, GN_THREADS>), grid);
    else GN_LAUNCH((k_gn_stats<T, V, false, cut, GN_THREADS>), grid);
    if (P.even) GN_LAUNCH((k_gn_apply<T, V, false, whole, GN_THREADS>), grid);
    else GN_LAUNCH((k_gn_apply<T, V, false, cut, GN_THREADS>), grid);
  }
  return OGL_OK;
}

template <typename T, int V>
int gn_backward(const gn_args& A, const gn_plan& P, void* dw, void* db, hipStream_t st) {
  typedef row_piece<T, V> cut;
  typedef row_even<T, V> even;
  typedef row_whole<T, V> whole;
  int64_t rows = 0, groups = 0;
  if (P.rows) {
    const int64_t sets = ogl_cdiv(A.G, A.tg), z = ogl_cdiv(sets, 65535);   // (a launch's y ends at 65535: 2^22 groups of one channel are 65536 sets)
    const dim3 grid((unsigned)A.chunks, (unsigned)ogl_cdiv(sets, z), (unsigned)z);
#define GN_ROWS(NV, R, BLOCK)                                                                                         \
  do {                                                                                                                \
    if (P.even) hipLaunchKernelGGL((k_gn_rows_bwd<T, V, NV, R, BLOCK, even>), grid, dim3(GN_THREADS), 0, st, A);      \
    else hipLaunchKernelGGL((k_gn_rows_bwd<T, V, NV, R, BLOCK, cut>), grid, dim3(GN_THREADS), 0, st, A);              \
  } while (0)
    if (P.block) {                                                     // (more than 320 pieces, in 16-bit types 192)
      if (P.nv == 2) GN_ROWS(2, 1, true);
      else if (P.nv > 2) GN_ROWS(4, 1, true);
      else if constexpr (V == 8) GN_ROWS(1, 1, true);
    } else {
      if (P.nv == 1 && P.r > 1) GN_ROWS(1, 2, false);
      else if (P.nv == 1) GN_ROWS(1, 1, false);
      else if (P.nv == 2) GN_ROWS(2, 1, false);
      else if (P.nv == 3) GN_ROWS(3, 1, false);
      else if constexpr (V == 4) GN_ROWS(5, 1, false);
    }
#undef GN_ROWS
    rows = A.chunks;
  } else if (A.tiles == 1) {
    const int64_t grid = (int64_t)A.grid_b * A.nw;
    if (P.wide) GN_LAUNCH((k_gn_sample_bwd<T, V, true, cut, GN_THREADS>), grid);
    else if (P.threads == 64 && P.even) GN_LAUNCH_N(64, (k_gn_sample_bwd<T, V, false, whole, 64>), grid);
    else if (P.threads == 64) GN_LAUNCH_N(64, (k_gn_sample_bwd<T, V, false, cut, 64>), grid);
    else if (P.even) GN_LAUNCH((k_gn_sample_bwd<T, V, false, whole, GN_THREADS>), grid);
    else GN_LAUNCH((k_gn_sample_bwd<T, V, false, cut, GN_THREADS>), grid);
    rows = A.grid_b;
  } else {
    if (P.wide) GN_LAUNCH((k_gn_bwd_sums<T, V, true, cut, GN_THREADS>), A.B * A.nw * A.tiles);
    else if (P.even) GN_LAUNCH((k_gn_bwd_sums<T, V, false, whole, GN_THREADS>), A.B * A.nw * A.tiles);
    else GN_LAUNCH((k_gn_bwd_sums<T, V, false, cut, GN_THREADS>), A.B * A.nw * A.tiles);
    rows = A.B * A.tiles;
    groups = A.write_dx ? A.B * A.G : 0;
  }
  const int64_t folds = dw || db ? ogl_cdiv(2 * (int64_t)A.C, 16) : 0;
  if ((groups + folds) * 1024 > (int64_t)UINT32_MAX) return OGL_EINVAL;
  if (groups + folds > 0)
    hipLaunchKernelGGL(k_gn_fold<T>, dim3((unsigned)(groups + folds)), dim3(1024), 0, st, A, groups, rows, dw, db);
  if (groups > 0) {
    if (P.wide) GN_LAUNCH((k_gn_bwd_apply<T, V, true, cut, GN_THREADS>), A.B * A.nw * A.tiles);
    else if (P.even) GN_LAUNCH((k_gn_bwd_apply<T, V, false, whole, GN_THREADS>), A.B * A.nw * A.tiles);
    else GN_LAUNCH((k_gn_bwd_apply<T, V, false, cut, GN_THREADS>), A.B * A.nw * A.tiles);
  }
  return OGL_OK;
}
