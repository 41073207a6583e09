// Group norm: which form a call takes, and its C entries (the kernels and their reasons: group_norm_kernels.h).
#include "group_norm.h"

static gn_plan gn_make(gn_args& A, int x_type, bool backward) {
  gn_plan P = {};
  const int V = x_type == OGL_F32 ? 4 : 8;
  const int pieces = (int)ogl_cdiv(A.Cg, V);
  A.by_cg = ogl_div::make((uint32_t)A.Cg);
  P.rows = A.L == 1 && pieces <= 4 * GN_THREADS;
  if (P.rows) {
    // A team inside a wave: a lane for each piece up to 64, then up to 5 pieces a lane (3 in the backward of 16-bit types, for its registers).  Above
    // that the block is the team.  Lanes that have no piece cost as much as those that do (the vector units bound these kernels), and so do teams of
    // fewer lanes with more pieces each: 62500 x 600 in 30 groups (5 pieces) takes 64 / 87 us forward / backward, with 2 lanes x 3 pieces 22 / 45 us more.
    const int most = backward && V == 8 ? 3 : 5;
    P.block = pieces > 64 * most;
    A.lanes = P.block ? 64 : std::min(pieces, 64);
    P.nv = (int)ogl_cdiv(pieces, P.block ? GN_THREADS : A.lanes);
    A.tw = 64 / A.lanes;
    A.tg = P.block ? 1 : (int)ogl_cdiv(A.G, ogl_cdiv(A.G, A.tw));      // groups of a wave: the row's, in equal shares
    A.rpw = P.block ? 1 : std::max(1, A.tw / A.tg);
    // Several rows a team where that still leaves eight blocks a CU, so that their loads are on their way together: forward 1 row 93 us, 2 68 us, 4 64 us,
    // 8 66 us; in the backward two pieces' registers are what a wave has room for.
    P.r = P.nv <= 2 && !P.block && A.B * A.G * A.lanes >= 4 * 2048 * GN_THREADS ? (backward ? 2 : 4) / P.nv : 1;
    // at most so many blocks: each leaves 2 C partial sums
    A.chunks = (int)std::min<int64_t>(ogl_cdiv(A.B, (P.block ? 1 : 4 * A.rpw) * P.r), std::max<int64_t>(1, 1024 / ogl_cdiv(A.G, A.tg)));
    A.by_lanes = ogl_div::make((uint32_t)A.lanes);
    P.even = A.Cg % V == 0;
    A.by_tg = ogl_div::make((uint32_t)A.tg);
    P.part = backward ? (int64_t)A.chunks * 2 * A.C : 0;
    A.by_g = ogl_div::make((uint32_t)A.G);
    return P;
  }
  // Small samples (up to 8 pieces a lane): a wave each, so that four times as many are on their way; a block's time goes into its steps' latencies, not
  // into its loads.  62500 x 2 x 256 bfloat16 forward / backward 295 / 507 -> 105 / 151 us, 20000 x 8 x 96 float32 147 / 148 -> 49 / 73 us; samples of
  // 2048 pieces are as fast in blocks (3000 x 16 x 512 float32 44 / 84 us, a wave each 50 / 86).
  P.threads = (int64_t)A.L * ogl_cdiv(A.C, V) <= 512 && pieces <= 64 && A.B >= 1024 ? 64 : GN_THREADS;
  // Windows of whole groups, at most a block's pieces wide, that keep most threads busy (pieces x positions side by side of a block) and waste least at
  // the last window; of equals the widest.  One group wider than that: WIDE.
  P.wide = pieces > GN_THREADS;
  A.gw = 1;
  if (!P.wide) {
    double best = -1;
    for (int gw = std::min(A.G, P.threads); gw >= 1; --gw) {
      const int nvec = (int)ogl_cdiv((int64_t)gw * A.Cg, V);
      if (nvec > P.threads) continue;
      if (gw < A.G && (int64_t)gw * A.Cg * (16 / V) < 128) break;      // windows of less than a line
      const double busy = (double)(P.threads / nvec * nvec) / P.threads * ((double)gw * A.Cg / ((double)nvec * V)) *
                          ((double)A.G / (double)(ogl_cdiv(A.G, gw) * gw));
      if (busy > best + 0.02) best = busy, A.gw = gw;
    }
  }
  A.nw = (int)ogl_cdiv(A.G, A.gw);
  A.nvec = (int)ogl_cdiv((int64_t)A.gw * A.Cg, V);
  A.rp = P.wide ? 1 : P.threads / A.nvec;
  P.even = A.C % V == 0 && (int64_t)A.gw * A.Cg % V == 0;
  // a block a sample window where there are enough of them to fill the card or little to do in each; else tiles of 8 positions a thread or more
  const int64_t blocks = A.B * A.nw;
  int64_t tiles = 1;
  if (blocks < 1024 && A.L > A.rp * 16) tiles = std::min<int64_t>(std::min<int64_t>(ogl_cdiv(A.L, A.rp * 8), ogl_cdiv(2048, blocks)), 256);
  A.tile_rows = (int)ogl_cdiv(A.L, tiles);
  A.tiles = (int)ogl_cdiv(A.L, A.tile_rows);
  A.by_nvec = ogl_div::make((uint32_t)A.nvec);
  A.by_nw = ogl_div::make((uint32_t)A.nw);
  A.by_tiles = ogl_div::make((uint32_t)A.tiles);
  // samples side by side: the backward's blocks each leave 2 C partial sums, the forward's only have to stay below 2^32 threads
  A.grid_b = (int)std::min<int64_t>(A.B, std::max<int64_t>(1, (!backward ? 1 << 23 : P.threads == 64 ? 4096 : 2048) / A.nw));
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
  A.past = (double)B * (double)L * C * (x_type == OGL_F32 ? 4 : 2) >= (double)ROW_NT_BYTES;
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
  A.past = (double)B * (double)L * C * (x_type == OGL_F32 ? 4 : 2) >= (double)ROW_NT_BYTES;
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
