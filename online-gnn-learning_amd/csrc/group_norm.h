// Group norm: what its host code (group_norm.hip) and its kernels (group_norm_kernels.h, a source file for each type of x) share.
#pragma once
#include <algorithm>
#include <type_traits>
#include "row_types.h"

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
  bool past;                     // y (dx) is stored past the caches
  float eps;
  // maps: windows of gw groups, nvec 16-byte pieces wide; rp positions side by side; tiles of tile_rows positions
  int gw, nw, nvec, rp, tiles, tile_rows, grid_b;
  // rows: lanes of a team, teams of a wave; the backward's wave has tg groups x rpw rows
  int lanes, tw, tg, rpw, chunks;
  ogl_div by_g, by_cg, by_lanes, by_tg, by_nvec, by_nw, by_tiles;
};

struct gn_plan {
  bool rows, block, wide;
  bool even;                   // every group (maps: window of groups) is whole pieces
  int threads;                 // maps: of a block
  int nv, r;                   // rows: pieces a lane, rows a team
  int64_t part, sums;          // floats of workspace
};

// the launches of a plan for x of type T in pieces of V
template <typename T, int V>
int gn_forward(const gn_args& A, const gn_plan& P, hipStream_t st);
template <typename T, int V>
int gn_backward(const gn_args& A, const gn_plan& P, void* dw, void* db, hipStream_t st);
