/*
 * ogl_rows.h — the row operators of libogl_hip.so: rows of float32, bfloat16 or float16, rows kept in 8 bits, and products of those.
 * Conventions and status codes are those of ogl_hip.h, the base header; these operators stand beside the train step, which calls them only where a
 * layer or a pass asks for them.
 * `ld*` count elements; rows need the alignment of one element only.  At most 2^32 - 1 threads a launch (about 3e10 elements): OGL_EINVAL above.
 */
#ifndef OGL_ROWS_H
#define OGL_ROWS_H

#include "ogl_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { OGL_F32 = 0, OGL_BF16 = 1, OGL_F16 = 2 };
enum { OGL_ROWS_INT8 = 0, OGL_ROWS_E4M3 = 1 };

/* A cache of n rows in 8 bits: codes [n, ldc] bytes (64-byte aligned, ldc a multiple of 64, zeros behind column `width`) and one float32 scale for
 * every `group` columns of a row, scales [n, ceil(width / group)] (a multiple of 8 columns, or group >= width: one scale a row).
 *   a = max(max |x|, 2^-80) over the group;  s = fl32(a / Q), Q = 127 (int8), 448 (e4m3);  code = the exact quotient x / s rounded to nearest even
 * A group that holds an infinity or a NaN: s = NaN, codes 0 — it reads back as NaN.
 *   write  row i of x goes to slots[i], or to start + i where slots is NULL (then [start, start + m) has to lie inside the cache).  Slots outside
 *          [0, n) are skipped; of rows with the same slot the LAST stands.  The workspace needs no particular contents and keeps none.
 *          m * groups and m below 2^31, n below 2^32, rows of x and of codes less than 2^31 elements apart.
 *   read   out[i, :] = fl32(code * s), rounded once to out_type, of row rows[i] (NULL: row i, m <= n); ids outside [0, n) yield zero rows.
 * Writes and reads of the same rows are ordered by their stream only. */
int64_t ogl_quant_rows_workspace_bytes(int64_t m, int64_t n, int by_slots);
int ogl_quant_rows_write(const void* x, int64_t ldx, int x_type, int64_t m, int width, const int64_t* slots, int64_t start, void* codes,
                         int64_t ldc, int format, float* scales, int64_t n, int group, void* workspace, int64_t workspace_bytes,
                         ogl_stream_t stream);
int ogl_quant_rows_read(const void* codes, int64_t ldc, int format, const float* scales, int64_t n, int width, int group, const int64_t* rows,
                        int64_t m, void* out, int64_t ldo, int out_type, ogl_stream_t stream);

/* y[m, n] = act((sx[r] sw[n]) * sum_k x[r, k] w[n, k] + bias[n]), r = rows[m] (NULL: m, then M <= nrows): the product of two caches in int8 with
 * one scale a row (a weight's rows are its output channels), act = relu or none, y in y_type.  The sum is exact; everything behind it is float32.
 * x [nrows, ldx], w [N, ldw]: 64-byte aligned, ld a multiple of 64, zeros behind column K in at least one of them; 1 <= K < 131072.
 * Rows outside [0, nrows) count as zero rows (y = act(bias); NaN where a weight's scale is).  Tables of 2^38 bytes and more, an empty table (nrows = 0
 * with M > 0), N of 2^31 - 256 and more (with M <= 16: 2^27 - 15 and more, the launch's threads): OGL_EINVAL. */
int ogl_linear_i8(const void* x, int64_t ldx, const float* sx, const int64_t* rows, int64_t nrows, int64_t M, int K, const void* w, int64_t ldw,
                  const float* sw, int N, const float* bias, int relu, void* y, int64_t ldy, int y_type, ogl_stream_t stream);

/* Group norm with an activation, channels last.  x [B, L, C]: element (b, l, c) at x[b xb + l xl + c]; G groups of C / G channels.
 *   mean, var over the L C / G values of a (sample, group);  rstd = 1 / sqrt(var + eps);  y = act((x - mean) rstd w[c] + b[c])
 * w, b (nullable: 1 and 0) in p_type, which is OGL_F32 or x_type; y, dy, dx in x_type; mean, rstd float32 [B, G] (both or neither in the forward).
 * silu is off by at most (1.25 |z| + 4) 2^-24 of its value (|z| <= 80), gelu by 3.2e-7 |z| (from a polynomial: 5e-4 of the value at z = -4, 4e-3 at -6).
 * The backward writes dx (nullable), dw and db (nullable, [C] in p_type); statistics and sums are float32 in a fixed order (no atomics).
 * L <= 2^30, C <= 2^22.  An empty x (B or L of 0): the forward has nothing to do, the backward returns OGL_EINVAL (its sums are zeros). */
enum { OGL_ACT_NONE = 0, OGL_ACT_RELU = 1, OGL_ACT_SILU = 2, OGL_ACT_GELU = 3 };
int64_t ogl_group_norm_workspace_bytes(int64_t B, int64_t L, int C, int G, int x_type, int backward);
int ogl_group_norm_fwd(const void* x, int64_t xb, int64_t xl, int x_type, int64_t B, int64_t L, int C, int G, const void* w, const void* b, int p_type,
                       float eps, int act, void* y, int64_t yb, int64_t yl, float* mean, float* rstd, void* workspace, int64_t workspace_bytes,
                       ogl_stream_t stream);
int ogl_group_norm_bwd(const void* dy, int64_t gb, int64_t gl, const void* x, int64_t xb, int64_t xl, int x_type, int64_t B, int64_t L, int C, int G,
                       const void* w, const void* b, int p_type, int act, const float* mean, const float* rstd, void* dx, int64_t dxb, int64_t dxl,
                       void* dw, void* db, void* workspace, int64_t workspace_bytes, ogl_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* OGL_ROWS_H */
