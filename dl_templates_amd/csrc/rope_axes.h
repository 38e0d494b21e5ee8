// Rotation by positions with several axes: operands, and the map of pairs to dims.
//
// Axis a turns R_a pairs of dims by (cos, sin) = table_a[position on axis a][pair]; pair i of axis a, with off_a = R_0 + .. + R_(a-1):
//   layout blocks: dims 2 off_a + i and 2 off_a + R_a + i   (an axis has a run of 2 R_a dims)
//   layout halves: dims off_a + i and P + off_a + i         (P = sum R: all first halves, then all second ones)
// A negative position leaves the axis' dims as they are; positions are clamped to the table's last row.
#pragma once
#include "dlt_internal.hpp"

struct RopeAxes {
  const int32_t* pos;      // NULL: the token's place in its sequence, on every axis (append)
  int64_t pa, pb, pn;      // its strides: axis, batch, token
  const float* tab[DLT_ROPE_AXES_MAX];
  int64_t ts[DLT_ROPE_AXES_MAX];
  int32_t len[DLT_ROPE_AXES_MAX], end[DLT_ROPE_AXES_MAX];   // end: off_a + R_a
  int32_t n, pairs, halves, inverse;
};

// axis of pair i, the first pair of that axis, and how many it has
DLT_HD int rope_axes_axis(const RopeAxes& r, int i, int& off, int& R) {
  int a = 0;
  off = 0;
  R = r.end[0];
#pragma unroll
  for (int k = 0; k + 1 < DLT_ROPE_AXES_MAX; k++)
    if (k + 1 < r.n && i >= r.end[k]) { a = k + 1; off = r.end[k]; R = r.end[k + 1] - off; }
  return a;
}

// y0 = x0 c - x1 s, y1 = x0 s + x1 c
__device__ inline float mix(float x, float c, float other, float s) {
#pragma clang fp contract(off)
  const float a = x * c, b = other * s;
  return a + b;
}

// Rows of the tables for token t_ of sequence b at `place` in it (of row 0 where it has no position, so that loads need no branch), bit a of `on`: axis a turns it
struct TableRows { const float* p[DLT_ROPE_AXES_MAX]; unsigned on; };
__device__ inline TableRows table_rows(const RopeAxes& r, int b, int t_, int place, bool live) {
  TableRows t;
  t.on = 0;
  int pos[DLT_ROPE_AXES_MAX];
#pragma unroll
  for (int a = 0; a < DLT_ROPE_AXES_MAX; a++) pos[a] = r.pos == nullptr ? place : a < r.n ? r.pos[a * r.pa + b * r.pb + t_ * r.pn] : -1;
#pragma unroll
  for (int a = 0; a < DLT_ROPE_AXES_MAX; a++) {
    t.p[a] = r.tab[a] + dlt_imax(dlt_imin(pos[a], r.len[a] - 1), 0) * r.ts[a];
    t.on |= (a < r.n && pos[a] >= 0 && live ? 1u : 0u) << a;
  }
  return t;
}
// row of a pair's axis, at the pair; its bit of `on`
__device__ inline const float* pair_row(const RopeAxes& r, const TableRows& t, int pair, bool& on) {
  const float* row = t.p[0];
  unsigned bit = 1;
  int off = 0;
#pragma unroll
  for (int a = 1; a < DLT_ROPE_AXES_MAX; a++)
    if (a < r.n && pair >= r.end[a - 1]) { row = t.p[a]; off = r.end[a - 1]; bit = 1u << a; }
  on = (t.on & bit) != 0;
  return row + 2 * (pair - off);
}

// One call of the kernels in rope_axes.hip: rows of up to three tensors, token by token
struct RotStream {
  const void* src;
  void* dst;
  int64_t ss[4], ds[4];   // batch (pages: page), head, token, dim
  int32_t H, C;           // heads, dims of a row
  int32_t rot;            // the rows are rotated
  int32_t paged;          // dst is a cache of pages
};
struct RotArgs {
  RotStream s[3];
  int32_t n;              // streams
  int32_t B, T, heads;    // tokens per sequence, heads of all streams
  int32_t hb;             // heads that a thread walks
  RopeAxes r;             // n = 0: nothing is rotated
  const int32_t *table, *seq, *n_new;   // pages; table NULL: none
  int64_t tbs;
  int32_t cols, n_pages, page;
};
int dlt_rotate_rows(RotArgs& a, int dtype, const char* who, hipStream_t stream);
// fills `r` after checking it against rows of n_dim dims
int dlt_rope_axes_make(const dlt_rope_axes_t* d, int64_t n_dim, bool need_pos, int inverse, const char* who, RopeAxes& r);
