// Rotation by positions with several axes (rope_axes.h), alone or on the way into a cache of pages, for gfx950.
//
// Pure streaming: every element is read once and written once.  A thread owns one (token, part of a row): up to 8 pairs of one axis, or up to 8 dims
// that are not rotated.  Its (cos, sin) pairs are fetched once and stay in registers while it walks the heads of q, k and v, so table traffic is
// shared by the heads; the first heads' elements are asked for before them, since nothing about them depends on positions or pages.
// A part's two runs of dims start wherever the sections put them: accesses are as wide as the part (16 bytes of a 2-byte type for 8 dims), at any alignment of
// the element, and parts of fewer than 8 pairs move in pieces of 4, 2 and 1.  Rows with other strides than 1 take a kernel of one pair per thread.
// Rotated values are formed in 32 bits, each product rounded before the sum as in the 2D rotation, and rounded once.
// 16 + 16 heads of 49152 tokens, d = 128, bf16: 149 us, 5.4 TB/s (a large copy: 5.15).  Memory bound; small calls take the launch.
#include "kernargs.h"
#include "rope_axes.h"

namespace {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
template <typename T> struct alignas(16) Vec8 { T v[8]; };

// N elements from any address of the element's alignment
template <int N, typename T>
__device__ inline void load_run(T* v, const T* p) { __builtin_memcpy(v, p, N * sizeof(T)); }
template <int N, typename T>
__device__ inline void store_run(T* p, const T* v) {
  // streaming stores: see attn_common.hpp; 163 -> 151 us for 16 + 16 heads of 49152 tokens, d = 128, 25 -> 22 us for the prompts of an append
  if constexpr (N * sizeof(T) == 16) {   // (32-bit elements: 32 bytes a lane in two stores, each of half lines: 20 -> 30 us for 120 MB)
    typedef unsigned uv4 __attribute__((ext_vector_type(4)));
    typedef uv4 uv __attribute__((aligned(2)));
    uv x[N * sizeof(T) / 16];
    __builtin_memcpy(x, v, N * sizeof(T));
#pragma unroll
    for (int i = 0; i < (int)(N * sizeof(T) / 16); i++) __builtin_nontemporal_store(x[i], reinterpret_cast<uv*>(p) + i);
  } else __builtin_memcpy(p, v, N * sizeof(T));
}
// A run of n <= 8 elements in slots: all 8, or pieces of 4 (slots 0 .. 3), 2 (slots 4, 5) and 1 (slot 6) one behind the other
__device__ inline int slot_off(int n, int j) { return n == 8 || j < 4 ? j : j < 6 ? (n & 4) + j - 4 : n & 6; }
__device__ inline bool slot_on(int n, int j) { return n == 8 || (j < 4 ? (n & 4) != 0 : j < 6 ? (n & 2) != 0 : j < 7 && (n & 1) != 0); }
struct Token {
  int b, t;
  bool live;        // a token of its sequence (not padding behind its last one)
  int place;        // in its sequence
  int page, row;    // where it goes; page -1: nowhere
};
__device__ inline Token token_of(const RotArgs& a, int b, int t) {
  Token k;
  k.b = b;
  k.t = t;
  k.live = true;
  k.page = -1;
  k.row = 0;
  k.place = t;
  if (a.table != nullptr) {
    const int n_new = a.n_new != nullptr ? dlt_imax(0, dlt_imin(a.n_new[b], a.T)) : a.T;
    k.live = t < n_new;
    const int64_t at = (int64_t)a.seq[b] - n_new + t;
    k.place = (int)(at < -1 ? -1 : at);
    if (k.live && at >= 0 && at < (int64_t)a.cols * a.page) {
      const unsigned col = (unsigned)at / (unsigned)a.page;   // cols * page < 2^31
      const int page = a.table[b * a.tbs + col];
      if (page >= 0 && page < a.n_pages) k.page = page;
      k.row = (int)((unsigned)at - col * (unsigned)a.page);
    }
  }
  return k;
}
struct RotPart {
  int pair, n;     // pairs [pair, pair + n) of all (in the blocks layout on one axis); pair -1: n dims that are not rotated
  int d0, d1;      // first of the first dims and of the second ones (-1: none)
};
// halves: runs of 8 pairs, of any axes (first dims then start at multiples of 8, and at most one part is short); blocks: runs of 8 pairs of an axis
__device__ inline RotPart part_of(const RopeAxes& r, int C, int part) {
  RotPart x;
  if (r.halves) {
    const int k = (r.pairs + 7) >> 3;
    if (part < k) {
      x.pair = x.d0 = 8 * part;
      x.n = dlt_imin(8, r.pairs - x.pair);
      x.d1 = x.d0 + r.pairs;
      return x;
    }
    part -= k;
  } else {
    int off = 0;
#pragma unroll
    for (int a = 0; a < DLT_ROPE_AXES_MAX; a++) {
      if (a >= r.n) break;
      const int R = r.end[a] - off, k = (R + 7) >> 3;
      if (part < k) {
        x.pair = off + 8 * part;
        x.n = dlt_imin(8, R - 8 * part);
        x.d0 = off + x.pair;
        x.d1 = x.d0 + R;
        return x;
      }
      part -= k;
      off = r.end[a];
    }
  }
  x.pair = -1;
  x.d0 = 2 * r.pairs + 8 * part;
  x.n = dlt_imin(8, C - x.d0);
  x.d1 = -1;
  return x;
}
DLT_HD int parts_of(const RopeAxes& r, int C) {
  int n = (C - 2 * r.pairs + 7) >> 3, off = 0;
  if (r.halves) return n + ((r.pairs + 7) >> 3);
  for (int a = 0; a < r.n; a++) { n += (r.end[a] - off + 7) >> 3; off = r.end[a]; }
  return n;
}

// (cos, sin) of a part's pairs, by slots; bit j of the result: slot j is rotated
__device__ inline unsigned cos_sin(const RopeAxes& r, const Token& k, const RotPart& x, float (&c)[8], float (&s)[8]) {
  const TableRows t = table_rows(r, k.b, k.t, k.place, k.live);
  if (t.on == 0) return 0;
  float2 v[8];
  unsigned turn = 0;
  int off, R;
  rope_axes_axis(r, x.pair, off, R);
  if (x.n == 8 && x.pair + 8 <= off + R) {   // all of one axis
    bool on;
    const float* row = pair_row(r, t, x.pair, on);
    turn = on ? 0xff : 0;
    __builtin_memcpy(v, row, sizeof(v));
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      bool on;
      const bool there = slot_on(x.n, j);
      v[j] = *reinterpret_cast<const float2*>(pair_row(r, t, x.pair + (there ? slot_off(x.n, j) : 0), on));
      turn |= (on && there ? 1u : 0u) << j;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; j++) {
    c[j] = v[j].x;
    s[j] = r.inverse ? -v[j].y : v[j].y;
  }
  return turn;
}
template <typename T>
__device__ inline T* dst_of(const RotArgs& a, const RotStream& s, const Token& k, int h) {
  T* d = reinterpret_cast<T*>(s.dst);
  if (!s.paged) return d + (k.b * s.ds[0] + h * s.ds[1] + k.t * s.ds[2]);
  return d + (k.page * s.ds[0] + h * s.ds[1] + k.row * s.ds[2]);
}

// the heads of a stream that lie in [h0, h1) of all heads
__device__ inline void heads_of(const RotStream& s, int& base, int h0, int h1, int& lo, int& hi) {
  lo = dlt_imax(h0 - base, 0);
  hi = dlt_imin(h1 - base, s.H);
  base += s.H;
}

// `room`: elements of the row from p on.  Where they are 8 or more a short part is read with what lies behind it, whose slots are then moved up.
template <typename T>
__device__ inline void load_part(Vec8<T>& v, const T* p, int n, int room) {
  if (n == 8) load_run<8>(v.v, p);
  else if (room >= 8) {
    Vec8<T> x;
    load_run<8>(x.v, p);
#pragma unroll
    for (int j = 0; j < 8; j++) v.v[j] = x.v[j];
    if (!(n & 4)) {   // runs of 1 to 3
      v.v[4] = x.v[0]; v.v[5] = x.v[1];
      v.v[6] = n & 2 ? x.v[2] : x.v[0];
    } else v.v[6] = n & 2 ? x.v[6] : x.v[4];
  } else {
    if (n & 4) load_run<4>(v.v, p);
    if (n & 2) load_run<2>(v.v + 4, p + (n & 4));
    if (n & 1) v.v[6] = p[n & 6];
  }
}
template <typename T>
__device__ inline void store_part(T* p, const Vec8<T>& v, int n) {
  if (n == 8) store_run<8>(p, v.v);
  else {
    if (n & 4) store_run<4>(p, v.v);
    if (n & 2) store_run<2>(p + (n & 4), v.v + 4);
    if (n & 1) p[n & 6] = v.v[6];
  }
}

// heads in flight
constexpr int UNR = 4;
// A large call aims for two workgroups a CU, since a thread that walks more heads fetches its cos and sin less often (us on 256 CUs, by 512 / 2048 / 256
// workgroups: prompts of 7 sequences of 2047 tokens, 16 + 8 + 8 heads, d = 64, 20.4 / 24.0 / 19.5; 6 of 1500, 32 + 8 + 8, d = 128, 41 / 46 / 45; 2 x 8192
// tokens, 16 + 16, d = 64, 29 / 32 / 28; 4096 tokens, 16 + 4, d = 128, 8.8 / 8.7 / 9.3)
constexpr int ROT_BLOCKS_CU = 2;

// WHOLE: every part has 8 dims or pairs (the others cost branches in front of every access)
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void rotate_rows_kernel(RotArgs a, int parts) {
  dlt_kernargs_in<sizeof(RotArgs)>();
  const int C = a.s[0].C;
  const uint64_t first = (uint64_t)blockIdx.x * 256 / (unsigned)parts;   // the workgroup's first token
  const unsigned rest = (unsigned)((uint64_t)blockIdx.x * 256 - first * parts) + threadIdx.x;
  const unsigned ti = (unsigned)first + rest / (unsigned)parts;
  const int part = (int)(rest % (unsigned)parts);
  if (ti >= (unsigned)(a.B * a.T)) return;   // B T < 2^31
  const int b = (int)(ti / (unsigned)a.T), t = (int)(ti - (unsigned)b * (unsigned)a.T);
  RotPart x = part_of(a.r, C, part);
  if constexpr (WHOLE) x.n = 8;

  Vec8<T> v[UNR], w[UNR];
  // elements of heads h .. h + UNR - 1 (the last one again behind it) of a rotated stream
  auto fetch = [&](const RotStream& st, int h, int hi) __attribute__((always_inline)) {
    const T* src = reinterpret_cast<const T*>(st.src) + (b * st.ss[0] + t * st.ss[2]);
#pragma unroll
    for (int u = 0; u < UNR; u++) {
      const T* p = src + dlt_imin(h + u, hi - 1) * st.ss[1];
      load_part(v[u], p + x.d0, x.n, C - x.d0);
      if (x.d1 >= 0) load_part(w[u], p + x.d1, x.n, C - x.d1);
    }
  };
  const int h0 = blockIdx.y * a.hb, h1 = dlt_imin(h0 + a.hb, a.heads);
  int lo, hi, base = 0;
  heads_of(a.s[0], base, h0, h1, lo, hi);
  const bool early = lo < hi && a.s[0].rot;
  if (early) fetch(a.s[0], lo, hi);

  const Token k = token_of(a, b, t);
  float c[8], s[8];
  const unsigned turn = x.pair >= 0 ? cos_sin(a.r, k, x, c, s) : 0u;
  base = 0;
#pragma unroll 1
  for (int z = 0; z < a.n; z++) {
    const RotStream& st = a.s[z];
    heads_of(st, base, h0, h1, lo, hi);
    if (lo >= hi || (st.paged && k.page < 0)) continue;
    T* dst = dst_of<T>(a, st, k, 0);
    if (st.rot == 0) {
      const T* src = reinterpret_cast<const T*>(st.src) + (b * st.ss[0] + t * st.ss[2]);
      for (int d = 8 * part; d < st.C; d += 8 * parts)
        for (int h = lo; h < hi; h += UNR) {
          const int n = WHOLE ? 8 : dlt_imin(8, st.C - d);
#pragma unroll
          for (int u = 0; u < UNR; u++) load_part(v[u], src + dlt_imin(h + u, hi - 1) * st.ss[1] + d, n, st.C - d);
#pragma unroll
          for (int u = 0; u < UNR; u++)
            if (h + u < hi) store_part(dst + (h + u) * st.ds[1] + d, v[u], n);
        }
      continue;
    }
    if (turn == 0 && !st.paged && st.dst == st.src) continue;   // in place: what is not rotated stays
    for (int h = lo; h < hi; h += UNR) {
      if (!(early && z == 0 && h == lo)) fetch(st, h, hi);
#pragma unroll
      for (int u = 0; u < UNR; u++) {
        if (h + u >= hi) continue;
        T* p = dst + (h + u) * st.ds[1];
        if (turn == 0xff) {
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float x0 = (float)v[u].v[j], x1 = (float)w[u].v[j];
            v[u].v[j] = (T)mix(x0, c[j], x1, -s[j]);
            w[u].v[j] = (T)mix(x1, c[j], x0, s[j]);
          }
        } else if (turn != 0) {
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float x0 = (float)v[u].v[j], x1 = (float)w[u].v[j];
            v[u].v[j] = turn >> j & 1 ? (T)mix(x0, c[j], x1, -s[j]) : v[u].v[j];
            w[u].v[j] = turn >> j & 1 ? (T)mix(x1, c[j], x0, s[j]) : w[u].v[j];
          }
        }
        store_part(p + x.d0, v[u], x.n);
        if (x.d1 >= 0) store_part(p + x.d1, w[u], x.n);
      }
    }
  }
}

// The same with 8 dims of whole, 16-byte aligned rows to a lane; partners, at any distance, come through the row in LDS, which belongs to the wave.  For
// sections whose parts would be short or whose second dims start between 16-byte pieces (2 x 10 heads of 7755
// tokens, d = 64, sections of 6, 11 and 11 pairs, fp16: 32 -> 11 us).
template <typename T>
__global__ __launch_bounds__(256) void rotate_rows_lds_kernel(RotArgs a, int parts) {
  dlt_kernargs_in<sizeof(RotArgs)>();
  __shared__ __align__(16) T sm[4][UNR][64 * 8];
  const int P = a.r.pairs;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tpw = 64 / parts, in = lane / parts;   // tokens of a wave, the lane's one
  const unsigned ti = (blockIdx.x * 4 + wave) * tpw + in;
  if (in >= tpw || ti >= (unsigned)(a.B * a.T)) return;   // rows do not span waves: nobody waits for these lanes
  const int b = (int)(ti / (unsigned)a.T), t = (int)(ti - (unsigned)b * (unsigned)a.T);
  const int d0 = 8 * (lane - in * parts);

  Vec8<T> v[UNR];
  auto fetch = [&](const RotStream& st, int h, int hi) __attribute__((always_inline)) {
    const T* src = reinterpret_cast<const T*>(st.src) + (b * st.ss[0] + t * st.ss[2] + d0);
#pragma unroll
    for (int u = 0; u < UNR; u++) v[u] = *reinterpret_cast<const Vec8<T>*>(src + dlt_imin(h + u, hi - 1) * st.ss[1]);
  };
  const int h0 = blockIdx.y * a.hb, h1 = dlt_imin(h0 + a.hb, a.heads);
  int lo, hi, base = 0;
  heads_of(a.s[0], base, h0, h1, lo, hi);
  const bool early = lo < hi && a.s[0].rot;
  if (early) fetch(a.s[0], lo, hi);

  const Token k = token_of(a, b, t);
  const TableRows rows = table_rows(a.r, k.b, k.t, k.place, k.live);
  float c[8], s[8];
  int other[8];
  unsigned turn = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int d = d0 + j;
    int pair = 0;
    bool first = true;
    other[j] = d;
    if (d < 2 * P) {
      int off, R;
      if (a.r.halves) {
        first = d < P;
        pair = first ? d : d - P;
        R = P;
      } else {
        rope_axes_axis(a.r, d >> 1, off, R);   // 2 off <= d < 2 (off + R)
        first = d < 2 * off + R;
        pair = d - off - (first ? 0 : R);
      }
      other[j] = first ? d + R : d - R;
    }
    bool on;
    const float2 cs = *reinterpret_cast<const float2*>(pair_row(a.r, rows, pair, on));
    c[j] = cs.x;
    s[j] = first != (a.r.inverse != 0) ? -cs.y : cs.y;
    turn |= (on && d < 2 * P ? 1u : 0u) << j;
  }
  base = 0;
#pragma unroll 1
  for (int z = 0; z < a.n; z++) {
    const RotStream& st = a.s[z];
    heads_of(st, base, h0, h1, lo, hi);
    if (lo >= hi || (st.paged && k.page < 0)) continue;
    T* dst = dst_of<T>(a, st, k, 0);
    if (st.rot == 0) {
      const T* src = reinterpret_cast<const T*>(st.src) + (b * st.ss[0] + t * st.ss[2]);
      for (int d = d0; d < st.C; d += 8 * parts)
        for (int h = lo; h < hi; h += UNR) {
#pragma unroll
          for (int u = 0; u < UNR; u++) v[u] = *reinterpret_cast<const Vec8<T>*>(src + dlt_imin(h + u, hi - 1) * st.ss[1] + d);
#pragma unroll
          for (int u = 0; u < UNR; u++)
            if (h + u < hi) store_run<8>(dst + (h + u) * st.ds[1] + d, v[u].v);
        }
      continue;
    }
    for (int h = lo; h < hi; h += UNR) {
      if (!(early && z == 0 && h == lo)) fetch(st, h, hi);
      // rows of this wave alone, written and read in order
#pragma unroll
      for (int u = 0; u < UNR; u++) *reinterpret_cast<Vec8<T>*>(&sm[wave][u][8 * lane]) = v[u];
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int u = 0; u < UNR; u++) {
        const T* row = &sm[wave][u][8 * in * parts];
        T w[8];
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = row[other[j]];
#pragma unroll
        for (int j = 0; j < 8; j++) v[u].v[j] = turn >> j & 1 ? (T)mix((float)v[u].v[j], c[j], (float)w[j], s[j]) : v[u].v[j];
        if (h + u < hi) store_run<8>(dst + (h + u) * st.ds[1] + d0, v[u].v);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  }
}

// any strides, one thread per (token, pair or dim that is not rotated)
template <typename T>
__global__ __launch_bounds__(256) void rotate_single_kernel(RotArgs a) {
  dlt_kernargs_in<sizeof(RotArgs)>();
  const int P = a.r.pairs;
  int dims = P;
  for (int z = 0; z < a.n; z++) dims = dlt_imax(dims, a.s[z].rot ? a.s[z].C - P : a.s[z].C);
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t ti = gid / dims;
  if (ti >= (int64_t)a.B * a.T) return;
  const int i = (int)(gid - ti * dims);
  const int b = (int)(ti / a.T), t = (int)(ti - (int64_t)b * a.T);
  const Token k = token_of(a, b, t);
  float c = 1.f, s = 0.f;
  bool turn = false;
  int d0 = 0, d1 = 0;
  if (i < P) {
    int off, R;
    rope_axes_axis(a.r, i, off, R);
    const float* row = pair_row(a.r, table_rows(a.r, k.b, k.t, k.place, k.live), i, turn);
    c = row[0];
    s = a.r.inverse ? -row[1] : row[1];
    d0 = a.r.halves ? i : i + off;
    d1 = d0 + (a.r.halves ? P : R);
  }
  const int h0 = blockIdx.y * a.hb, h1 = dlt_imin(h0 + a.hb, a.heads);
  int base = 0;
#pragma unroll 1
  for (int z = 0; z < a.n; z++) {
    const RotStream& st = a.s[z];
    int lo, hi;
    heads_of(st, base, h0, h1, lo, hi);
    if (st.paged && k.page < 0) continue;
    for (int h = lo; h < hi; h++) {
      const T* src = reinterpret_cast<const T*>(st.src) + (k.b * st.ss[0] + h * st.ss[1] + k.t * st.ss[2]);
      T* dst = dst_of<T>(a, st, k, h);
      if (!st.rot || i >= P) {
        const int d = st.rot ? i + P : i;
        if (d < st.C) dst[d * st.ds[3]] = src[d * st.ss[3]];
        continue;
      }
      const T x0 = src[d0 * st.ss[3]], x1 = src[d1 * st.ss[3]];
      dst[d0 * st.ds[3]] = turn ? (T)mix((float)x0, c, (float)x1, -s) : x0;
      dst[d1 * st.ds[3]] = turn ? (T)mix((float)x1, c, (float)x0, s) : x1;
    }
  }
}

template <typename T>
int launch(RotArgs& a, bool vec, bool vec16, const char* who, hipStream_t stream) {
  const RopeAxes& r = a.r;
  const int C = a.s[0].C;
  const int64_t tokens = (int64_t)a.B * a.T;
  if (tokens > 0x7fffffff) return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: too many tokens (%lld)", who, (long long)tokens);
  // whole rows through LDS where a part's runs would not be aligned 16-byte pieces
  bool pieces = r.halves ? r.pairs % 8 == 0 : true;
  if (!r.halves)
    for (int i = 0; i < r.n; i++) pieces = pieces && r.end[i] % 8 == 0;
  bool whole = pieces && (C - 2 * r.pairs) % 8 == 0;
  for (int z = 0; z < a.n; z++) whole = whole && a.s[z].C % 8 == 0;
  const bool rows = vec16 && !pieces && C <= 512;
  const int parts = rows ? C / 8 : parts_of(r, C);
  int dims = r.pairs;
  for (int z = 0; z < a.n; z++) dims = dlt_imax(dims, a.s[z].rot ? a.s[z].C - r.pairs : a.s[z].C);
  const int64_t gx = rows ? (tokens + 4 * (64 / parts) - 1) / (4 * (64 / parts)) : (tokens * (vec ? parts : dims) + 255) / 256;
  if (gx > 0x7fffffff) return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: too much work for one launch (%lld tokens)", who, (long long)tokens);
  // heads of a thread: all of them while that leaves ROT_BLOCKS_CU workgroups a CU, else fewer, in groups as they are in flight together, and fewer than those
  // while CUs are idle
  const int64_t cus = dlt_device_cus();
  a.hb = (a.heads + UNR - 1) / UNR * UNR;
  while (a.hb > UNR && gx * ((a.heads + a.hb - 1) / a.hb) < ROT_BLOCKS_CU * cus) a.hb = (a.hb / 2 + UNR - 1) / UNR * UNR;
  while (a.hb > 1 && gx * ((a.heads + a.hb - 1) / a.hb) < cus) a.hb = (a.hb + 1) / 2;
  if ((a.heads + a.hb - 1) / a.hb > 65535) a.hb = (a.heads + 65534) / 65535;
  const dim3 grid((unsigned)gx, (unsigned)((a.heads + a.hb - 1) / a.hb)), block(256);
  dlt_timing_before(DLT_K_ROPE, stream);
  if (rows) hipLaunchKernelGGL(rotate_rows_lds_kernel<T>, grid, block, 0, stream, a, parts);
  else if (vec && whole) hipLaunchKernelGGL((rotate_rows_kernel<T, true>), grid, block, 0, stream, a, parts);
  else if (vec) hipLaunchKernelGGL((rotate_rows_kernel<T, false>), grid, block, 0, stream, a, parts);
  else hipLaunchKernelGGL(rotate_single_kernel<T>, grid, block, 0, stream, a);
  dlt_timing_after(stream);
  DLT_CHECK_LAUNCH(who);
  return DLT_OK;
}

}  // namespace

int dlt_rotate_rows(RotArgs& a, int dtype, const char* who, hipStream_t stream) {
  a.heads = 0;
  const int es = dlt_elem_size(dtype);
  bool vec = true, vec16 = true;
  for (int z = 0; z < a.n; z++) {
    const RotStream& s = a.s[z];
    a.heads += s.H;
    vec = vec && s.ss[3] == 1 && s.ds[3] == 1;
    vec16 = vec16 && s.C % 8 == 0 && (uintptr_t)s.src % 16 == 0 && (uintptr_t)s.dst % 16 == 0;
    for (int i = 0; i < 3; i++) vec16 = vec16 && s.ss[i] * es % 16 == 0 && s.ds[i] * es % 16 == 0;
  }
  if ((int64_t)a.B * a.T == 0 || a.heads == 0) return DLT_OK;
  vec16 = vec16 && vec;
  switch (dtype) {
    case DLT_BF16: return launch<bf16_t>(a, vec, vec16, who, stream);
    case DLT_FP16: return launch<f16_t>(a, vec, vec16, who, stream);
    default: return launch<float>(a, vec, vec16, who, stream);
  }
}

int dlt_rope_axes_make(const dlt_rope_axes_t* d, int64_t n_dim, bool need_pos, int inverse, const char* who, RopeAxes& r) {
  r = RopeAxes{};
  if (d == nullptr) return DLT_OK;
  DLT_REQUIRE(d->n_axes >= 1 && d->n_axes <= DLT_ROPE_AXES_MAX, "%s: %d axes, expected 1 to %d", who, d->n_axes, DLT_ROPE_AXES_MAX);
  DLT_REQUIRE(d->layout == DLT_ROPE_BLOCKS || d->layout == DLT_ROPE_HALVES, "%s: bad layout %d", who, d->layout);
  DLT_REQUIRE(d->pos != nullptr || !need_pos, "%s: pos is NULL", who);
  r.n = d->n_axes;
  r.halves = d->layout == DLT_ROPE_HALVES;
  r.inverse = inverse ? 1 : 0;
  r.pos = d->pos;
  r.pa = d->pos_strides[0]; r.pb = d->pos_strides[1]; r.pn = d->pos_strides[2];
  int64_t pairs = 0;
  for (int i = 0; i < r.n; i++) {
    DLT_REQUIRE(d->n_rdim[i] >= 0, "%s: axis %d turns %d pairs", who, i, d->n_rdim[i]);
    if (d->n_rdim[i] > 0) {
      DLT_REQUIRE(d->table[i] != nullptr && d->len[i] > 0, "%s: cos/sin table of axis %d is empty", who, i);
      DLT_REQUIRE(d->table_stride0[i] >= 2 * d->n_rdim[i] && d->table_stride0[i] % 2 == 0 && (uintptr_t)d->table[i] % 8 == 0,
                  "%s: rows of the table of axis %d must hold its pairs and start at multiples of 8 bytes", who, i);
    }
    pairs += d->n_rdim[i];
    DLT_REQUIRE(2 * pairs <= n_dim, "%s: the axes turn %lld pairs, more than half of %lld dims", who, (long long)pairs, (long long)n_dim);
    r.tab[i] = d->table[i];
    r.ts[i] = d->table_stride0[i];
    r.len[i] = d->len[i];
    r.end[i] = (int32_t)pairs;
  }
  r.pairs = (int32_t)pairs;
  return DLT_OK;
}

// q and k (or one tensor) of one call, in place (dst == src) or out of place
extern "C" int dlt_rope_axes(const void* q, const int64_t q_strides[4], void* q_out, const int64_t q_out_strides[4], int32_t Hq,
                             const void* k, const int64_t k_strides[4], void* k_out, const int64_t k_out_strides[4], int32_t Hk,
                             int32_t B, int64_t n_tokens, int64_t n_dim, const dlt_rope_axes_t* rope, int inverse, int dtype, void* stream) {
  DLT_REQUIRE(dtype == DLT_BF16 || dtype == DLT_FP16 || dtype == DLT_FP32, "rope_axes: bad dtype %d", dtype);
  DLT_REQUIRE(B >= 0 && Hq >= 0 && Hk >= 0 && n_tokens >= 0 && n_dim > 0 && n_tokens <= 0x7fffffff && n_dim <= 0x7fffffff && (int64_t)B * Hq <= 0x7fffffff &&
                  (int64_t)B * Hk <= 0x7fffffff && (int64_t)Hq + Hk <= 0x7fffffff, "rope_axes: bad shape");
  DLT_REQUIRE(rope != nullptr, "rope_axes: descriptor is NULL");
  RotArgs a{};
  int rc = dlt_rope_axes_make(rope, n_dim, true, inverse, "rope_axes", a.r);
  if (rc != DLT_OK) return rc;
  const void* src[2] = {q, k};
  void* dst[2] = {q_out, k_out};
  const int64_t *ss[2] = {q_strides, k_strides}, *ds[2] = {q_out_strides, k_out_strides};
  const int32_t H[2] = {Hq, Hk};
  for (int z = 0; z < 2; z++) {
    if (H[z] == 0 || (int64_t)B * n_tokens == 0) continue;
    DLT_REQUIRE(src[z] != nullptr && dst[z] != nullptr && ss[z] != nullptr && ds[z] != nullptr, "rope_axes: tensor argument %d is NULL", z);
    RotStream& s = a.s[a.n++];
    s.src = src[z]; s.dst = dst[z];
    for (int i = 0; i < 4; i++) { s.ss[i] = ss[z][i]; s.ds[i] = ds[z][i]; }
    DLT_REQUIRE(src[z] != dst[z] || (s.ss[0] == s.ds[0] && s.ss[1] == s.ds[1] && s.ss[2] == s.ds[2] && s.ss[3] == s.ds[3]), "rope_axes: in place with two sets of strides");
    s.H = H[z];
    s.C = (int32_t)n_dim;
    s.rot = 1;
  }
  if (a.n == 0) return DLT_OK;
  a.B = B;
  a.T = (int32_t)n_tokens;
  return dlt_rotate_rows(a, dtype, "rope_axes launch", (hipStream_t)stream);
}
