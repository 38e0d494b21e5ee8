// Rotation by positions with several axes (rope_axes.h), alone or on the way into a cache of pages, for gfx950.
//
// Pure streaming: every element is read once and written once.  A thread owns one (token, part of a row): its 8 (cos, sin) pairs are
// fetched once and stay in registers while it walks the heads of q, k and v, so table traffic is shared by the heads.  What a part is:
//   chunks  8 pairs whose two halves are aligned 8-element chunks (P a multiple of 8 in the halves layout, every R_a in blocks), or 8 dims
//           that are not rotated
//   rows    8 dims; the partners, at any distance, come through a row in LDS that belongs to the wave
//   single  one pair or one dim, any strides
// Rotated values are formed in 32 bits, each product rounded before the sum as in the 2D rotation, and rounded once.
#include "rope_axes.h"

namespace {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
template <typename T> struct alignas(16) Vec8 { T v[8]; };

// y0 = x0 c - x1 s, y1 = x0 s + x1 c
__device__ inline float mix(float x, float c, float other, float s) {
#pragma clang fp contract(off)
  const float a = x * c, b = other * s;
  return a + b;
}

struct Token {
  int b, t;
  bool live;        // a token of its sequence (not padding behind its last one)
  int place;        // in its sequence
  int page, row;    // where it goes; page -1: nowhere
};
__device__ inline Token token_of(const RotArgs& a, unsigned i) {
  Token k;
  k.b = (int)(i / (unsigned)a.T);
  k.t = (int)(i - (unsigned)k.b * (unsigned)a.T);
  k.live = true;
  k.page = -1;
  k.row = 0;
  k.place = k.t;
  if (a.table != nullptr) {
    const int n_new = a.n_new != nullptr ? dlt_imax(0, dlt_imin(a.n_new[k.b], a.T)) : a.T;
    k.live = k.t < n_new;
    const int64_t at = (int64_t)a.seq[k.b] - n_new + k.t;
    k.place = (int)(at < -1 ? -1 : at);
    if (k.live && at >= 0 && at < (int64_t)a.cols * a.page) {
      const unsigned col = (unsigned)at / (unsigned)a.page;   // cols * page < 2^31
      const int page = a.table[k.b * a.tbs + col];
      if (page >= 0 && page < a.n_pages) k.page = page;
      k.row = (int)((unsigned)at - col * (unsigned)a.page);
    }
  }
  return k;
}
// (cos, sin) of a pair; false: not rotated
__device__ inline bool cos_sin(const RopeAxes& r, const Token& k, int pair, float& c, float& s) {
  c = 1.f;
  s = 0.f;
  int off;
  const int ax = rope_axes_axis(r, pair, off);
  const float* tab = r.tab[0];
  int64_t ts = r.ts[0];
  int len = r.len[0];
#pragma unroll
  for (int i = 1; i < DLT_ROPE_AXES_MAX; i++)
    if (i == ax) { tab = r.tab[i]; ts = r.ts[i]; len = r.len[i]; }
  const int p = r.pos != nullptr ? r.pos[ax * r.pa + k.b * r.pb + k.t * r.pn] : k.place;
  if (!k.live || p < 0) return false;
  const float2 v = *reinterpret_cast<const float2*>(tab + dlt_imin(p, len - 1) * ts + 2 * (pair - off));
  c = v.x;
  s = r.inverse ? -v.y : v.y;
  return true;
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

// ROWS false: parts are chunks.  UNR heads in flight.
template <typename T, bool ROWS>
__global__ __launch_bounds__(256) void rotate_rows_kernel(RotArgs a) {
  constexpr int UNR = 4;
  const int C = a.s[0].C, P = a.r.pairs;
  const int parts = ROWS ? C / 8 : P / 8 + (C - 2 * P) / 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // whole tokens per wave where rows go through LDS, any number per workgroup otherwise
  const int tpw = 64 / parts;
  unsigned ti;
  int part;
  if (ROWS) {
    ti = (blockIdx.x * 4 + wave) * tpw + lane / parts;
    part = lane - lane / parts * parts;
    if (lane >= tpw * parts) return;
  } else {
    const uint64_t first = (uint64_t)blockIdx.x * 256 / (unsigned)parts;   // the workgroup's first token
    const unsigned rest = (unsigned)((uint64_t)blockIdx.x * 256 - first * parts) + threadIdx.x;
    ti = (unsigned)first + rest / (unsigned)parts;
    part = (int)(rest % (unsigned)parts);
  }
  if (ti >= (unsigned)(a.B * a.T)) return;   // B T < 2^31
  const Token k = token_of(a, ti);
  __shared__ T rows[ROWS ? 4 * 64 * 8 : 1];
  T* own_row = rows + (wave * 64 + lane / parts * parts) * 8;

  float c[8], s[8];
  unsigned turn = 0;   // bit j: element j is rotated
  int d0, d1 = -1, other[8];
  if (ROWS) {
    d0 = 8 * part;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      c[j] = 1.f; s[j] = 0.f;
      other[j] = d0 + j;
      if (d0 + j < 2 * P) {
        bool first;
        const int pair = rope_axes_pair(a.r, d0 + j, first, other[j]);
        if (cos_sin(a.r, k, pair, c[j], s[j])) turn |= 1u << j;
        if (first) s[j] = -s[j];
      }
    }
  } else if (part < P / 8) {
    bool first;
    d0 = 8 * part;
    if (!a.r.halves) {   // the part-th chunk of first dims
      int off;
      rope_axes_axis(a.r, 8 * part, off);
      d0 += off;
    }
    rope_axes_pair(a.r, d0, first, d1);
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (cos_sin(a.r, k, 8 * part + j, c[j], s[j])) turn |= 1u << j;
  } else {
    d0 = 2 * P + 8 * (part - P / 8);
  }

  const int h0 = blockIdx.y * a.hb, h1 = dlt_imin(h0 + a.hb, a.heads);
  int base = 0;
#pragma unroll 1
  for (int z = 0; z < a.n; z++) {
    const RotStream& st = a.s[z];
    int lo, hi;
    heads_of(st, base, h0, h1, lo, hi);
    if (lo >= hi || (st.paged && k.page < 0)) continue;
    const T* src = reinterpret_cast<const T*>(st.src) + (k.b * st.ss[0] + k.t * st.ss[2]);
    T* dst = dst_of<T>(a, st, k, 0);
    if (st.rot == 0) {
      for (int x = 8 * part; x < st.C; x += 8 * parts)
        for (int h = lo; h < hi; h += UNR) {
          Vec8<T> v[UNR];
#pragma unroll
          for (int u = 0; u < UNR; u++) v[u] = *reinterpret_cast<const Vec8<T>*>(src + dlt_imin(h + u, hi - 1) * st.ss[1] + x);
#pragma unroll
          for (int u = 0; u < UNR; u++)
            if (h + u < hi) *reinterpret_cast<Vec8<T>*>(dst + (h + u) * st.ds[1] + x) = v[u];
        }
      continue;
    }
    if (!ROWS && d1 < 0 && dst == src) continue;   // in place: dims that are not rotated stay
    for (int h = lo; h < hi; h += UNR) {
      Vec8<T> v[UNR], w[UNR];
#pragma unroll
      for (int u = 0; u < UNR; u++) {
        const T* p = src + dlt_imin(h + u, hi - 1) * st.ss[1];
        v[u] = *reinterpret_cast<const Vec8<T>*>(p + d0);
        if (!ROWS && d1 >= 0) w[u] = *reinterpret_cast<const Vec8<T>*>(p + d1);
      }
#pragma unroll
      for (int u = 0; u < UNR; u++) {
        if (ROWS) {
          // the row in LDS is read and written by this wave alone, in order
          *reinterpret_cast<Vec8<T>*>(own_row + d0) = v[u];
          __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
          __builtin_amdgcn_wave_barrier();
          __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
          for (int j = 0; j < 8; j++) w[u].v[j] = own_row[other[j]];
          __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
          __builtin_amdgcn_wave_barrier();
          __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
        if (h + u >= hi) continue;
        T* p = dst + (h + u) * st.ds[1];
        if (ROWS) {
#pragma unroll
          for (int j = 0; j < 8; j++)
            if (turn >> j & 1) v[u].v[j] = (T)mix((float)v[u].v[j], c[j], (float)w[u].v[j], s[j]);
          *reinterpret_cast<Vec8<T>*>(p + d0) = v[u];
        } else if (d1 >= 0) {
          Vec8<T> y, z2;
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float x0 = (float)v[u].v[j], x1 = (float)w[u].v[j];
            y.v[j] = turn >> j & 1 ? (T)mix(x0, c[j], x1, -s[j]) : v[u].v[j];
            z2.v[j] = turn >> j & 1 ? (T)mix(x1, c[j], x0, s[j]) : w[u].v[j];
          }
          *reinterpret_cast<Vec8<T>*>(p + d0) = y;
          *reinterpret_cast<Vec8<T>*>(p + d1) = z2;
        } else {
          *reinterpret_cast<Vec8<T>*>(p + d0) = v[u];
        }
      }
    }
  }
}

// any strides, one thread per (token, pair or dim that is not rotated)
template <typename T>
__global__ __launch_bounds__(256) void rotate_single_kernel(RotArgs a) {
  const int P = a.r.pairs;
  int dims = P;
  for (int z = 0; z < a.n; z++) dims = dlt_imax(dims, a.s[z].rot ? a.s[z].C - P : a.s[z].C);
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t ti = gid / dims;
  if (ti >= (int64_t)a.B * a.T) return;
  const int i = (int)(gid - ti * dims);
  const Token k = token_of(a, (unsigned)ti);
  float c = 1.f, s = 0.f;
  const bool turn = i < P && cos_sin(a.r, k, i, c, s);
  int d0 = 0, d1 = 0;
  if (i < P) {
    int off;
    bool first;
    rope_axes_axis(a.r, i, off);
    d0 = a.r.halves ? i : i + off;
    rope_axes_pair(a.r, d0, first, d1);
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
int launch(RotArgs& a, bool vec, const char* who, hipStream_t stream) {
  const RopeAxes& r = a.r;
  const int C = a.s[0].C;
  bool chunks = r.pairs % 8 == 0;
  if (!r.halves)
    for (int i = 0; i < r.n; i++) chunks = chunks && r.end[i] % 8 == 0;
  const int64_t tokens = (int64_t)a.B * a.T;
  if (tokens > 0x7fffffff) return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: too many tokens (%lld)", who, (long long)tokens);
  int64_t gx;
  int parts;
  if (vec && chunks) {
    parts = r.pairs / 8 + (C - 2 * r.pairs) / 8;
    gx = (tokens * parts + 255) / 256;
  } else if (vec && C <= 512) {
    parts = C / 8;
    gx = (tokens + 4 * (64 / parts) - 1) / (4 * (64 / parts));
  } else {
    int dims = r.pairs;
    for (int z = 0; z < a.n; z++) dims = dlt_imax(dims, a.s[z].rot ? a.s[z].C - r.pairs : a.s[z].C);
    vec = false;
    gx = (tokens * dims + 255) / 256;
  }
  if (gx > 0x7fffffff) return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: too much work for one launch (%lld tokens)", who, (long long)tokens);
  a.hb = a.heads;
  while (a.hb > 1 && gx * ((a.heads + a.hb - 1) / a.hb) < 1024) a.hb = (a.hb + 1) / 2;
  if ((a.heads + a.hb - 1) / a.hb > 65535) a.hb = (a.heads + 65534) / 65535;
  const dim3 grid((unsigned)gx, (unsigned)((a.heads + a.hb - 1) / a.hb)), block(256);
  dlt_timing_before(DLT_K_ROPE, stream);
  if (vec && chunks) hipLaunchKernelGGL((rotate_rows_kernel<T, false>), grid, block, 0, stream, a);
  else if (vec) hipLaunchKernelGGL((rotate_rows_kernel<T, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL(rotate_single_kernel<T>, grid, block, 0, stream, a);
  dlt_timing_after(stream);
  DLT_CHECK_LAUNCH(who);
  return DLT_OK;
}

}  // namespace

int dlt_rotate_rows(RotArgs& a, int dtype, const char* who, hipStream_t stream) {
  const int es = dlt_elem_size(dtype);
  a.heads = 0;
  bool vec = true;
  for (int z = 0; z < a.n; z++) {
    const RotStream& s = a.s[z];
    a.heads += s.H;
    vec = vec && s.C % 8 == 0 && s.ss[3] == 1 && s.ds[3] == 1 && (uintptr_t)s.src % 16 == 0 && (uintptr_t)s.dst % 16 == 0;
    for (int i = 0; i < 3; i++) vec = vec && s.ss[i] * es % 16 == 0 && s.ds[i] * es % 16 == 0;
  }
  if ((int64_t)a.B * a.T == 0 || a.heads == 0) return DLT_OK;
  switch (dtype) {
    case DLT_BF16: return launch<bf16_t>(a, vec, who, stream);
    case DLT_FP16: return launch<f16_t>(a, vec, who, stream);
    default: return launch<float>(a, vec, who, stream);
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
