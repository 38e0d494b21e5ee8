// New keys and values into a cache of pages held in 8 bits, with a scale for each block of tokens and head, rotated on the way (dlt_paged8_append), for gfx950.
//
// A block's scale is 2^e with the least e at which the largest element of its new tokens fits the format, and no less than the e that older tokens of the block have;
// where those have a smaller one their numbers are rounded to the new scale.  Powers of two make that harmless: numbers of e4m3 keep every bit that is not shifted
// out of its subnormals, whole numbers lose at most half a step of the new scale, less than a step over all growths (1/2 + 1/4 + ..).
//
// An item is a block, a head and a tensor (K or V): its tokens are fetched once, rotated in 32 bits, held in registers until their largest element is known, and written as
// 8-bit numbers, some heads one after the other under one fetch of cos and sin, the next head's rows on their way.  8 dims to a lane, as many rows to a wave as fit.
// Few new tokens a block: a wave to an item (nothing waits for another wave); else four or eight, which exchange their maxima through LDS (blocks of 128, d = 128, by four
// waves with twice the rows in registers: 60 us for 36).  Rows of q are rotated by workgroups of their own in the same launch, a wave to some tokens, the heads one after
// the other under one fetch of cos and sin.
//
// Memory bound: 4 sequences of 1500 tokens, 32 + 8 + 8 heads, d = 128, blocks of 64 30 us, 4.5 TB/s (from fp32 59, 4.4 TB/s); 7 of up to 2047, 16 + 8 + 8, d = 64, blocks of 16 17 to 19 us, 80 MB with
// the rows of q that hold no token.  A token each of 64 sequences: 5 us on the GPU, latency: length, page, row.
#include <algorithm>
#include "attn_common.hpp"
#include "page_cvt8.h"
#include "kernargs.h"
#include "rope_axes.h"

namespace {

struct App8Side {           // keys or values
  const void* src;
  uint8_t *dst, *scale;
  int64_t ss[3], ds[3], es[3];   // batch, head, token; page, head, row; page, head, block of the page
  int32_t D, rot;
};
struct App8Args {
  App8Side s[2];
  const void* q;
  void* q_out;
  int64_t qs[3], qos[3];
  int32_t B, H, Hkv, T;
  int32_t page, n_pages, cols, block;
  int32_t nb;               // blocks that T tokens of a sequence can touch
  int32_t kv_blocks;        // workgroups of keys and values; behind them those of q
  int32_t hk, kv_heads, kv_chunks;   // heads of K or V that an item walks; of K, rounded up to whole runs; runs of K and V
  int32_t hq, q_chunks;     // heads of q that a wave walks, such chunks
  int32_t whole;            // a lane's 8 dims are one run of pairs of one axis
  const int32_t *table, *seq, *n_new;
  int64_t tbs;
  RopeAxes r;
  uint32_t mT, sT, mb, sb, mp, sp, mc, sc, mn, sn;   // divisions by T, block, page, runs of heads, blocks of a sequence
};

// 8 elements as they come
template <typename T>
struct Raw8 { u32x4 w[sizeof(T) / 2]; };
template <typename T>
DLT_DEV void fetch8(Raw8<T>& r, const T* p) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); i++) r.w[i] = *reinterpret_cast<const u32x4*>(p + 8 * i / (sizeof(T) / 2));
}
template <typename T>
DLT_DEV void widen8(float (&f)[8], const Raw8<T>& r) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = __uint_as_float(r.w[i >> 2][i & 3]);
  } else unpack8<T>(r.w[0], f);
}

// A lane's 8 dims d0 .. d0 + 7 of a token: cos, sin (with the sign of their dim's half), where their partners are, which of them turn
struct Turn {
  float c[8], s[8];
  int other;          // whole: first of the partners' 8 dims
  unsigned on;
};
DLT_DEV void half_of(const RopeAxes& r, int d, int& pair, int& other, bool& first) {   // d < 2 P
  const int P = r.pairs;
  int off, R;
  if (r.halves) {
    first = d < P;
    pair = first ? d : d - P;
    R = P;
  } else {
    rope_axes_axis(r, d >> 1, off, R);   // 2 off <= d < 2 (off + R)
    first = d < 2 * off + R;
    pair = d - off - (first ? 0 : R);
  }
  other = first ? d + R : d - R;
}
template <bool WHOLE>
DLT_DEV Turn turn_of(const RopeAxes& r, int d0, int b, int t, int place, bool live) {
  Turn x;
  x.on = 0;
  x.other = d0;
#pragma unroll
  for (int j = 0; j < 8; j++) { x.c[j] = 1.f; x.s[j] = 0.f; }
  if (d0 >= 2 * r.pairs) return x;
  const TableRows rows = table_rows(r, b, t, place, live);
  if constexpr (WHOLE) {
    int pair;
    bool first, on;
    half_of(r, d0, pair, x.other, first);
    float2 v[8];
    __builtin_memcpy(v, pair_row(r, rows, pair, on), sizeof(v));
    x.on = on ? 0xff : 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      x.c[j] = v[j].x;
      x.s[j] = first ? -v[j].y : v[j].y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if (d0 + j >= 2 * r.pairs) continue;
      int pair, other;
      bool first, on;
      half_of(r, d0 + j, pair, other, first);
      const float2 v = *reinterpret_cast<const float2*>(pair_row(r, rows, pair, on));
      x.c[j] = v.x;
      x.s[j] = first ? -v.y : v.y;
      x.on |= (on ? 1u : 0u) << j;
    }
  }
  return x;
}
// A row's 8 dims and their partners
template <typename T, bool WHOLE>
struct Pair8 {
  Raw8<T> own, far;
  DLT_DEV void fetch(const RopeAxes& r, const T* row, int d0, const Turn& x) {
    fetch8(own, row + d0);
    if (x.on == 0) return;
    if constexpr (WHOLE) {
      fetch8(far, row + x.other);
    } else {
      T v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        int pair, other = d0 + j;
        bool first;
        if (d0 + j < 2 * r.pairs) half_of(r, d0 + j, pair, other, first);
        v[j] = row[other];
      }
      __builtin_memcpy(&far, v, sizeof(far));
    }
  }
  DLT_DEV void rotated(float (&y)[8], const Turn& x) const {
    widen8<T>(y, own);
    if (x.on == 0) return;
    float w[8];
    widen8<T>(w, far);
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = x.on >> j & 1 ? mix(y[j], x.c[j], w[j], x.s[j]) : y[j];
  }
};

// Rows of q: tokens of all sequences in a row, `rpw` to a wave, `hq` heads to a wave
template <typename T, bool WHOLE>
DLT_DEV void rotate_q(const App8Args& a, int item, int lane) {
  const int D = a.s[0].D, parts = D >> 3, rpw = 64 / parts;
  const int grp = item / a.q_chunks, h0 = (item - grp * a.q_chunks) * a.hq, h1 = dlt_imin(h0 + a.hq, a.H);
  const int in = lane / parts, d0 = 8 * (lane - in * parts);
  const int64_t ti = (int64_t)grp * rpw + in;
  if (in >= rpw || ti >= (int64_t)a.B * a.T) return;
  const int b = (int)dlt_fastdiv((uint32_t)ti, a.mT, a.sT), t = (int)ti - b * a.T;
  const int n_new = a.n_new != nullptr ? dlt_imax(0, dlt_imin(a.n_new[b], a.T)) : a.T;
  const int64_t at = (int64_t)a.seq[b] - n_new + t;
  Turn x;
  x.on = 0;
  if (a.r.n > 0) x = turn_of<WHOLE>(a.r, d0, b, t, (int)(at < -1 ? -1 : at), t < n_new);
  const T* src = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + t * a.qs[2];
  T* dst = reinterpret_cast<T*>(a.q_out) + b * a.qos[0] + t * a.qos[2] + d0;
  constexpr int UNR = 4;   // heads on their way together
  for (int h = h0; h < h1; h += UNR) {
    Pair8<T, WHOLE> v[UNR];
#pragma unroll
    for (int u = 0; u < UNR; u++) v[u].fetch(a.r, src + dlt_imin(h + u, h1 - 1) * a.qs[1], d0, x);
#pragma unroll
    for (int u = 0; u < UNR; u++) {
      if (h + u >= h1) continue;
      Raw8<T> out = v[u].own;   // as it is, bit for bit, where nothing turns
      if (x.on != 0) {
        float y[8];
        v[u].rotated(y, x);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int i = 0; i < 8; i++) out.w[i >> 2][i & 3] = __float_as_uint(y[i]);
        } else out.w[0] = pack8<T>(y);
      }
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) / 2); i++) __builtin_nontemporal_store(out.w[i], reinterpret_cast<u32x4*>(dst + (h + u) * a.qos[1]) + i);
    }
  }
}

// Waves a CU that the heads an item (or a wave of q) walks have to leave: more heads fetch cos and sin, lengths and pages less often.  us, 4 / 8 / 16 / 32 waves of keys and
// values: 4 sequences of 1500 tokens, 32 + 8 + 8 heads, d = 128, blocks of 64 34.6 / 33.7 / 35.3 / 41.1, of 16 29.4 / 29.5 / 32.5 / 36.2; 7 of up to 2047, 16 + 8 + 8, d = 64,
// blocks of 16 22.4 / 18.3 / 19.6 / 24.0.  4 / 8 / 16 waves of q beside 8 of those: 36.7 / 33.7 / 30.0; 30.5 / 29.5 / 27.5; 18.7 / 18.3 / 17.6.
constexpr int APP8_WAVES = 8, APP8_Q_WAVES = 16;

// NW waves to an item, MAXP rows of registers to a lane
template <typename T, int FMT, bool WHOLE, int NW, int MAXP>
__global__ __launch_bounds__(NW == 8 ? 512 : 256) void paged8_append_kernel(const App8Args a) {
  dlt_kernargs_in<sizeof(App8Args)>();
  __shared__ unsigned big[2][8];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x >= a.kv_blocks) {
    rotate_q<T, WHOLE>(a, ((int)blockIdx.x - a.kv_blocks) * (NW == 8 ? 8 : 4) + wave, lane);
    return;
  }
  // item: runs of `hk` heads of K and V innermost, then blocks, sequences
  const int item = NW > 1 ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave, mine = NW > 1 ? wave : 0;
  const int bj = (int)dlt_fastdiv((uint32_t)item, a.mc, a.sc);
  if (bj >= a.B * a.nb) return;   // (NW = 1: no wave waits for another)
  const int b = (int)dlt_fastdiv((uint32_t)bj, a.mn, a.sn), j = bj - b * a.nb;
  int h = (item - bj * a.kv_chunks) * a.hk;
  const bool vals = h >= a.kv_heads;   // heads of V behind those of K, in chunks of their own
  if (vals) h -= a.kv_heads;
  const int h1 = dlt_imin(h + a.hk, a.Hkv);
  const App8Side& s = a.s[vals ? 1 : 0];
  const bool rot = !vals && a.r.n > 0;

  // new tokens lo .. hi - 1 of the sequence, n0 .. n1 - 1 of them in the block
  const int n_new = a.n_new != nullptr ? dlt_imax(0, dlt_imin(a.n_new[b], a.T)) : a.T;
  const int64_t held = (int64_t)a.seq[b] - n_new;
  const int64_t room = (int64_t)a.cols * a.page;
  const int lo = (int)(held < 0 ? 0 : held < room ? held : room), hi = (int)(held + n_new < 0 ? 0 : held + n_new < room ? held + n_new : room);
  const int blk = (int)dlt_fastdiv((uint32_t)lo, a.mb, a.sb) + j, base = blk * a.block;
  const int n0 = dlt_imax(lo, base), n1 = dlt_imin(hi, base + a.block);
  if (n0 >= n1) return;
  const int col = (int)dlt_fastdiv((uint32_t)base, a.mp, a.sp), row0 = base - col * a.page;
  const int page = a.table[b * a.tbs + col];   // on its way beside the rows

  const int D = s.D, parts = D >> 3, rpw = 64 / parts, in = lane / parts, d0 = 8 * (lane - in * parts);
  const bool lane_on = in < rpw;
  Turn turn[MAXP];   // cos and sin of the lane's rows, for all heads
  auto turn_at = [&](int p) __attribute__((always_inline)) {
    const int tok = n0 + (p * NW + mine) * rpw + in;
    if (rot && lane_on && tok < n1) return turn_of<WHOLE>(a.r, d0, b, (int)(tok - held), tok, true);
    Turn x;
    x.on = 0;
    x.other = d0;
    return x;
  };
#pragma unroll
  for (int p = 0; p < MAXP; p++) turn[p] = turn_at(p);
  Pair8<T, WHOLE> x[MAXP];
  auto fetch = [&](int head) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < MAXP; p++) {
      const int tok = n0 + (p * NW + mine) * rpw + in;
      if (lane_on && tok < n1) x[p].fetch(a.r, reinterpret_cast<const T*>(s.src) + (b * s.ss[0] + head * s.ss[1] + (int)(tok - held) * s.ss[2]), d0, turn[p]);
    }
  };
  fetch(h);
  if (page < 0 || page >= a.n_pages) return;

#pragma unroll 1
  for (int round = 0; h < h1; h++, round ^= 1) {
    uint8_t* dst = s.dst + (page * s.ds[0] + h * s.ds[1] + row0 * s.ds[2]);
    uint8_t* sc = s.scale + (page * s.es[0] + h * s.es[1] + (int)dlt_fastdiv((uint32_t)row0, a.mb, a.sb) * s.es[2]);
    const bool older = base < n0;
    const int e_old = older ? *sc : 0;

    float y[MAXP][8];
    unsigned m = 0, odd_bits = 0;   // of the largest finite magnitude; nonzero: an element that is none
#pragma unroll
    for (int p = 0; p < MAXP; p++) {
      const int tok = n0 + (p * NW + mine) * rpw + in;
#pragma unroll
      for (int i = 0; i < 8; i++) y[p][i] = 0.f;
      if (lane_on && tok < n1) x[p].rotated(y[p], turn[p]);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const unsigned v = __float_as_uint(y[p][i]) & 0x7fffffffu;
        const bool fin = v < 0x7f800000u;
        odd_bits |= fin ? 0u : 1u;
        m = fin && v > m ? v : m;
      }
    }
    if (h + 1 < h1) fetch(h + 1);   // beside what follows
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) {
      const unsigned o = (unsigned)__shfl_xor((int)m, k);
      m = m > o ? m : o;
    }
    bool odd = __builtin_amdgcn_ballot_w64(odd_bits != 0) != 0;
    if constexpr (NW > 1) {
      asm volatile("" ::"v"(e_old));   // read before another wave may write it
      if (lane == 0) big[round][wave] = m | (odd ? 0x80000000u : 0u);
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; w++) {
        const unsigned o = big[round][w];
        odd = odd || (o >> 31) != 0;
        m = m > (o & 0x7fffffffu) ? m : (o & 0x7fffffffu);
      }
    }
    const int need = cvt8_exponent<FMT>(m);          // biased
    const int e = dlt_imax(need, e_old);             // 255, NaN, stays
    const int e_new = FMT == DLT_INT8 && odd ? 255 : e;
    const float inv = cvt8_inverse(e);
    const float most = std::is_same<T, f16_t>::value ? cvt8_most_f16<FMT>(e) : cvt8_most<FMT>();
    // older tokens of the block at a larger scale
    if (older && e > e_old && e_new != 255) {
      keep_branch();
      const float by = e - e_old > 60 ? 0.f : __uint_as_float((unsigned)(127 - (e - e_old)) << 23);
      if (lane_on)
#pragma unroll 4
        for (int r = mine * rpw + in; r < n0 - base; r += NW * rpw) {
          uint8_t* p = dst + r * s.ds[2] + d0;
          float f[8];
          cvt8_get8<FMT>(*reinterpret_cast<const u32x2*>(p), f);
#pragma unroll
          for (int i = 0; i < 8; i++) f[i] *= by;
          *reinterpret_cast<u32x2*>(p) = cvt8_put8<FMT>(f, most);
        }
    }
    if (mine == 0 && lane == 0 && (!older || e_new != e_old)) *sc = (uint8_t)e_new;
#pragma unroll
    for (int p = 0; p < MAXP; p++) {
      const int r = n0 - base + (p * NW + mine) * rpw + in;
      if (lane_on && r < n1 - base) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = y[p][i] * inv;
        *reinterpret_cast<u32x2*>(dst + r * s.ds[2] + d0) = cvt8_put8<FMT>(f, most);
      }
    }
  }
}

template <typename T, int FMT, bool WHOLE>
int launch(const App8Args& a, int nw, int passes, int64_t grid, hipStream_t stream) {
  dlt_timing_before(DLT_K_ROPE, stream);
  const dim3 g((unsigned)grid), t(nw == 8 ? 512 : 256);
  if (nw == 1) hipLaunchKernelGGL((paged8_append_kernel<T, FMT, WHOLE, 1, 2>), g, t, 0, stream, a);
  else if (nw == 4 && passes == 1) hipLaunchKernelGGL((paged8_append_kernel<T, FMT, WHOLE, 4, 1>), g, t, 0, stream, a);
  else if (nw == 4) hipLaunchKernelGGL((paged8_append_kernel<T, FMT, WHOLE, 4, 2>), g, t, 0, stream, a);
  else if (passes <= 2) hipLaunchKernelGGL((paged8_append_kernel<T, FMT, WHOLE, 8, 2>), g, t, 0, stream, a);
  else hipLaunchKernelGGL((paged8_append_kernel<T, FMT, WHOLE, 8, 4>), g, t, 0, stream, a);
  dlt_timing_after(stream);
  DLT_CHECK_LAUNCH("paged8_append launch");
  return DLT_OK;
}
template <typename T>
int launch_t(const App8Args& a, int fmt, int nw, int passes, int64_t grid, hipStream_t stream) {
  if (fmt == DLT_FP8_E4M3) return a.whole ? launch<T, DLT_FP8_E4M3, true>(a, nw, passes, grid, stream) : launch<T, DLT_FP8_E4M3, false>(a, nw, passes, grid, stream);
  return a.whole ? launch<T, DLT_INT8, true>(a, nw, passes, grid, stream) : launch<T, DLT_INT8, false>(a, nw, passes, grid, stream);
}

int check8(const char* who, const char* name, const void* p, const int64_t* st, int es, int align, bool empty) {
  DLT_REQUIRE(st != nullptr && (p != nullptr || empty), "%s: %s is NULL", who, name);
  if (empty) return DLT_OK;
  bool ok = st[3] == 1 && (uintptr_t)p % align == 0;
  for (int i = 0; i < 3; i++) ok = ok && st[i] * es % align == 0;
  DLT_REQUIRE(ok, "%s: rows of %s must be contiguous and start at multiples of %d bytes", who, name, align);
  return DLT_OK;
}

}  // namespace

int dlt_scales8_check(const char* who, const dlt_scales8_t* s, int page) {
  DLT_REQUIRE(s != nullptr, "%s: scales is NULL", who);
  DLT_REQUIRE(s->format == DLT_FP8_E4M3 || s->format == DLT_INT8, "%s: bad format %d", who, s->format);
  DLT_REQUIRE(s->block > 0 && page % s->block == 0, "%s: pages of %d tokens do not hold whole blocks of %d", who, page, s->block);
  if (s->block % 16 != 0 || s->block > DLT_BLOCK8_MAX)
    return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: blocks of %d tokens, expected a multiple of 16 up to %d", who, s->block, DLT_BLOCK8_MAX);
  DLT_REQUIRE(s->k_scale != nullptr && s->v_scale != nullptr, "%s: a tensor of scales is NULL", who);
  for (int i = 0; i < 3; i++) DLT_REQUIRE(s->k_strides[i] >= 0 && s->v_strides[i] >= 0, "%s: negative stride of the scales", who);
  return DLT_OK;
}

extern "C" int dlt_paged8_append(const void* k, const int64_t k_strides[4], const void* v, const int64_t v_strides[4], const void* q, const int64_t q_strides[4],
                                 void* q_out, const int64_t q_out_strides[4], void* k_cache, const int64_t k_cache_strides[4], void* v_cache,
                                 const int64_t v_cache_strides[4], const dlt_scales8_t* scales, const int32_t* table, int64_t table_stride, const int32_t* seq_len,
                                 const int32_t* n_new, const dlt_rope_axes_t* rope, const dlt_paged_shape_t* s, void* stream) {
  const char* who = "paged8_append";
  DLT_REQUIRE(s != nullptr, "%s: shape is NULL", who);
  DLT_REQUIRE(s->dtype == DLT_BF16 || s->dtype == DLT_FP16 || s->dtype == DLT_FP32, "%s: bad dtype %d", who, s->dtype);
  DLT_REQUIRE(s->B > 0 && s->H >= 0 && s->Hkv > 0 && s->T >= 0 && s->dk > 0 && s->dv > 0, "%s: B=%d H=%d Hkv=%d T=%d dk=%d dv=%d", who, s->B, s->H, s->Hkv, s->T, s->dk,
              s->dv);
  DLT_REQUIRE(s->cols > 0 && s->n_pages > 0 && s->page > 0 && (int64_t)s->cols * s->page < 1 << 30, "%s: cols=%d n_pages=%d page=%d", who, s->cols, s->n_pages, s->page);
  DLT_REQUIRE((int64_t)s->H + 2 * (int64_t)s->Hkv <= 0x7fffffff, "%s: too many heads", who);
  if (s->dk > 128 || s->dv > 128 || s->dk % 8 != 0 || s->dv % 8 != 0)
    return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: head dims dk=%d dv=%d must be multiples of 8 up to 128", who, s->dk, s->dv);
  DLT_REQUIRE(table != nullptr && seq_len != nullptr && table_stride >= 0, "%s: table or seq_len is NULL, or the table's stride negative", who);
  int rc = dlt_scales8_check(who, scales, s->page);
  if (rc != DLT_OK) return rc;
  App8Args a{};
  if ((rc = dlt_rope_axes_make(rope, s->dk, false, 0, who, a.r)) != DLT_OK) return rc;
  const bool none = s->T == 0;
  const int es = dlt_elem_size(s->dtype);
  if ((rc = check8(who, "k", k, k_strides, es, 16, none)) != DLT_OK || (rc = check8(who, "v", v, v_strides, es, 16, none)) != DLT_OK) return rc;
  if ((rc = check8(who, "k_cache", k_cache, k_cache_strides, 1, 8, false)) != DLT_OK || (rc = check8(who, "v_cache", v_cache, v_cache_strides, 1, 8, false)) != DLT_OK)
    return rc;
  if (s->H > 0) {
    if ((rc = check8(who, "q", q, q_strides, es, 16, none)) != DLT_OK || (rc = check8(who, "q_out", q_out, q_out_strides, es, 16, none)) != DLT_OK) return rc;
    DLT_REQUIRE(none || q != q_out, "%s: q and q_out must be two buffers", who);
  }
  if (none) return DLT_OK;
  a.s[0].src = k; a.s[1].src = v;
  a.s[0].dst = (uint8_t*)k_cache; a.s[1].dst = (uint8_t*)v_cache;
  a.s[0].scale = (uint8_t*)scales->k_scale; a.s[1].scale = (uint8_t*)scales->v_scale;
  for (int i = 0; i < 3; i++) {
    a.s[0].ss[i] = k_strides[i]; a.s[1].ss[i] = v_strides[i];
    a.s[0].ds[i] = k_cache_strides[i]; a.s[1].ds[i] = v_cache_strides[i];
    a.s[0].es[i] = scales->k_strides[i]; a.s[1].es[i] = scales->v_strides[i];
    if (s->H > 0) { a.qs[i] = q_strides[i]; a.qos[i] = q_out_strides[i]; }
  }
  a.s[0].D = s->dk; a.s[1].D = s->dv;
  a.s[0].rot = 1;
  a.q = q; a.q_out = q_out;
  a.B = s->B; a.H = s->H; a.Hkv = s->Hkv; a.T = s->T;
  a.page = s->page; a.n_pages = s->n_pages; a.cols = s->cols; a.block = scales->block;
  a.table = table; a.seq = seq_len; a.n_new = n_new; a.tbs = table_stride;
  dlt_fastdiv_make((uint32_t)s->T, a.mT, a.sT);
  dlt_fastdiv_make((uint32_t)a.block, a.mb, a.sb);
  dlt_fastdiv_make((uint32_t)a.page, a.mp, a.sp);
  a.whole = 1;
  for (int i = 0; i < a.r.n; i++) a.whole = a.whole && a.r.end[i] % 8 == 0;
  // waves of an item: as many as hold what a block can get in two rounds of their rows (up to four for eight waves: 128 rows of 128 dims)
  const int rows = 64 / (std::max(s->dk, s->dv) / 8), most = std::min(s->T, a.block);
  const int nw = most <= 2 * rows ? 1 : most <= 8 * rows ? 4 : 8, passes = (most + nw * rows - 1) / (nw * rows);
  a.nb = (s->T + a.block - 2) / a.block + 1;
  // heads of an item: all of K's or V's while that leaves APP8_WAVES a CU, fewer otherwise
  const int64_t cus = dlt_device_cus(), blocks = (int64_t)s->B * a.nb;
  a.hk = s->Hkv;
  while (a.hk > 1 && blocks * nw * 2 * ((s->Hkv + a.hk - 1) / a.hk) < APP8_WAVES * cus) a.hk = (a.hk + 1) / 2;
  const int runs = (s->Hkv + a.hk - 1) / a.hk;
  a.kv_heads = runs * a.hk;
  a.kv_chunks = 2 * runs;
  dlt_fastdiv_make((uint32_t)a.kv_chunks, a.mc, a.sc);
  dlt_fastdiv_make((uint32_t)a.nb, a.mn, a.sn);
  const int64_t items = blocks * a.kv_chunks;
  a.kv_blocks = (int32_t)std::min<int64_t>(nw > 1 ? items : (items + 3) / 4, 0x7fffffff);
  int64_t grid = a.kv_blocks;
  if (s->H > 0) {
    const int64_t groups = ((int64_t)s->B * s->T + 64 / (s->dk / 8) - 1) / (64 / (s->dk / 8));
    a.hq = s->H;
    while (a.hq > 1 && groups * ((s->H + a.hq - 1) / a.hq) < APP8_Q_WAVES * cus) a.hq = (a.hq + 1) / 2;
    a.q_chunks = (s->H + a.hq - 1) / a.hq;
    grid += nw == 8 ? (groups * a.q_chunks + 7) / 8 : (groups * a.q_chunks + 3) / 4;
  }
  if (items > 0x7fffff00 || grid > 0x7fffffff || (int64_t)s->B * s->T > 0x7fffffff) return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: too much work for one launch", who);
  switch (s->dtype) {
    case DLT_BF16: return launch_t<bf16_t>(a, scales->format, nw, passes, grid, (hipStream_t)stream);
    case DLT_FP16: return launch_t<f16_t>(a, scales->format, nw, passes, grid, (hipStream_t)stream);
    default: return launch_t<float>(a, scales->format, nw, passes, grid, (hipStream_t)stream);
  }
}
