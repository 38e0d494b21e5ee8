// Entry points of the 1D window attention, the paged cache's attention and append: argument checks, how a call is cut into workgroups, and
// the launches that sum partial results.
#include <cmath>
#include "band_common.h"
#include "band_shapes.h"
#include "rope_axes.h"

namespace {

// ---- sums of shares -------------------------------------------------------------------------------------------------------------
// Forward: partial outputs [bh][share][row][dv] and, behind them, {maximum in log2 units, sum} of each row, joined in the order of the shares.
// WG: a workgroup to a row; every wave forms the weights of all shares (a lane each), adds up every fourth share, and the four sums are added.  Else (up to 8
// shares) a wave to a row.  One thread per 4 dims walking all shares: 36 us for 96 rows of 64 shares, this way 4.8; 8192 rows of 4 shares 14.4 by workgroups,
// 6.2 by waves.
DLT_DEV float band_share_weight(const float2& x, float m) {
  // a share that held no key of the row has (-inf, 0); a sum that is infinite or NaN goes through
  return x.x == -INFINITY ? (x.y == 0.f ? 0.f : 1.f) : fast_exp2(x.x - m);
}
template <typename TIO, bool WG>
__global__ __launch_bounds__(256) void band_join_kernel(const BandArgs a) {
  dlt_kernargs_in<sizeof(BandArgs)>();
  __shared__ float sum[WG ? 4 : 1][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t at = WG ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  if (!WG && at >= (int64_t)a.B * a.Hkv * a.rows) return;
  const int bh = (int)(at / a.rows), r = (int)(at - (int64_t)bh * a.rows), b = bh / a.Hkv, h = bh - b * a.Hkv;
  const int n_q = a.pg.n_new != nullptr ? dlt_imax(0, dlt_imin(a.pg.n_new[b], a.Lq)) : a.Lq;
  const bool on = r < n_q * a.G;   // the others have no partial results
  const float2* ml = reinterpret_cast<const float2*>(a.part + (int64_t)a.B * a.Hkv * a.shares * a.rows * a.dv_) + (int64_t)bh * a.shares * a.rows + r;
  const float* part = a.part + ((int64_t)bh * a.shares * a.rows + r) * a.dv_ + 2 * dlt_imin(lane, a.dv_ / 2 - 1);
  const int64_t step = (int64_t)a.rows * a.dv_;
  float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
  // with a weight of 0 too: an infinite or NaN part holds such a value of a key that the row sees, and 0 times it is NaN
  auto add = [&](const float2& v, float f) __attribute__((always_inline)) {
    o[0] = fmaf(v.x, f, o[0]);
    o[1] = fmaf(v.y, f, o[1]);
  };
  if constexpr (WG) {
    static_assert(BAND_SHARES_MAX == 128, "two weights a lane");
    float2 x[2];
    float wgt[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int s = 64 * i + lane;
      x[i] = on && s < a.shares ? ml[(int64_t)s * a.rows] : float2{-INFINITY, 0.f};
      m = fmaxf(m, x[i].x);
    }
    m = band_wave_max(m);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      wgt[i] = band_share_weight(x[i], m);
      l = fmaf(x[i].y, wgt[i], l);
    }
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) l += __shfl_xor(l, k);
    if (on)
      for (int s0 = wave; s0 < a.shares; s0 += 32) {
        float2 v[8];
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] = *reinterpret_cast<const float2*>(part + dlt_imin(s0 + 4 * u, a.shares - 1) * step);
#pragma unroll
        for (int u = 0; u < 8; u++) {
          const int s = s0 + 4 * u;
          const float f = s < 64 ? band_lane(wgt[0], s) : band_lane(wgt[1], s - 64);
          if (s < a.shares) add(v[u], f);
        }
      }
    sum[wave][2 * lane] = o[0];
    sum[wave][2 * lane + 1] = o[1];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int j = 0; j < 2; j++) o[j] = ((sum[0][2 * lane + j] + sum[1][2 * lane + j]) + sum[2][2 * lane + j]) + sum[3][2 * lane + j];
  } else if (on) {
    float2 x[8], v[8];
#pragma unroll
    for (int s = 0; s < 8; s++) {
      const int c = dlt_imin(s, a.shares - 1);
      x[s] = ml[(int64_t)c * a.rows];
      v[s] = *reinterpret_cast<const float2*>(part + c * step);
    }
#pragma unroll
    for (int s = 0; s < 8; s++) m = fmaxf(m, x[s].x);   // the last share again behind it
#pragma unroll
    for (int s = 0; s < 8; s++) {
      if (s >= a.shares) break;
      const float f = band_share_weight(x[s], m);
      l = fmaf(x[s].y, f, l);
      add(v[s], f);
    }
  }
  const int n_k = a.pg.seq != nullptr ? dlt_imax(0, dlt_imin(a.pg.seq[b], a.Lk)) : a.Lk;
  const float f = on ? band_inverse(l, n_k - n_q + band_row(a, r).tok) : 0.f;
  TIO* p = band_row_ptr(reinterpret_cast<TIO*>(a.out) + b * a.os[0] + (int64_t)h * a.G * a.os[1], a.os, a, r);
  if (2 * lane < a.dv_) *reinterpret_cast<unsigned*>(p + 2 * lane) = pack2<TIO>(o[0] * f, o[1] * f);
  TIO* low = a.low != nullptr ? band_low<TIO>(a, b, h, r) : nullptr;
  if (low != nullptr && 2 * lane < a.dv_) *reinterpret_cast<unsigned*>(low + 2 * lane) = pack2<TIO>(band_dropped<TIO>(o[0] * f), band_dropped<TIO>(o[1] * f));
  if (lane == 0 && a.lse != nullptr) a.lse[at] = m + fast_log2(l);
}

// dQ: partial rows [bh][share][row][dk], added in the order of the shares (WG: every wave every fourth one, then the four)
template <typename TIO, bool WG>
__global__ __launch_bounds__(256) void band_join_q_kernel(const BandArgs a) {
  dlt_kernargs_in<sizeof(BandArgs)>();
  __shared__ float2 sum[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t at = WG ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  if (!WG && at >= (int64_t)a.B * a.Hkv * a.rows) return;
  const int bh = (int)(at / a.rows), r = (int)(at - (int64_t)bh * a.rows), b = bh / a.Hkv, h = bh - b * a.Hkv;
  const bool on = 2 * lane < a.dk_;
  const int64_t step = (int64_t)a.rows * a.dk_;
  const float* part = a.part + ((int64_t)bh * a.shares * a.rows + r) * a.dk_ + (on ? 2 * lane : 0);
  float2 s = {0.f, 0.f};
#pragma unroll 8
  for (int i = WG ? wave : 0; i < a.shares; i += WG ? 4 : 1) {
    const float2 v = *reinterpret_cast<const float2*>(part + i * step);
    s.x += v.x;
    s.y += v.y;
  }
  if constexpr (WG) {
    sum[wave][lane] = s;
    __syncthreads();
    if (wave != 0) return;
    for (int i = 1; i < 4; i++) { s.x += sum[i][lane].x; s.y += sum[i][lane].y; }
  }
  const float f = a.off + band_row(a, r).tok == 0 ? 0.f : a.grad_scale;   // a row at position 0 sees one key
  TIO* p = band_row_ptr(reinterpret_cast<TIO*>(a.dq) + b * a.dqs[0] + (int64_t)h * a.G * a.dqs[1], a.dqs, a, r);
  if (on) *reinterpret_cast<unsigned*>(p + 2 * lane) = pack2<TIO>(s.x * f, s.y * f);
}

// dK (times sm_scale) or dV: partial sums of the keys that have any (BandParts), added in the order of the shares.  Keys with far sums, of which there are up
// to hundreds, come first, a workgroup to a key, where 8 runs of threads take every eighth sum (one run: 9 us for 16 keys of 112 sums on 4 heads, this way
// 5.5).
template <typename TIO>
__global__ __launch_bounds__(256) void band_join_kv_kernel(const BandArgs a) {
  dlt_kernargs_in<sizeof(BandArgs)>();
  __shared__ f32x4 run[8][32];
  const bool keys = blockIdx.y == 0;
  const int dims = keys ? a.dk_ : a.dv_, per = dims / 4;
  const BandParts P(a);
  const float *part = a.part + (keys ? 0 : P.v_at), *fpart = a.part + (keys ? P.far_at : P.v_at + P.v_far_at);
  const int n_far = (int)dlt_imin64(P.far_keys, P.keys), far_blocks = a.B * a.Hkv * n_far;
  const bool far = (int)blockIdx.x < far_blocks;
  int bh, j, d;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (far) {
    bh = blockIdx.x / n_far;
    j = blockIdx.x - bh * n_far;
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5, n = 4 * a.far;
    d = 4 * c;
    if (c < per) {
      const float* p = fpart + ((int64_t)bh * n * P.far_keys + j) * dims + d;
#pragma unroll 4
      for (int i = r; i < n; i += 8) s += *reinterpret_cast<const f32x4*>(p + (int64_t)i * P.far_keys * dims);
    }
    run[r][c] = s;
    __syncthreads();
    if (r != 0 || c >= per) return;
    for (int i = 1; i < 8; i++) s += run[i][c];
  } else {
    const int64_t gid = (int64_t)(blockIdx.x - far_blocks) * 256 + threadIdx.x, at = gid / per, n = P.keys - n_far;
    d = 4 * (int)(gid - at * per);
    if (at >= (int64_t)a.B * a.Hkv * n) return;
    bh = (int)(at / n);
    j = n_far + (int)(at - bh * n);
  }
#pragma unroll 4
  for (int i = 0; i < a.shares; i++) s += *reinterpret_cast<const f32x4*>(part + (((int64_t)bh * a.shares + i) * P.keys + j) * dims + d);
  if (keys) s *= a.grad_scale;
  const int b = bh / a.Hkv, h = bh - b * a.Hkv;
  TIO* p = keys ? reinterpret_cast<TIO*>(a.dk) + b * a.dks[0] + h * a.dks[1] + j * a.dks[2]
                : reinterpret_cast<TIO*>(a.dv) + b * a.dvs[0] + h * a.dvs[1] + j * a.dvs[2];
  u32x2 w;
  w.x = pack2<TIO>(s[0], s[1]);
  w.y = pack2<TIO>(s[2], s[3]);
  store_stream8(p + d, w);
}

int join_q(const BandArgs& a, int dtype, hipStream_t stream) {
  if (a.shares <= 1) return DLT_OK;
  const int64_t rows = (int64_t)a.B * a.Hkv * a.rows;
  const bool wg = a.shares > 8;
  const dim3 grid((unsigned)(wg ? rows : (rows + 3) / 4));
  dlt_timing_before(DLT_K_BWD_Q, stream);
  if (dtype == DLT_BF16) {
    if (wg) hipLaunchKernelGGL((band_join_q_kernel<bf16_t, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((band_join_q_kernel<bf16_t, false>), grid, dim3(256), 0, stream, a);
  } else {
    if (wg) hipLaunchKernelGGL((band_join_q_kernel<f16_t, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((band_join_q_kernel<f16_t, false>), grid, dim3(256), 0, stream, a);
  }
  dlt_timing_after(stream);
  DLT_CHECK_LAUNCH("window dQ sum launch");
  return DLT_OK;
}

int join(const BandArgs& a, bool backward, int dtype, hipStream_t stream) {
  if (backward ? a.part_keys == 0 : a.shares <= 1) return DLT_OK;
  const int64_t bh = (int64_t)a.B * a.Hkv, rows = bh * a.rows, far = backward ? bh * dlt_imin64(BandParts(a).far_keys, a.part_keys) : 0;
  const int per = dlt_imax(a.dk_, a.dv_) / 4;
  const bool wg = a.shares > 8;
  const dim3 grid((unsigned)(backward ? far + ((bh * a.part_keys - far) * per + 255) / 256 : wg ? rows : (rows + 3) / 4), backward ? 2 : 1);
  dlt_timing_before(backward ? DLT_K_BWD_KV : DLT_K_FWD, stream);
  if (backward) {
    if (dtype == DLT_BF16) hipLaunchKernelGGL(band_join_kv_kernel<bf16_t>, grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(band_join_kv_kernel<f16_t>, grid, dim3(256), 0, stream, a);
  } else {
    if (dtype == DLT_BF16) {
      if (wg) hipLaunchKernelGGL((band_join_kernel<bf16_t, true>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((band_join_kernel<bf16_t, false>), grid, dim3(256), 0, stream, a);
    } else {
      if (wg) hipLaunchKernelGGL((band_join_kernel<f16_t, true>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((band_join_kernel<f16_t, false>), grid, dim3(256), 0, stream, a);
    }
  }
  dlt_timing_after(stream);
  DLT_CHECK_LAUNCH("window sum launch");
  return DLT_OK;
}

// ---- checks ------------------------------------------------------------------------------------------------------------------------
// span: largest offset inside a slab that must fit 32 bits, elements
int check_rows(const char* who, const char* name, const void* p, const int64_t* st, bool empty, int64_t span) {
  DLT_REQUIRE(st != nullptr && (p != nullptr || empty), "%s: %s is NULL", who, name);
  if (empty) return DLT_OK;
  DLT_REQUIRE(st[3] == 1 && (uintptr_t)p % 16 == 0 && st[0] % 8 == 0 && st[1] % 8 == 0 && st[2] % 8 == 0,
              "%s: rows of %s must be contiguous and start at multiples of 16 bytes", who, name);
  DLT_REQUIRE(st[0] >= 0 && st[1] >= 0 && st[2] >= 0, "%s: negative stride of %s", who, name);
  if (span >= (int64_t)1 << 30) return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: strides of %s are too large", who, name);
  return DLT_OK;
}

int check_common(const char* who, int B, int H, int Hkv, int dk, int dv, int window, int n_sink, float sm_scale, int dtype) {
  DLT_REQUIRE(B > 0 && H > 0 && Hkv > 0, "%s: B=%d H=%d Hkv=%d must be positive", who, B, H, Hkv);
  DLT_REQUIRE(H % Hkv == 0, "%s: %d query heads do not share %d key heads evenly", who, H, Hkv);
  DLT_REQUIRE(dk > 0 && dv > 0, "%s: dk=%d dv=%d must be positive", who, dk, dv);
  DLT_REQUIRE(window >= 1 && n_sink >= 0, "%s: window %d must be at least 1, n_sink %d at least 0", who, window, n_sink);
  DLT_REQUIRE(std::isfinite(sm_scale) && sm_scale > 0.f, "%s: sm_scale must be positive and finite", who);
  DLT_REQUIRE(dtype == DLT_BF16 || dtype == DLT_FP16 || dtype == DLT_FP32, "%s: bad dtype %d", who, dtype);
  if (dtype == DLT_FP32) return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: fp32 tensors are not covered, expected bfloat16 or float16", who);
  if (dk > 128 || dv > 128 || dk % 8 != 0 || dv % 8 != 0)
    return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: head dims dk=%d dv=%d must be multiples of 8 up to 128", who, dk, dv);
  return DLT_OK;
}

void set_scalars(BandArgs& a, float sm_scale, int Hkv, int G) {
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  a.Hkv = Hkv;
  a.G = G;
  dlt_fastdiv_make((uint32_t)G, a.mG, a.sG);
  a.q16 = 16 % G == 0;
}

constexpr int LOW_KEYS = 16;
int window_problem(const char* who, const dlt_window_shape_t* s, BandArgs& a) {
  DLT_REQUIRE(s != nullptr, "%s: shape is NULL", who);
  const int rc = check_common(who, s->B, s->H, s->Hkv, s->dk, s->dv, s->window, s->n_sink, s->sm_scale, s->dtype);
  if (rc != DLT_OK) return rc;
  DLT_REQUIRE(s->Lq >= 0 && s->Lk >= 0, "%s: negative length", who);
  const int G = s->H / s->Hkv;
  if ((int64_t)s->Lq * G >= 1 << 30 || s->Lk >= 1 << 30) return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: too many tokens", who);
  a = BandArgs{};
  a.B = s->B; a.Lq = s->Lq; a.Lk = s->Lk; a.dk_ = s->dk; a.dv_ = s->dv;
  a.W = dlt_imin(s->window, dlt_imax(s->Lk, 1));
  a.S = dlt_imin(s->n_sink, s->Lk);
  a.off = s->Lk - s->Lq;
  a.rows = s->Lq * G;
  a.shares = 1;
  set_scalars(a, s->sm_scale, s->Hkv, G);
  a.grad_scale = (a.W == 1 && a.S == 0) || a.Lk == 1 ? 0.f : s->sm_scale;
  // rows with low parts (band_low): all of a short window, else those of the first positions
  a.low_rows = G * (a.W + a.S <= LOW_KEYS ? a.Lq : dlt_imax(0, dlt_imin(LOW_KEYS - a.off, a.Lq)));
  a.group = flash_causal_group(dlt_imax(s->Lk, 1), s->dk, s->dv);
  return DLT_OK;
}

int paged_problem(const char* who, const dlt_paged_shape_t* s, BandArgs& a) {
  DLT_REQUIRE(s != nullptr, "%s: shape is NULL", who);
  const int rc = check_common(who, s->B, s->H, s->Hkv, s->dk, s->dv, s->window, s->n_sink, s->sm_scale, s->dtype);
  if (rc != DLT_OK) return rc;
  DLT_REQUIRE(s->T >= 0 && s->cols > 0 && s->n_pages > 0 && s->page > 0, "%s: T=%d cols=%d n_pages=%d page=%d", who, s->T, s->cols, s->n_pages, s->page);
  if (s->page % 16 != 0) return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: pages of %d tokens, expected a multiple of 16", who, s->page);
  const int G = s->H / s->Hkv;
  if ((int64_t)s->T * G >= 1 << 30 || (int64_t)s->cols * s->page >= 1 << 30) return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: too many tokens", who);
  a = BandArgs{};
  a.B = s->B; a.Lq = s->T; a.Lk = s->cols * s->page; a.dk_ = s->dk; a.dv_ = s->dv;
  a.W = dlt_imin(s->window, a.Lk);
  a.S = dlt_imin(s->n_sink, a.Lk);
  a.rows = s->T * G;
  a.shares = 1;
  set_scalars(a, s->sm_scale, s->Hkv, G);
  a.group = 1;
  a.pg.cols = s->cols;
  a.pg.n_pages = s->n_pages;
  a.pg.p16 = s->page / 16;
  dlt_fastdiv_make((uint32_t)a.pg.p16, a.pg.m16, a.pg.s16);
  return DLT_OK;
}

void set_map(BandArgs& a) {
  auto div = [](int64_t d) {
    BandDiv x;
    dlt_fastdiv_make((uint32_t)dlt_imin64(dlt_imax64(d, 1), 0x7fffffff), x.m, x.s);   // (more workgroups than that are refused)
    return x;
  };
  a.units = (int)dlt_imin64((int64_t)a.nblk * a.shares, 0x7fffffff);
  a.by_group_units = div((int64_t)a.group * a.units);
  a.by_group = div(a.group);
  a.by_last = div((int64_t)a.B * a.Hkv % a.group);
  a.by_shares = div(a.shares);
  a.by_heads = div(a.Hkv);
}
// ---- cutting a call into workgroups ---------------------------------------------------------------------------------------------------
// Rows: how many a workgroup has, and how many workgroups share the keys of a block of rows.
//   BAND_TWO     128 rows, where that makes two workgroups a CU (8 kv heads of 6000 tokens, d = 64, one and a half a CU: forward 29 us by 64 rows, 37 by 128;
//                dQ 33, 42)
//   BAND_ONE     64 rows otherwise, and in a forward pass over few keys at d <= 64, whose set-up weighs more than its reads of LDS (64 kv heads of 4444 rows,
//                window 300, d = 64: 78 -> 72 us; window 500 78 -> 76; window 1024 69 -> 70; at d = 128 107 -> 114; dQ 74 -> 82)
//   BAND_HALVES  64 rows, their keys over two groups of waves, while one workgroup a CU is all there is and the keys of a block are too few, or the workgroups
//                too many, to be shared: a wave alone on its SIMD waits out every latency.  8 heads of 2048 queries, d = 64 / 128, us: 2560 keys each 32 -> 25
//                / 46 -> 35; 640 keys 11.7 -> 11.7 / 16.4 -> 15.2; 4 heads, 640 keys, 10.1 + 6.3 for the sum of 4 shares -> 11.0 / 14.6 + 5.9 -> 14.0; but 12
//                heads (384 workgroups) 14.6 -> 19.7 / 20 -> 26
//   BAND_FEW     16 rows, where that makes no more than a workgroup a CU, few keys: a wave has 32-key chunks of its own, a quarter of the dependent work.  us,
//                against HALVES: 4 heads of 200 tokens, window 64, d = 64, 6.7 -> 5.2; of 1000 tokens, window 300, 9.4 -> 7.0, d = 128 11.8 -> 8.6; 8 heads of
//                500, window 200, d = 128, 10.4 -> 7.8; one token on 300 keys, 8 heads, 8.2 -> 7.6.  With two workgroups a CU 7.7 -> 10.2 (8 heads of 1000,
//                window 100, d = 64); with more keys the shares win: 8 tokens of 8 heads on 900 keys, d = 128, 15.2 -> 8.4 + 3.8
// Shares: up to two workgroups a CU (one round of them: 4 kv heads, 200 queries of two heads on 8000 keys, d = 128, 19 shares of 28
// blocks 24 us, 18 shares 18), at least four chunks each; dQ: while its blocks fill half of the CUs (us with the sum of the parts: 4 kv heads, 200 queries of
// two heads on 8000 keys, d = 128, 132 -> 28; 2 heads, 10 queries of 4 heads on 2000, d = 64, 27 -> 12; but 1000 queries of 8 heads on 1000 keys, 250 blocks,
// 18 -> 20).  Contexts in pages differ in length, and a workgroup does not know its own before it runs: four a CU then (32 sequences of up to 5000 keys, 8 kv
// heads, d = 64 / 128: 47 -> 31 + 5 us / 88 -> 74 + 5; of up to 10000 keys 101 -> 71 + 5 / 169 -> 129 + 5).  Above one and a half workgroups a CU they lose: 64
// sequences, 8 kv heads, d = 128, us without / with shares and their sum: of 5000 keys 212 / 219, of 590 to 5000 165 / 169, 8 of 20000 and 56 of 2500 573 /
// 579; 56 of 600 to 5000 154 / 160.  They would win, and not by much, where one context is far longer than the rest (65536 among 63 of 500: 1170 / 600, its
// bytes take 77).  Both rules go by the table's width, since lengths stay on the device: 300 keys in a table for 8192 are planned as 8192 (9.4 us; 6.8 in a
// table for 300).
int plan_rows(BandArgs& a, bool forward) {
  const int cus = dlt_device_cus();
  const int64_t bh = (int64_t)a.B * a.Hkv;
  const bool paged = a.pg.cols != 0;
  auto blocks = [&](int own) { return (a.rows + own - 1) / own; };
  auto chunks = [&](int own) { return (int)dlt_imin64((int64_t)a.W + a.S + own / a.G + 1, a.Lk) / 64 + 1; };   // of 64 keys, of a block
  int kind = a.rows <= 64 || bh * blocks(128) < 2 * cus ? BAND_ONE : BAND_TWO;
  if (forward && band_class(a.dk_, a.dv_) == 64 && chunks(128) <= 12) kind = BAND_ONE;
  const int64_t one = bh * blocks(64);
  const bool uneven = paged && 2 * one > cus && 2 * one <= 3 * cus && chunks(64) > 32;
  if (forward && kind == BAND_ONE && one <= cus && !uneven) {
    if (bh * blocks(16) <= cus && chunks(16) <= (band_class(a.dk_, a.dv_) == 64 ? 16 : 10)) kind = BAND_FEW;
    else if (chunks(64) <= 12 || 2 * one > cus) kind = BAND_HALVES;
  }
  const int own = kind == BAND_TWO ? 128 : kind == BAND_FEW ? 16 : 64;
  a.nblk = blocks(own);
  a.shares = 1;
  const int64_t wgs = bh * a.nblk;
  if (kind == BAND_ONE && wgs > 0 && (forward ? wgs < cus || uneven : 2 * wgs <= cus)) {
    int64_t n = dlt_imin64(dlt_imin64((uneven ? 4 : 2) * cus / wgs, chunks(own) / 4), BAND_SHARES_MAX);
    const int64_t row_bytes = bh * a.rows * (forward ? a.dv_ + 2 : a.dk_) * 4;
    n = dlt_imin64(n, DLT_WINDOW_WORKSPACE_MAX / dlt_imin64(row_bytes > 0 ? row_bytes : 1, DLT_WINDOW_WORKSPACE_MAX));
    a.shares = n < 1 ? 1 : (int)n;
  }
  set_map(a);
  return kind;
}
int64_t rows_bytes(const BandArgs& a) { return a.shares > 1 ? (int64_t)a.B * a.Hkv * a.shares * a.rows * (a.dv_ + 2) * 4 : 0; }
int64_t q_bytes(const BandArgs& a) { return a.shares > 1 ? (int64_t)a.B * a.Hkv * a.shares * a.rows * a.dk_ * 4 : 0; }
int64_t keys_bytes(const BandArgs& a) { return a.part_keys > 0 ? BandParts(a).floats * 4 : 0; }
// Keys: the rows that see a block of keys taken by several workgroups where blocks are few, the far rows of sinks always
void plan_keys(BandArgs& a) {
  const int cus = dlt_device_cus();
  const int64_t bh = (int64_t)a.B * a.Hkv;
  constexpr int own = BAND_KV_OWN, group = 16;
  a.nblk = (a.Lk + own - 1) / own;
  a.shares = 1;
  a.far = a.far_groups = a.part_keys = 0;
  const int64_t wgs = bh * a.nblk;
  const int64_t near_chunks = dlt_imin64((int64_t)(a.W + own) * a.G, a.rows) / 64 + 1;   // of a block without sinks
  a.cycle = (int)near_chunks;
  // at least 4 chunks a share, 8 at d = 128, whose partial sums weigh more (us with the sum of the parts, 4 / 8 chunks: 2 kv heads of 2000 tokens, 4 query
  // heads each, window 500, 29.8 / 27.6; 4 of 1500, window 300, 37.4 / 30.0; at d = 64 one of 600, window 200, 13.8 / 17.1)
  const int64_t least = band_class(a.dk_, a.dv_) == 64 ? 4 : 8;
  const int64_t want = wgs > 0 && wgs < cus ? (2 * cus + wgs - 1) / wgs : 1;
  const int64_t key_bytes = dlt_imax64(bh * a.Lk * (a.dk_ + a.dv_) * 4, 1);
  a.shares = (int)dlt_imax64(1, dlt_imin64(dlt_imin64(want, near_chunks / least), DLT_WINDOW_WORKSPACE_MAX / 2 / key_bytes));
  const int64_t near_end = dlt_imin64((int64_t)dlt_imax(dlt_imin(own, a.Lk) - 1 - a.off + a.W, 0) * a.G, a.rows);
  const int64_t far_chunks = (a.rows - near_end + 63) / 64;
  if (a.S > 0 && far_chunks > 4) {
    // 16 chunks each, and no more than a near workgroup has: short beside those, which start as these end
    a.far_groups = (a.S + group - 1) / group;
    const int64_t most = dlt_imin64(16, dlt_imax64(4, near_chunks / a.shares));
    const int64_t far_bytes = bh * 4 * a.far_groups * group * (a.dk_ + a.dv_) * 4;
    a.far = (int)dlt_imax64(1, dlt_imin64((far_chunks + most - 1) / most, DLT_WINDOW_WORKSPACE_MAX / 4 / far_bytes));
    a.part_keys = dlt_imin((a.S + own - 1) / own * own, a.Lk);
  }
  if (a.shares > 1) a.part_keys = a.Lk;
  if (keys_bytes(a) > DLT_WINDOW_WORKSPACE_MAX) {   // sinks of very many heads
    a.far = a.far_groups = 0;
    a.part_keys = a.shares > 1 ? a.Lk : 0;
  }
  set_map(a);
}

int check_ws(const char* who, const void* ws, int64_t have, int64_t need) {
  DLT_REQUIRE(need == 0 || (ws != nullptr && have >= need && (uintptr_t)ws % 16 == 0), "%s: needs %lld bytes of 16-byte aligned workspace, got %lld", who,
              (long long)need, (long long)(ws != nullptr ? have : 0));
  return DLT_OK;
}
int check_grid(const char* who, const BandArgs& a) {
  if ((int64_t)a.B * a.Hkv * ((int64_t)a.nblk * a.shares + (int64_t)a.far * a.far_groups) > 0x7fffffff)
    return dlt_set_error(DLT_ERR_UNSUPPORTED, "%s: too many workgroups", who);
  return DLT_OK;
}
void strides3(int64_t (&to)[3], const int64_t* st) {
  for (int i = 0; i < 3; i++) to[i] = st[i];
}
// queries of a (batch, kv head) are addressed with 32-bit offsets over 16 tokens and the heads of the group; keys over 16 tokens
int64_t row_span(const int64_t* st, int G) { return st == nullptr ? 0 : 17 * st[2] + (int64_t)G * st[1]; }
int64_t key_span(const int64_t* st) { return st == nullptr ? 0 : 17 * st[2]; }

}  // namespace

extern "C" int dlt_window_workspace(const dlt_window_shape_t* shape, int backward, int64_t* bytes) {
  DLT_REQUIRE(bytes != nullptr, "window_workspace: bytes is NULL");
  BandArgs a;
  const int rc = window_problem("window_workspace", shape, a);
  if (rc != DLT_OK) return rc;
  if (backward) {   // the passes use the workspace one after the other
    plan_rows(a, false);
    *bytes = q_bytes(a);
    plan_keys(a);
    *bytes = dlt_imax64(*bytes, keys_bytes(a));
  } else {
    plan_rows(a, true);
    *bytes = rows_bytes(a);
  }
  return DLT_OK;
}

extern "C" int dlt_window_low_tokens(const dlt_window_shape_t* shape, int32_t* tokens) {
  DLT_REQUIRE(tokens != nullptr, "window_low_tokens: tokens is NULL");
  BandArgs a;
  const int rc = window_problem("window_low_tokens", shape, a);
  if (rc != DLT_OK) return rc;
  *tokens = a.low_rows / a.G;
  return DLT_OK;
}

extern "C" int dlt_window_fwd(const void* q, const int64_t q_strides[4], const void* k, const int64_t k_strides[4], const void* v, const int64_t v_strides[4],
                              void* o, const int64_t o_strides[4], void* o_low, float* lse2, const dlt_window_shape_t* shape, void* ws, int64_t ws_bytes, void* stream_) {
  const char* who = "window_fwd";
  hipStream_t stream = (hipStream_t)stream_;
  BandArgs a;
  int rc = window_problem(who, shape, a);
  if (rc != DLT_OK) return rc;
  if ((rc = check_rows(who, "q", q, q_strides, a.Lq == 0, row_span(q_strides, a.G))) != DLT_OK) return rc;
  if ((rc = check_rows(who, "k", k, k_strides, a.Lk == 0, key_span(k_strides))) != DLT_OK) return rc;
  if ((rc = check_rows(who, "v", v, v_strides, a.Lk == 0, key_span(v_strides))) != DLT_OK) return rc;
  if ((rc = check_rows(who, "o", o, o_strides, a.Lq == 0, 0)) != DLT_OK) return rc;
  DLT_REQUIRE((uintptr_t)o_low % 16 == 0, "%s: o_low must start at a multiple of 16 bytes", who);
  const int kind = plan_rows(a, true);
  if ((rc = check_ws(who, ws, ws_bytes, rows_bytes(a))) != DLT_OK) return rc;
  if ((rc = check_grid(who, a)) != DLT_OK) return rc;
  if (dlt_route_note(DLT_FAMILY_BAND) || a.Lq == 0) return DLT_OK;
  a.q = q; a.k = k; a.v = v; a.out = o; a.low = o_low; a.lse = lse2; a.part = (float*)ws;
  strides3(a.qs, q_strides); strides3(a.ks, k_strides); strides3(a.vs, v_strides); strides3(a.os, o_strides);
  rc = band_class(a.dk_, a.dv_) == 64 ? dlt_band_fwd_64(a, shape->dtype, kind, stream) : dlt_band_fwd_128(a, shape->dtype, kind, stream);
  return rc != DLT_OK ? rc : join(a, false, shape->dtype, stream);
}

extern "C" int dlt_window_bwd(const void* q, const int64_t q_strides[4], const void* k, const int64_t k_strides[4], const void* v, const int64_t v_strides[4],
                              const void* o, const int64_t o_strides[4], const void* o_low, const void* d_o, const int64_t do_strides[4], const float* lse2, float* delta,
                              void* dq, const int64_t dq_strides[4], void* dk, const int64_t dk_strides[4], void* dv, const int64_t dv_strides[4],
                              const dlt_window_shape_t* shape, void* ws, int64_t ws_bytes, void* stream_) {
  const char* who = "window_bwd";
  hipStream_t stream = (hipStream_t)stream_;
  BandArgs a;
  int rc = window_problem(who, shape, a);
  if (rc != DLT_OK) return rc;
  const bool nq = a.Lq == 0, nk = a.Lk == 0;
  struct { const char* name; const void* p; const int64_t* st; bool none; int64_t span; } ts[] = {
      {"q", q, q_strides, nq, row_span(q_strides, a.G)}, {"k", k, k_strides, nk, key_span(k_strides)}, {"v", v, v_strides, nk, key_span(v_strides)},
      {"o", o, o_strides, nq, 0}, {"d_o", d_o, do_strides, nq, row_span(do_strides, a.G)}, {"dq", dq, dq_strides, nq, 0}, {"dk", dk, dk_strides, nk, 0},
      {"dv", dv, dv_strides, nk, 0}};
  for (const auto& t : ts)
    if ((rc = check_rows(who, t.name, t.p, t.st, t.none, t.span)) != DLT_OK) return rc;
  DLT_REQUIRE((lse2 != nullptr && delta != nullptr) || nq, "%s: lse2 or delta is NULL", who);
  DLT_REQUIRE((uintptr_t)o_low % 16 == 0, "%s: o_low must start at a multiple of 16 bytes", who);
  BandArgs kv = a;
  plan_keys(kv);
  const int kind = plan_rows(a, false);
  if ((rc = check_ws(who, ws, ws_bytes, dlt_imax64(q_bytes(a), keys_bytes(kv)))) != DLT_OK) return rc;
  if ((rc = check_grid(who, a)) != DLT_OK || (rc = check_grid(who, kv)) != DLT_OK) return rc;
  if (dlt_route_note(DLT_FAMILY_BAND)) return DLT_OK;
  for (BandArgs* x : {&a, &kv}) {
    x->q = q; x->k = k; x->v = v; x->o = o; x->d_o = d_o; x->dq = dq; x->dk = dk; x->dv = dv;
    x->low = const_cast<void*>(o_low); x->lse = const_cast<float*>(lse2); x->delta = delta; x->part = (float*)ws;
    strides3(x->qs, q_strides); strides3(x->ks, k_strides); strides3(x->vs, v_strides); strides3(x->os, o_strides); strides3(x->dos, do_strides);
    strides3(x->dqs, dq_strides); strides3(x->dks, dk_strides); strides3(x->dvs, dv_strides);
  }
  const bool small = band_class(a.dk_, a.dv_) == 64;
  if (!nq && (rc = small ? dlt_band_bwd_q_64(a, shape->dtype, kind, stream) : dlt_band_bwd_q_128(a, shape->dtype, kind, stream)) != DLT_OK) return rc;
  if (!nq && (rc = join_q(a, shape->dtype, stream)) != DLT_OK) return rc;
  if (nk) return DLT_OK;
  if ((rc = small ? dlt_band_bwd_kv_64(kv, shape->dtype, stream) : dlt_band_bwd_kv_128(kv, shape->dtype, stream)) != DLT_OK) return rc;
  return join(kv, true, shape->dtype, stream);
}

extern "C" int dlt_paged_workspace(const dlt_paged_shape_t* shape, int64_t* bytes) {
  DLT_REQUIRE(bytes != nullptr, "paged_workspace: bytes is NULL");
  BandArgs a;
  const int rc = paged_problem("paged_workspace", shape, a);
  if (rc != DLT_OK) return rc;
  plan_rows(a, true);
  *bytes = rows_bytes(a);
  return DLT_OK;
}

extern "C" int dlt_paged_attn(const void* q, const int64_t q_strides[4], const void* k_cache, const int64_t k_cache_strides[4], const void* v_cache,
                              const int64_t v_cache_strides[4], void* o, const int64_t o_strides[4], const int32_t* table, int64_t table_stride, const int32_t* seq_len,
                              const int32_t* n_new, const dlt_paged_shape_t* shape, void* ws, int64_t ws_bytes, void* stream_) {
  const char* who = "paged_attn";
  hipStream_t stream = (hipStream_t)stream_;
  BandArgs a;
  int rc = paged_problem(who, shape, a);
  if (rc != DLT_OK) return rc;
  if ((rc = check_rows(who, "q", q, q_strides, a.Lq == 0, row_span(q_strides, a.G))) != DLT_OK) return rc;
  if ((rc = check_rows(who, "k_cache", k_cache, k_cache_strides, false, key_span(k_cache_strides))) != DLT_OK) return rc;
  if ((rc = check_rows(who, "v_cache", v_cache, v_cache_strides, false, key_span(v_cache_strides))) != DLT_OK) return rc;
  if ((rc = check_rows(who, "o", o, o_strides, a.Lq == 0, 0)) != DLT_OK) return rc;
  DLT_REQUIRE(table != nullptr && seq_len != nullptr, "%s: table or seq_len is NULL", who);
  DLT_REQUIRE(table_stride >= 0, "%s: negative table stride", who);
  const int kind = plan_rows(a, true);
  if ((rc = check_ws(who, ws, ws_bytes, rows_bytes(a))) != DLT_OK) return rc;
  if ((rc = check_grid(who, a)) != DLT_OK) return rc;
  if (dlt_route_note(DLT_FAMILY_BAND) || a.Lq == 0) return DLT_OK;
  a.q = q; a.k = k_cache; a.v = v_cache; a.out = o; a.part = (float*)ws;
  strides3(a.qs, q_strides); strides3(a.ks, k_cache_strides); strides3(a.vs, v_cache_strides); strides3(a.os, o_strides);
  a.pg.table = table; a.pg.seq = seq_len; a.pg.n_new = n_new; a.pg.ts = table_stride;
  rc = band_class(a.dk_, a.dv_) == 64 ? dlt_band_paged_64(a, shape->dtype, kind, stream) : dlt_band_paged_128(a, shape->dtype, kind, stream);
  return rc != DLT_OK ? rc : join(a, false, shape->dtype, stream);
}

extern "C" int dlt_paged_append(const void* k, const int64_t k_strides[4], const void* v, const int64_t v_strides[4], const void* q, const int64_t q_strides[4],
                                void* q_out, const int64_t q_out_strides[4], void* k_cache, const int64_t k_cache_strides[4], void* v_cache,
                                const int64_t v_cache_strides[4], const int32_t* table, int64_t table_stride, const int32_t* seq_len, const int32_t* n_new,
                                const dlt_rope_axes_t* rope, const dlt_paged_shape_t* s, void* stream) {
  const char* who = "paged_append";
  DLT_REQUIRE(s != nullptr, "%s: shape is NULL", who);
  DLT_REQUIRE(s->dtype == DLT_BF16 || s->dtype == DLT_FP16 || s->dtype == DLT_FP32, "%s: bad dtype %d", who, s->dtype);
  DLT_REQUIRE(s->B > 0 && s->H >= 0 && s->Hkv > 0 && s->T >= 0 && s->dk > 0 && s->dv > 0, "%s: B=%d H=%d Hkv=%d T=%d dk=%d dv=%d", who, s->B, s->H, s->Hkv, s->T, s->dk,
              s->dv);
  DLT_REQUIRE(s->cols > 0 && s->n_pages > 0 && s->page > 0 && (int64_t)s->cols * s->page < 1 << 30, "%s: cols=%d n_pages=%d page=%d", who, s->cols, s->n_pages, s->page);
  DLT_REQUIRE((int64_t)s->H + 2 * (int64_t)s->Hkv <= 0x7fffffff, "%s: too many heads", who);
  DLT_REQUIRE(table != nullptr && seq_len != nullptr && table_stride >= 0, "%s: table or seq_len is NULL, or the table's stride negative", who);
  RotArgs a{};
  const int rc = dlt_rope_axes_make(rope, s->dk, false, 0, who, a.r);
  if (rc != DLT_OK) return rc;
  auto stream_of = [&](const void* src, const int64_t* ss, const void* dst, const int64_t* ds, int H, int C, int rot, int paged) {
    RotStream& x = a.s[a.n++];
    x.src = src; x.dst = const_cast<void*>(dst);
    for (int i = 0; i < 4; i++) { x.ss[i] = ss[i]; x.ds[i] = ds[i]; }
    x.H = H; x.C = C; x.rot = rot; x.paged = paged;
  };
  const bool none = s->T == 0;
  DLT_REQUIRE(k_strides != nullptr && v_strides != nullptr && k_cache_strides != nullptr && v_cache_strides != nullptr && k_cache != nullptr && v_cache != nullptr &&
                  (none || (k != nullptr && v != nullptr)), "%s: a tensor of keys or values is NULL", who);
  if (s->H > 0) {
    DLT_REQUIRE(q_strides != nullptr && q_out_strides != nullptr && (none || (q != nullptr && q_out != nullptr)), "%s: q or q_out is NULL", who);
    DLT_REQUIRE(none || q != q_out, "%s: q and q_out must be two buffers", who);
    stream_of(q, q_strides, q_out, q_out_strides, s->H, s->dk, 1, 0);
  }
  stream_of(k, k_strides, k_cache, k_cache_strides, s->Hkv, s->dk, 1, 1);
  stream_of(v, v_strides, v_cache, v_cache_strides, s->Hkv, s->dv, 0, 1);
  if (none) return DLT_OK;
  a.B = s->B; a.T = s->T;
  a.table = table; a.seq = seq_len; a.n_new = n_new; a.tbs = table_stride;
  a.cols = s->cols; a.n_pages = s->n_pages; a.page = s->page;
  return dlt_rotate_rows(a, s->dtype, "paged_append launch", (hipStream_t)stream);
}
