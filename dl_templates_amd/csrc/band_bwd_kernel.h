// Backward pass of attention over a 1D window with sinks and grouped heads (band_common.h).
//
//   P = exp2(scale q.k - lse2), dP = dO.v, dS = P (dP - delta), delta = rowsum(dO o)
//   dQ = sm_scale dS K  (rows own, K and V stream; this kernel runs first and stores delta)
//   dK = sm_scale dS^T Q, dV = P^T dO  (keys own; the rows of all heads of the group stream, so the sum over the heads that share a
//   key is part of the product: no atomics, one order of summation)
// P and dS are rounded to 16 bits for the second products, as their operands have to be; sums stay in 32 bits to the end.
#pragma once
#include "band_common.h"

// ---- dQ ---------------------------------------------------------------------------------------------------------------------------
template <typename TIO, int D, int NP, int CK, int NW, int PAD>
__global__ __launch_bounds__(64 * NW, NW == 4 && D <= 64 ? 3 : 2) void band_bwd_q_kernel(const BandArgs a) {
  dlt_kernargs_in<sizeof(BandArgs)>();
  typedef BandBuf<D, CK> B;
  extern __shared__ __align__(16) char smem[];
  constexpr int KC = band_kc(D, PAD), KB = 2 * KC, NKB = CK / 32, OWN = 16 * NP * NW;
  constexpr int NBUF = band_nbuf(B::BUF), AHEAD = NBUF - 1;
  constexpr int NG = CK / NW / 16;
  static_assert(NG >= 1 && NG * NW * 16 == CK, "whole groups of 16 tokens per wave");
  constexpr int PER_CHUNK = 2 * NG * BandStage<D>::NI;

  const int tid = threadIdx.x;
  const int lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  const int lin = xcd_remap(blockIdx.x, gridDim.x);
  int b, h, blk, share;
  band_block(a, lin, true, b, h, blk, share);
  const int x0 = blk * OWN, bh = b * a.Hkv + h;
  const TIO* qb = reinterpret_cast<const TIO*>(a.q) + b * a.qs[0] + (int64_t)h * a.G * a.qs[1];
  const TIO* dob = reinterpret_cast<const TIO*>(a.d_o) + b * a.dos[0] + (int64_t)h * a.G * a.dos[1];
  const TIO* ob = reinterpret_cast<const TIO*>(a.o) + b * a.os[0] + (int64_t)h * a.G * a.os[1];
  const TIO* kh = reinterpret_cast<const TIO*>(a.k) + b * a.ks[0] + h * a.ks[1];
  const TIO* vh = reinterpret_cast<const TIO*>(a.v) + b * a.vs[0] + h * a.vs[1];

  BandWalk<CK> W;
  const int xl = dlt_imin(x0 + OWN, a.rows) - 1;
  const int first = a.off + band_row(a, x0).tok, last = a.off + band_row(a, xl).tok;
  W.init(first, last, a.W, a.S);
  // chunks of this share: few rows on many keys (BAND_ONE) are split over workgroups, whose partial sums a second launch adds
  const int per = NP == 1 ? (W.n + a.shares - 1) / a.shares : W.n;
  const int i_beg = NP == 1 ? dlt_imin(share * per, W.n) : 0, i_end = NP == 1 ? dlt_imin(i_beg + per, W.n) : W.n;

  BandStage<D> stk, stv;
  stk.init(lane, a.dk_, a.ks[2]);
  stv.init(lane, a.dv_, a.vs[2]);
  if constexpr (PAD) {
#pragma unroll
    for (int i = 0; i < NBUF; i++) {
      flashd_zero_pads<D>(smem + i * B::BUF, CK, a.dk_ >> 3, tid, 64 * NW);
      flashd_zero_pads<D>(smem + i * B::BUF + B::REG, CK, a.dv_ >> 3, tid, 64 * NW);
    }
  }
  auto issue = [&](int i, char* buf) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NG; u++) {
      const int t0 = W.tok(CK * i + wave * 16 * NG + 16 * u);
      char* dst = buf + (wave * 16 * NG + 16 * u) * 2 * D;
      if (t0 + 16 <= a.Lk) {
        stk.template issue<PAD>(reinterpret_cast<const char*>(kh + (int64_t)t0 * a.ks[2]), dst);
        stv.template issue<PAD>(reinterpret_cast<const char*>(vh + (int64_t)t0 * a.vs[2]), dst + B::REG);
      } else {
        keep_branch();
        const int tc = dlt_imin(t0, a.Lk - 1);
        stk.template issue_clamped<PAD>(reinterpret_cast<const char*>(kh + (int64_t)tc * a.ks[2]), a.Lk - 1 - tc, dst);
        stv.template issue_clamped<PAD>(reinterpret_cast<const char*>(vh + (int64_t)tc * a.vs[2]), a.Lk - 1 - tc, dst + B::REG);
      }
    }
  };
#pragma unroll 1
  for (int i = 0; i < AHEAD; i++)
    if (i_beg + i < i_end) issue(i_beg + i, smem + i * B::BUF);

  const int wq0 = x0 + wave * 16 * NP;
  u32x4 qf[NP][KC], dof[NP][KC];
  float nlse[NP], del[NP];
  int hi[NP], lo[NP];
  const int64_t row0 = (int64_t)bh * a.rows;
#pragma unroll
  for (int p = 0; p < NP; p++) {
    const int r = wq0 + 16 * p + n;
    const bool on = r < a.rows;
    const int rc = on ? r : 0, pos = a.off + band_row(a, rc).tok;
    hi[p] = on ? pos - W.jump : -1;   // the row sees places lo < y <= hi, and the sinks
    lo[p] = pos - a.W - W.jump;
    band_load_own<KC>(qf[p], band_row_ptr(qb, a.qs, a, rc), on, a.dk_, g);
    band_load_own<KC>(dof[p], band_row_ptr(dob, a.dos, a, rc), on, a.dv_, g);
    nlse[p] = on ? -a.lse[row0 + r] : 0.f;
    u32x4 of[KC];
    band_load_own<KC>(of, band_row_ptr(ob, a.os, a, rc), on, a.dv_, g);
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < KC; c++) {
      float fo[8], fd[8];
      unpack8<TIO>(of[c], fo);
      unpack8<TIO>(dof[p][c], fd);
#pragma unroll
      for (int j = 0; j < 8; j++) sum += fo[j] * fd[j];
    }
    const TIO* low = on && a.low != nullptr ? band_low<TIO>(a, b, h, r) : nullptr;
    if (low != nullptr) {
      band_load_own<KC>(of, low, true, a.dv_, g);
#pragma unroll
      for (int c = 0; c < KC; c++) {
        float fo[8], fd[8];
        unpack8<TIO>(of[c], fo);
        unpack8<TIO>(dof[p][c], fd);
#pragma unroll
        for (int j = 0; j < 8; j++) sum += fo[j] * fd[j];
      }
    }
    del[p] = wave_sum4(sum);
    if (g == 0 && on && share == 0) store_stream4(a.delta + row0 + r, del[p]);
  }
  const int wl = dlt_imin(wq0 + 16 * NP, a.rows) - 1;
  const int pa = wl >= wq0 ? a.off + band_row(a, wq0).tok - W.jump : 0, pb = wl >= wq0 ? a.off + band_row(a, wl).tok - W.jump : -1;

  f32x4 acc[NP][KB];
#pragma unroll
  for (int p = 0; p < NP; p++)
#pragma unroll
    for (int d = 0; d < KB; d++) acc[p][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float scale = a.scale_log2;
  FlashDLane<D> L;
  flashd_lane_init(L, n, g);

  swa2_wait_copies();
  pin_loaded(qf);
  pin_loaded(dof);
#pragma unroll
  for (int p = 0; p < NP; p++) { pin_loaded(nlse[p]); pin_loaded(del[p]); }
  // the dP products start from -delta: the matrix pipe delivers dP - delta
  f32x4 dinit[NP];
#pragma unroll
  for (int p = 0; p < NP; p++) dinit[p] = f32x4{-del[p], -del[p], -del[p], -del[p]};
  __syncthreads();

  auto consume = [&](const int x, Swa2Lds __restrict__ cur, auto mask_tag) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    Swa2Lds sK = cur, sV = cur + B::REG;
    constexpr int N1H = 2 * KC, N1 = 2 * N1H, NB = N1 + KB, NT = NKB * NB;
    constexpr int RD = 1;   // LDS reads ahead of the matrix instruction (2 to 6: no faster)
    u32x4 ring[RD + 1];
    auto rd = [&](auto kc) __attribute__((always_inline)) {
      constexpr int k = decltype(kc)::value;
      constexpr int kb = k / NB, j = k % NB;
      if constexpr (j < N1) {
        constexpr int mb = j / N1H, r = j % N1H, T0 = 32 * kb + 16 * mb;
        if constexpr (r < KC) ring[k % (RD + 1)] = swa2_lds16(sK + T0 * FlashDRow<D>::ROW + L.a[r]);
        else ring[k % (RD + 1)] = swa2_lds16(sV + T0 * FlashDRow<D>::ROW + L.a[r - KC]);
      } else {
        ring[k % (RD + 1)] = flashd_read_tr<D, 32 * kb>(sK, L, j - N1);
      }
    };
    BandEdge edge[NP];
    if constexpr (MASK) {
#pragma unroll
      for (int p = 0; p < NP; p++) edge[p] = band_edge(hi[p], lo[p], a.S, x, g);
    }
    swa2_for<0, RD>([&](auto kc) __attribute__((always_inline)) { rd(kc); });
    swa2_for<0, NKB>([&](auto kbc) __attribute__((always_inline)) {
      constexpr int kb = decltype(kbc)::value;
      float ds[NP][8];
      f32x4 sv[NP], dp[NP];
      u32x4 dsb[NP];
      swa2_for<0, NB>([&](auto jc) __attribute__((always_inline)) {
        constexpr int j = decltype(jc)::value, k = kb * NB + j;
        if constexpr (k + RD < NT) rd(std::integral_constant<int, k + RD>{});
        __builtin_amdgcn_sched_barrier(0);
        const u32x4 op = ring[k % (RD + 1)];
        if constexpr (j < N1) {
          constexpr int mb = j / N1H, r = j % N1H;
#pragma unroll
          for (int p = 0; p < NP; p++) {
            if constexpr (r < KC) sv[p] = Mma<TIO>::mfma(op, qf[p][r], r == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sv[p]);
            else dp[p] = Mma<TIO>::mfma(op, dof[p][r - KC], r == KC ? dinit[p] : dp[p]);
          }
          if constexpr (r == N1H - 1) {
#pragma unroll
            for (int p = 0; p < NP; p++)
#pragma unroll
              for (int i = 0; i < 4; i++) {
                float v = fast_exp2(fmaf(sv[p][i], scale, nlse[p])) * dp[p][i];
                if constexpr (MASK) {
                  v = band_formed(v);
                  v = band_edge_sees(edge[p], 32 * kb + 16 * mb + i) ? v : 0.f;
                }
                ds[p][4 * mb + i] = v;
              }
            if constexpr (mb == 1) {
#pragma unroll
              for (int p = 0; p < NP; p++) dsb[p] = pack8<TIO>(ds[p]);
            }
          }
        } else {
#pragma unroll
          for (int p = 0; p < NP; p++) acc[p][j - N1] = Mma<TIO>::mfma(op, dsb[p], acc[p][j - N1]);
        }
      });
    });
  };
  auto chunk = [&](int i, char* buf, auto mask_tag) __attribute__((always_inline)) {
    const int x = CK * i;
    if (decltype(mask_tag)::value && (x > pb || (x + CK - 1 <= pa - a.W && x >= a.S))) return;
    consume(x, (Swa2Lds)buf, mask_tag);
  };
  int f0, f1;
  W.whole(first, last, a.W, i_beg, i_end, f0, f1);
  // loops of their own: BandWalk::whole
  int bi = 0, i = i_beg, stop = f0;
  auto buf_of = [&](int i) { return smem + (i >= NBUF ? i - NBUF : i) * B::BUF; };
  auto step = [&](auto mask_tag) __attribute__((always_inline)) {
    const bool more = i + AHEAD < i_end;
    if (more) issue(i + AHEAD, buf_of(bi + AHEAD));
    chunk(i, buf_of(bi), mask_tag);
    if (more) flashd_wait_copies<(AHEAD - 1) * PER_CHUNK>();
    else swa2_wait_copies();
    bi = bi + 1 == NBUF ? 0 : bi + 1;
    i++;
    __syncthreads();
  };
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    while (i < stop) step(std::true_type{});
    if (i >= i_end) break;
#pragma unroll 1
    while (i < f1) step(std::false_type{});
    stop = i_end;
  }
  __syncthreads();
  float mul[NP];
  unsigned odd[NP];
#pragma unroll
  for (int p = 0; p < NP; p++) {
    mul[p] = hi[p] + W.jump == 0 ? 0.f : a.grad_scale;   // a row at position 0 sees one key
    const uint64_t bad = __builtin_amdgcn_ballot_w64(wq0 + 16 * p + n < a.rows && band_odd_row(acc, p));
    odd[p] = (unsigned)((bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffff);
  }
  // a row with an infinite or NaN sum once more, over the keys of the share that it sees alone (band_common.h): two dims, without the factor
  auto exact = [&](int r, float (&sum)[2]) __attribute__((always_inline)) {
    const int pos = a.off + band_row(a, r).tok;
    const TIO *q = band_row_ptr(qb, a.qs, a, r), *d_o = band_row_ptr(dob, a.dos, a, r);
    const TIO* low = a.low != nullptr ? band_low<TIO>(a, b, h, r) : nullptr;
    const float lse = a.lse[row0 + r], delta = band_dot(band_row_ptr(ob, a.os, a, r), d_o, a.dv_) + (low != nullptr ? band_dot(low, d_o, a.dv_) : 0.f);
    sum[0] = sum[1] = 0.f;
#pragma unroll 1
    for (int c = i_beg; c < i_end; c++)
#pragma unroll 1
      for (int x = CK * c; x < CK * c + CK; x += 64) {
        const int j = W.tok(x + lane);
        const bool sees = j < a.Lk && band_sees(pos, j, a.W, a.S);
        uint64_t left = __builtin_amdgcn_ballot_w64(sees);
        float ds = 0.f;
        if (sees) ds = fast_exp2(band_dot(q, kh + j * a.ks[2], a.dk_) * scale - lse) * (band_dot(d_o, vh + j * a.vs[2], a.dv_) - delta);
        for (; left != 0; left &= left - 1) {
          const int u = __builtin_ctzll(left);
          band_axpy(sum, band_lane(ds, u), kh + W.tok(x + u) * a.ks[2], a.dk_, lane);
        }
      }
  };
  if (NP == 1 && a.shares > 1) {
    float* part = a.part + ((int64_t)bh * a.shares + share) * a.rows * a.dk_;
    flash_share_put<NP>(part, acc, a.dk_, wq0 + n, a.rows, g);
    for (unsigned todo = odd[0]; todo != 0; todo &= todo - 1) {
      const int r = wq0 + __builtin_ctz(todo);
      float sum[2];
      exact(r, sum);
      __threadfence();   // behind the wave's own stores of the row
      if (2 * lane < a.dk_) *reinterpret_cast<float2*>(part + (int64_t)r * a.dk_ + 2 * lane) = float2{sum[0], sum[1]};
    }
    return;
  }
  TIO* dqb = reinterpret_cast<TIO*>(a.dq) + b * a.dqs[0] + (int64_t)h * a.G * a.dqs[1];
  constexpr int PT = D * 2 + 16;
  band_store_rows<D, NP, TIO>(smem, acc, mul, NW, 1, true, a.dk_, wave, n, g, tid,
                              [&](int row) -> TIO* { return x0 + row < a.rows ? band_row_ptr(dqb, a.dqs, a, x0 + row) : nullptr; },
                              [&]() {
#pragma unroll 1
                                for (int p = 0; p < NP; p++)
                                  for (unsigned todo = odd[p]; todo != 0; todo &= todo - 1) {
                                    const int w = 16 * p + __builtin_ctz(todo), r = wq0 + w;
                                    float sum[2];
                                    exact(r, sum);
                                    const float f = a.off + band_row(a, r).tok == 0 ? 0.f : a.grad_scale;
                                    if (2 * lane < D)
                                      *reinterpret_cast<unsigned*>(smem + (wave * 16 * NP + w) * PT + 4 * lane) = pack2<TIO>(sum[0] * f, sum[1] * f);
                                  }
                              });
}

// Sinks are seen by every later row, so a block of keys with sinks would have the rows of the whole sequence where others have those of a
// window.  The rows behind the block's window ("far" rows) are therefore taken by workgroups of their own, a share of the rows each: the 16 keys
// of a far workgroup belong to all its waves, which take 16 of a chunk's 64 rows each, with half-filled second products.  Far workgroups
// and the blocks with sinks leave partial sums, which a second launch adds in a fixed order.  16 heads on 4, 8192 tokens, window 1024, 4 sinks,
// d = 128: 876 us with the far rows in the block, 187 with workgroups of 1024 far rows, launched first, beside it.
// ---- dK / dV -------------------------------------------------------------------------------------------------------------------------
template <typename TIO, int D, int PAD>
__global__ __launch_bounds__(256, 2) void band_bwd_kv_kernel(const BandArgs a) {
  dlt_kernargs_in<sizeof(BandArgs)>();
  constexpr int CK = 64, NW = 4;   // rows of a chunk; waves, of 16 keys each
  typedef BandBuf<D, CK> B;
  extern __shared__ __align__(16) char smem[];
  constexpr int KC = band_kc(D, PAD), KB = 2 * KC, NQB = CK / 32, OWN = 16 * NW;
  constexpr int NBUF = band_nbuf(B::BUF), AHEAD = NBUF - 1;
  constexpr int NG = CK / NW / 16;
  static_assert(NG >= 1 && NG * NW * 16 == CK && CK == 64, "whole groups of 16 rows per wave; one copy of scalars a chunk");
  constexpr int PER_CHUNK = 2 * NG * BandStageRows<D>::NI;   // waves 0 and 1: one more

  const int tid = threadIdx.x;
  const int lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // far workgroups are launched first: behind the others, which fill the chip in whole rounds, they would be a tail of their own
  const int n_far = a.far * a.far_groups, all_far = a.B * a.Hkv * n_far;
  const bool far = (int)blockIdx.x < all_far;
  const int lin = far ? xcd_remap(blockIdx.x, all_far) : xcd_remap((int)blockIdx.x - all_far, (int)gridDim.x - all_far);
  int b, h, share, x0;
  if (far) {
    const int bh = lin / n_far;
    const int rest = lin - bh * n_far, grp = rest / a.far;
    share = rest - grp * a.far;
    x0 = grp * 16;
    b = band_div(bh, a.by_heads);
    h = bh - b * a.Hkv;
  } else {
    int blk;
    band_block(a, lin, false, b, h, blk, share);
    x0 = blk * OWN;
  }
  const int bh = b * a.Hkv + h;
  const int xe = dlt_imin(x0 + (far ? 16 : OWN), a.Lk);
  const char* qb = reinterpret_cast<const char*>(reinterpret_cast<const TIO*>(a.q) + b * a.qs[0] + (int64_t)h * a.G * a.qs[1]);
  const char* dob = reinterpret_cast<const char*>(reinterpret_cast<const TIO*>(a.d_o) + b * a.dos[0] + (int64_t)h * a.G * a.dos[1]);
  const TIO* kh = reinterpret_cast<const TIO*>(a.k) + b * a.ks[0] + h * a.ks[1];
  const TIO* vh = reinterpret_cast<const TIO*>(a.v) + b * a.vs[0] + h * a.vs[1];
  const int64_t row0 = (int64_t)bh * a.rows;

  // rows [r_beg, r_end) see some own key; key j is seen by rows [rlo(j), rhi(j))
  auto rlo_of = [&](int j) { return (int)dlt_imin64((int64_t)dlt_imax(j - a.off, 0) * a.G, a.rows); };
  // far rows start behind the last row whose window holds a key of the block (far workgroups: of the block that their keys lie in)
  auto near_end = [&](int last) { return (int)dlt_imin64((int64_t)dlt_imax(last - a.off + a.W, 0) * a.G, a.rows); };
  const int r_beg = far ? near_end(dlt_imin(x0 / OWN * OWN + OWN, a.Lk) - 1) : rlo_of(x0);
  const int r_end = far ? a.rows : x0 < a.S && a.far == 0 ? a.rows : near_end(xe - 1);
  auto rhi_of = [&](int j) { return j < a.S ? r_end : near_end(j); };
  const int nch = r_end > r_beg ? (r_end - r_beg + CK - 1) / CK : 0;
  const int n_shares = far ? a.far : a.shares;
  const int per = (nch + n_shares - 1) / n_shares;
  const int i_beg = dlt_imin(share * per, nch), i_end = dlt_imin(i_beg + per, nch);

  BandStageRows<D> stq, std_;
  stq.init(a, lane, a.dk_, a.qs);
  std_.init(a, lane, a.dv_, a.dos);
  if constexpr (PAD) {
#pragma unroll
    for (int i = 0; i < NBUF; i++) {
      flashd_zero_pads<D>(smem + i * B::BUF_KV, CK, a.dk_ >> 3, tid, 64 * NW);
      flashd_zero_pads<D>(smem + i * B::BUF_KV + B::REG, CK, a.dv_ >> 3, tid, 64 * NW);
    }
  }
  const float* scal = (wave == 0 ? a.lse : a.delta) + row0;
  auto issue = [&](int i, char* buf) __attribute__((always_inline)) {
    const int r0 = r_beg + i * CK;
#pragma unroll
    for (int u = 0; u < NG; u++) {
      const int at = wave * 16 * NG + 16 * u;
      stq.template issue<PAD>(a, qb, a.qs, r0 + at, a.rows - 1, buf + at * 2 * D);
      std_.template issue<PAD>(a, dob, a.dos, r0 + at, a.rows - 1, buf + B::REG + at * 2 * D);
    }
    if (wave < 2)
      dlt_copy4_to_lds(reinterpret_cast<const char*>(scal + r0), (uint32_t)dlt_imin(lane, a.rows - 1 - r0) * 4u, buf + 2 * B::REG + wave * (CK * 4));
  };
  // Chunks are taken cyclically from one whose place is a multiple of `cycle` on: a block's rows overlap those of its neighbours, which then ask for the same
  // chunk at the same time. Each from its own first one, the workgroups of an XCD would spread over more rows than its L2 holds (8192 tokens, window 1024, 16
  // heads on 4, d = 128: 860 MB fetched for 84, now 144; 188 -> 184 us; 4 sequences, window 512, 32 heads on 8, 665 -> 632)
  const int n_ch = i_end - i_beg;
  int start = 0;
  if (!far) {
    const int c = (r_beg / CK + i_beg) % a.cycle;
    start = c != 0 && a.cycle - c < n_ch ? a.cycle - c : 0;
  }
  auto at = [&](int s) { const int c = s + start; return i_beg + (c >= n_ch ? c - n_ch : c); };
#pragma unroll 1
  for (int i = 0; i < AHEAD; i++)
    if (i < n_ch) issue(at(i), smem + i * B::BUF_KV);

  const int wk0 = far ? x0 : x0 + wave * 16;
  u32x4 kf[KC], vf[KC];
  const int own = wk0 + n;
  const bool on = own < a.Lk;
  const int rlo = on ? rlo_of(own) : a.rows, rhi = on ? rhi_of(own) : 0;
  band_load_own<KC>(kf, kh + (on ? own : 0) * a.ks[2], on, a.dk_, g);
  band_load_own<KC>(vf, vh + (on ? own : 0) * a.vs[2], on, a.dv_, g);
  // rows that see some key of the wave: [wlo, whi)
  const int wk1 = dlt_imin(wk0 + 16, xe) - 1;
  const bool wave_on = wk1 >= wk0;
  const int wlo = wave_on ? rlo_of(wk0) : 0, whi = !wave_on ? 0 : wk0 < a.S ? r_end : rhi_of(wk1);

  f32x4 dk_acc[1][KB], dv_acc[1][KB];   // as the helpers of several blocks a wave take them
#pragma unroll
  for (int d = 0; d < KB; d++) dk_acc[0][d] = dv_acc[0][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float scale = a.scale_log2;
  FlashDLane<D> L;
  flashd_lane_init(L, n, g);

  swa2_wait_copies();
  pin_loaded(kf);
  pin_loaded(vf);
  // the own values are negated and the dP products start from the rows' delta: the matrix pipe delivers -(dP - delta)
#pragma unroll
  for (int c = 0; c < KC; c++) {
    vf[c].x ^= 0x80008000u; vf[c].y ^= 0x80008000u; vf[c].z ^= 0x80008000u; vf[c].w ^= 0x80008000u;
  }
  __syncthreads();

  auto consume = [&](const int q0, Swa2Lds __restrict__ cur, auto mask_tag) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    Swa2Lds sQ = cur, sDO = cur + B::REG;
    Swa2Lds sLse = cur + 2 * B::REG + 16 * g, sDel = sLse + CK * 4;
    // the first products (S, dP) of every 16-row half, then the second ones (dV, dK) block by block; the element-wise work of a half is
    // issued in pieces behind the matrix instructions of the following segment
    constexpr int N1H = 2 * KC, NH = 2 * NQB, N1 = NH * N1H, NSEG = 2 * KB, NT = N1 + NQB * NSEG;
    constexpr int NU = 2;   // element-wise pieces of a half
    // Each sum is a chain of products that wait for each other: at d = 128 S and dP take turns (8192 tokens, window 1024, 16 heads on 4 179 -> 173 us; 8 x 8 kv
    // heads of 4 query heads, 1111 tokens, 138 -> 129), at d = 64, where three workgroups share a CU, one follows the other (98 against 100, 76 against 76)
    constexpr auto score = [](int r) { return D > 64 ? r % 2 == 0 : r < KC; };
    constexpr auto dims = [](int r) { return D > 64 ? r / 2 : r % KC; };
    static_assert(NSEG >= NU && N1H >= NU, "a segment must have room for the element-wise pieces of a half");
    constexpr int RD = 3;   // 1: 197 us, 3: 187 for 16 heads on 4, 8192 tokens, window 1024, d = 128; more: spills
    u32x4 ring[RD + 1];
    auto rd = [&](auto kc) __attribute__((always_inline)) {
      constexpr int k = decltype(kc)::value;
      if constexpr (k < N1) {
        constexpr int hh = k / N1H, r = k % N1H, T0 = 16 * hh;
        ring[k % (RD + 1)] = swa2_lds16((score(r) ? sQ : sDO) + T0 * FlashDRow<D>::ROW + L.a[dims(r)]);
      } else {
        constexpr int qb_ = (k - N1) / NSEG, d = (k - N1) % NSEG;
        if constexpr (d < KB) ring[k % (RD + 1)] = flashd_read_tr<D, 32 * qb_>(sDO, L, d);
        else ring[k % (RD + 1)] = flashd_read_tr<D, 32 * qb_>(sQ, L, d - KB);
      }
    };
    int elo, ehi;   // row 16 hh + 4 g + i of the chunk is seen iff elo <= 16 hh + i < ehi (see band_edge)
    if constexpr (MASK) {
      int at = q0 + 4 * g;
      asm volatile("" : "+v"(at));
      elo = rlo - at;
      ehi = rhi - at;
    }
    swa2_for<0, RD>([&](auto kc) __attribute__((always_inline)) { rd(kc); });
    f32x4 sv[2], dp[2], lq[2], dl[2];   // by the parity of the half
    dl[0] = __builtin_bit_cast(f32x4, swa2_lds16(sDel));
    u32x4 pb[NQB], dsb[NQB];
    auto ew = [&](auto hhc, auto uc) __attribute__((always_inline)) {
      constexpr int hh = decltype(hhc)::value, u = decltype(uc)::value;
      constexpr int qb_ = hh / 2, mb = hh % 2, i0_ = 2 * u;
      float pr[2], ds[2];
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const int i = i0_ + t;
        float pv = fast_exp2(fmaf(sv[hh & 1][i], scale, -lq[hh & 1][i]));
        float dv = -pv * dp[hh & 1][i];
        if constexpr (MASK) {
          const bool sees = 16 * hh + i >= elo && 16 * hh + i < ehi;
          pv = band_formed(pv);
          dv = band_formed(dv);
          pv = sees ? pv : 0.f;
          dv = sees ? dv : 0.f;
        }
        pr[t] = pv;
        ds[t] = dv;
      }
      const unsigned pw = pack2<TIO>(pr[0], pr[1]), dw = pack2<TIO>(ds[0], ds[1]);
      if constexpr (mb == 0 && i0_ == 0) { pb[qb_].x = pw; dsb[qb_].x = dw; }
      if constexpr (mb == 0 && i0_ == 2) { pb[qb_].y = pw; dsb[qb_].y = dw; }
      if constexpr (mb == 1 && i0_ == 0) { pb[qb_].z = pw; dsb[qb_].z = dw; }
      if constexpr (mb == 1 && i0_ == 2) { pb[qb_].w = pw; dsb[qb_].w = dw; }
    };
    swa2_for<0, NT>([&](auto kc) __attribute__((always_inline)) {
      constexpr int k = decltype(kc)::value;
      if constexpr (k + RD < NT) rd(std::integral_constant<int, k + RD>{});
      if constexpr (k < N1 && k % N1H == 0) {
        constexpr int hh = k / N1H;
        lq[hh & 1] = __builtin_bit_cast(f32x4, swa2_lds16(sLse + 16 * hh * 4));
      }
      if constexpr (k < N1 && k % N1H == KC && k / N1H + 1 < NH) {
        constexpr int hn = k / N1H + 1;
        dl[hn & 1] = __builtin_bit_cast(f32x4, swa2_lds16(sDel + 16 * hn * 4));
      }
      __builtin_amdgcn_sched_barrier(0);
      const u32x4 op = ring[k % (RD + 1)];
      if constexpr (k < N1) {
        constexpr int hh = k / N1H, r = k % N1H;
        if constexpr (score(r)) sv[hh & 1] = Mma<TIO>::mfma(op, kf[dims(r)], dims(r) == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sv[hh & 1]);
        else dp[hh & 1] = Mma<TIO>::mfma(op, vf[dims(r)], dims(r) == 0 ? dl[hh & 1] : dp[hh & 1]);
        if constexpr (hh >= 1 && r < NU) {
          ew(std::integral_constant<int, hh - 1>{}, std::integral_constant<int, r>{});
          SWA2_MIX(1, 12)
        }
      } else {
        constexpr int qb_ = (k - N1) / NSEG, d = (k - N1) % NSEG;
        if constexpr (d < KB) dv_acc[0][d] = Mma<TIO>::mfma(op, pb[qb_], dv_acc[0][d]);
        else dk_acc[0][d - KB] = Mma<TIO>::mfma(op, dsb[qb_], dk_acc[0][d - KB]);
        if constexpr (qb_ == 0 && d < NU) {
          ew(std::integral_constant<int, NH - 1>{}, std::integral_constant<int, d>{});
          SWA2_MIX(1, 12)
        }
      }
    });
  };
  // far: rows 16 wave .. + 15 of the chunk
  auto consume_far = [&](const int q0, Swa2Lds __restrict__ cur) __attribute__((always_inline)) {
    Swa2Lds sQ = cur + 16 * wave * FlashDRow<D>::ROW, sDO = sQ + B::REG;
    Swa2Lds sLse = cur + 2 * B::REG + 16 * g + 64 * wave, sDel = sLse + CK * 4;
    const f32x4 lq = __builtin_bit_cast(f32x4, swa2_lds16(sLse)), dl = __builtin_bit_cast(f32x4, swa2_lds16(sDel));
    f32x4 sv, dp;
#pragma unroll
    for (int r = 0; r < KC; r++) {
      const u32x4 x = swa2_lds16(sQ + L.a[r]), y = swa2_lds16(sDO + L.a[r]);
      sv = Mma<TIO>::mfma(x, kf[r], r == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sv);
      dp = Mma<TIO>::mfma(y, vf[r], r == 0 ? dl : dp);
    }
    float pr[4], ds[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int r = q0 + 16 * wave + 4 * g + i;
      const bool sees = r >= rlo && r < rhi;
      const float pv = fast_exp2(fmaf(sv[i], scale, -lq[i]));
      pr[i] = sees ? pv : 0.f;
      ds[i] = sees ? -pv * dp[i] : 0.f;
    }
    const u32x4 pb = {pack2<TIO>(pr[0], pr[1]), pack2<TIO>(pr[2], pr[3]), 0u, 0u}, dsb = {pack2<TIO>(ds[0], ds[1]), pack2<TIO>(ds[2], ds[3]), 0u, 0u};
#pragma unroll
    for (int d = 0; d < KB; d++) {
      const u32x2 x = swa2_lds_tr(sDO + L.tr[d]), y = swa2_lds_tr(sQ + L.tr[d]);
      dv_acc[0][d] = Mma<TIO>::mfma(u32x4{x.x, x.y, 0u, 0u}, pb, dv_acc[0][d]);
      dk_acc[0][d] = Mma<TIO>::mfma(u32x4{y.x, y.y, 0u, 0u}, dsb, dk_acc[0][d]);
    }
  };
  struct Far {};
  auto chunk = [&](int i, char* buf, auto tag) __attribute__((always_inline)) {
    const int q0 = r_beg + i * CK;
    if constexpr (std::is_same<decltype(tag), Far>::value) consume_far(q0, (Swa2Lds)buf);
    else {
      if (decltype(tag)::value && (q0 >= whi || q0 + CK <= wlo)) return;
      consume(q0, (Swa2Lds)buf, tag);
    }
  };
  // chunks whose rows see all keys of the workgroup: rows [rlo of the last key, rhi of the first one without sinks)
  const int all_lo = rlo_of(xe - 1), all_hi = x0 >= a.S ? rhi_of(x0) : xe <= a.S ? r_end : rhi_of(a.S);
  const int f0 = dlt_imin(dlt_imax(i_beg, (all_lo - r_beg + CK - 1) / CK), i_end);
  const int f1 = dlt_imax(f0, dlt_imin(i_end, all_hi > r_beg ? (all_hi - r_beg) / CK : 0));
  // loops of their own (BandWalk::whole), counted from `start`: masked chunks up to `stop`, whole ones up to `whole`, masked ones up to m1, whole ones
  const int g0 = f0 - i_beg, g1 = f1 - i_beg;   // whole chunks
  int bi = 0, i = 0;
  int stop = start < g0 ? g0 - start : start < g1 ? 0 : n_ch - start + g0, whole = start < g1 ? g1 - start : n_ch - start + g1;
  const int m1 = start >= g0 && start < g1 ? n_ch - start + g0 : n_ch;
  auto buf_of = [&](int i) { return smem + (i >= NBUF ? i - NBUF : i) * B::BUF_KV; };
  auto step = [&](auto mask_tag) __attribute__((always_inline)) {
    const bool more = i + AHEAD < n_ch;
    if (more) issue(at(i + AHEAD), buf_of(bi + AHEAD));
    chunk(at(i), buf_of(bi), mask_tag);
    if (more) flashd_wait_copies<(AHEAD - 1) * PER_CHUNK>();
    else swa2_wait_copies();
    bi = bi + 1 == NBUF ? 0 : bi + 1;
    i++;
    __syncthreads();
  };
  if (far) {
#pragma unroll 1
    while (i < n_ch) step(Far{});
  }
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    while (i < stop) step(std::true_type{});
    if (i >= n_ch) break;
#pragma unroll 1
    while (i < whole) step(std::false_type{});
    stop = m1;
    whole = n_ch;
  }
  __syncthreads();

  // ---- epilogue
  const float mulk[1] = {a.grad_scale}, mulv[1] = {1.f};
  const uint64_t bad = __builtin_amdgcn_ballot_w64(own < a.Lk && (band_odd_row(dk_acc, 0) || band_odd_row(dv_acc, 0)));
  const unsigned odd = (unsigned)((bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffff);   // keys of the wave to be taken again
  // one own key once more over the rows of chunks [i_beg, i_end) that see it: two dims of dK (without sm_scale) and dV
  auto exact = [&](int xk, float (&sk)[2], float (&sv)[2]) __attribute__((always_inline)) {
    const TIO *k = kh + xk * a.ks[2], *v = vh + xk * a.vs[2];
    const int lo = dlt_imax(rlo_of(xk), r_beg + i_beg * CK), hi = dlt_imin(rhi_of(xk), r_beg + i_end * CK);
    sk[0] = sk[1] = sv[0] = sv[1] = 0.f;
#pragma unroll 1
    for (int r0 = lo; r0 < hi; r0 += 64) {
      const int r = r0 + lane;
      float p = 0.f, ds = 0.f;
      const bool mine = r < hi && (!far || ((r - r_beg) >> 4 & 3) == wave);
      const uint64_t todo = __builtin_amdgcn_ballot_w64(mine);
      if (mine) {
        const TIO *q = band_row_ptr(reinterpret_cast<const TIO*>(qb), a.qs, a, r), *d_o = band_row_ptr(reinterpret_cast<const TIO*>(dob), a.dos, a, r);
        p = fast_exp2(band_dot(q, k, a.dk_) * scale - a.lse[row0 + r]);
        ds = p * (band_dot(d_o, v, a.dv_) - a.delta[row0 + r]);
      }
      for (uint64_t left = todo; left != 0; left &= left - 1) {
        const int u = __builtin_ctzll(left);
        band_axpy(sv, band_lane(p, u), band_row_ptr(reinterpret_cast<const TIO*>(dob), a.dos, a, r0 + u), a.dv_, lane);
        band_axpy(sk, band_lane(ds, u), band_row_ptr(reinterpret_cast<const TIO*>(qb), a.qs, a, r0 + u), a.dk_, lane);
      }
    }
  };
  if (far || a.shares > 1 || (a.far != 0 && x0 < a.S)) {
    const BandParts P(a);
    const int64_t row = far ? (((int64_t)bh * a.far + share) * 4 + wave) * P.far_keys : ((int64_t)bh * a.shares + share) * P.keys;
    float* pk = a.part + (far ? P.far_at : 0) + row * a.dk_;
    float* pv = a.part + P.v_at + (far ? P.v_far_at : 0) + row * a.dv_;
    const int len = far ? (int)P.far_keys : a.Lk;
    flash_share_put<1>(pk, dk_acc, a.dk_, wk0 + n, len, g);
    flash_share_put<1>(pv, dv_acc, a.dv_, wk0 + n, len, g);
    for (unsigned todo = odd; todo != 0; todo &= todo - 1) {
      const int xk = wk0 + __builtin_ctz(todo);
      float sk[2], sv[2];
      exact(xk, sk, sv);
      __threadfence();   // behind the wave's own stores of the row
      if (2 * lane < a.dk_) *reinterpret_cast<float2*>(pk + (int64_t)xk * a.dk_ + 2 * lane) = float2{sk[0], sk[1]};
      if (2 * lane < a.dv_) *reinterpret_cast<float2*>(pv + (int64_t)xk * a.dv_ + 2 * lane) = float2{sv[0], sv[1]};
    }
    return;
  }
  constexpr int PT = D * 2 + 16;
  auto again = [&](bool keys) __attribute__((always_inline)) {
    for (unsigned todo = odd; todo != 0; todo &= todo - 1) {
      const int w = __builtin_ctz(todo);
      float sk[2], sv[2];
      exact(wk0 + w, sk, sv);
      const float f = keys ? a.grad_scale : 1.f;
      const float x = (keys ? sk[0] : sv[0]) * f, y = (keys ? sk[1] : sv[1]) * f;
      if (2 * lane < D) *reinterpret_cast<unsigned*>(smem + (wave * 16 + w) * PT + 4 * lane) = pack2<TIO>(x, y);
    }
  };
  TIO* dkb = reinterpret_cast<TIO*>(a.dk) + b * a.dks[0] + h * a.dks[1];
  TIO* dvb = reinterpret_cast<TIO*>(a.dv) + b * a.dvs[0] + h * a.dvs[1];
  band_store_rows<D, 1, TIO>(smem, dk_acc, mulk, NW, 1, true, a.dk_, wave, n, g, tid,
                              [&](int row) -> TIO* { return x0 + row < a.Lk ? dkb + (x0 + row) * a.dks[2] : nullptr; }, [&]() { again(true); });
  band_store_rows<D, 1, TIO>(smem, dv_acc, mulv, NW, 1, true, a.dv_, wave, n, g, tid,
                              [&](int row) -> TIO* { return x0 + row < a.Lk ? dvb + (x0 + row) * a.dvs[2] : nullptr; }, [&]() { again(false); });
}
