// Forward pass of attention over a 1D window with sinks and grouped heads (band_common.h), keys and values dense or in pages.
//
// A workgroup of NW waves owns 16 NP NW rows (query token, head) of one group; K and V stream through LDS in chunks of CK keys, copied
// asynchronously, 16 tokens a wave (in pages: one page lookup).  Per chunk: S^T = K Q^T, one update of the running maximum and sum, O^T +=
// V^T P^T.  Chunks that every row of a wave sees whole run without a mask, chunks that no row sees are left out.
// P is rounded to 16 bits for the second product, as its operand has to be; sums, maxima and outputs stay in 32 bits to the end.
#pragma once
#include "band_common.h"

// What one sequence of a call holds
struct BandSeq {
  int off, n_q, n_k;   // position of query token 0, query tokens, keys
};
template <bool PAGED>
DLT_DEV BandSeq band_seq(const BandArgs& a, int b) {
  BandSeq s{a.off, a.Lq, a.Lk};
  if constexpr (PAGED) {
    s.n_q = a.pg.n_new != nullptr ? dlt_imax(0, dlt_imin(a.pg.n_new[b], a.Lq)) : a.Lq;
    s.n_k = dlt_imax(0, dlt_imin(a.pg.seq[b], a.Lk));   // Lk: what the table's row can hold
    s.off = s.n_k - s.n_q;
  }
  return s;
}
// Page of the 16 tokens that hold position 16 t16.  A number outside the pool is the caller's mistake: the nearest page is read.
DLT_DEV int band_page(const BandPages& pg, const int32_t* row, int t16, int& in16) {
  const int pi = (int)dlt_fastdiv((uint32_t)t16, pg.m16, pg.s16);
  in16 = t16 - pi * pg.p16;
  return dlt_imax(0, dlt_imin(row[pi], pg.n_pages - 1));
}
// Element offset of key j inside the tensor at the head's base
template <bool PAGED>
DLT_DEV int64_t band_key_off(const BandArgs& a, const int32_t* row, const int64_t (&st)[3], int j) {
  if constexpr (!PAGED) return j * st[2];
  int in16;
  const int page = band_page(a.pg, row, j >> 4, in16);
  return page * st[0] + (in16 * 16 + (j & 15)) * st[2];
}

// A cached key or value in 8 bits, at the head's base: its numbers, the factor of their scale
struct BandKey8 { const uint8_t* p; float scale; };
DLT_DEV BandKey8 band_key8(const Band8Args& a, const int32_t* row, const void* base, const int64_t (&st)[3], const uint8_t* sc, const int64_t (&ss)[3], int j) {
  int in16;
  const int page = band_page(a.pg, row, j >> 4, in16);
  return BandKey8{reinterpret_cast<const uint8_t*>(base) + (page * st[0] + (in16 * 16 + (j & 15)) * st[2]),
                  cvt8_scale(sc[page * ss[0] + (int)dlt_fastdiv((uint32_t)in16, a.mB, a.sB) * ss[2]])};
}
template <int FMT, typename TIO>
DLT_DEV float band_dot8(const TIO* x, const BandKey8& y, int dims) {
  float s = 0.f;
  for (int d = 0; d < dims; d += 8) {
    float fx[8], fy[8];
    const u32x2 w = *reinterpret_cast<const u32x2*>(y.p + d);
    unpack8<TIO>(*reinterpret_cast<const u32x4*>(x + d), fx);
    unpack8<TIO>(cvt8_eight<FMT, TIO>(w[0], w[1], y.scale), fy);
#pragma unroll
    for (int j = 0; j < 8; j++) s = fmaf(fx[j], fy[j], s);
  }
  return s;
}

// One row again over the keys of chunks [i0, i1) that it sees: maximum (log2 units), sum, two dims of the unnormalised output
template <typename TIO, bool PAGED, int CK, int F8 = 0>
DLT_DEV void band_fwd_exact(const typename BandArgsOf<F8>::type& a, int h, const TIO* q, const TIO* kb, const TIO* vb, const int32_t* pages, const BandWalk<CK>& W, int i0, int i1, int pos,
                            int n_k, int lane, float& m, float& l, float (&acc)[2]) {
  m = -INFINITY;
  l = acc[0] = acc[1] = 0.f;
#pragma unroll 1
  for (int i = i0; i < i1; i++)
#pragma unroll 1
    for (int x = CK * i; x < CK * i + CK; x += 64) {
      const int j = W.tok(x + lane);
      const bool sees = j < n_k && (CK >= 64 || lane < CK) && band_sees(pos, j, a.W, a.S);
      uint64_t todo = __builtin_amdgcn_ballot_w64(sees);
      if (todo == 0) continue;
      float s = -INFINITY;
      if constexpr (F8 == 0) s = sees ? band_dot(q, kb + band_key_off<PAGED>(a, pages, a.ks, j), a.dk_) * a.scale_log2 : -INFINITY;
      else if (sees) s = band_dot8<F8 - 1, TIO>(q, band_key8(a, pages, kb, a.ks, a.k_sc + h * a.kss[1], a.kss, j), a.dk_) * a.scale_log2;
      const float m_new = fmaxf(m, band_wave_max(s));
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - ref);
      const float p = sees ? fast_exp2(s - ref) : 0.f;
      m = m_new;
      l *= alpha; acc[0] *= alpha; acc[1] *= alpha;
      while (todo != 0) {
        const int u = __builtin_ctzll(todo);
        todo &= todo - 1;
        const float w = band_lane(p, u);
        l += w;
        if constexpr (F8 == 0) band_axpy(acc, w, vb + band_key_off<PAGED>(a, pages, a.vs, W.tok(x + u)), a.dv_, lane);
        else {
          const BandKey8 v = band_key8(a, pages, vb, a.vs, a.v_sc + h * a.vss[1], a.vss, W.tok(x + u));
          if (2 * lane < a.dv_) {
            const unsigned p2 = cvt8_pair<F8 - 1, TIO>(*reinterpret_cast<const uint16_t*>(v.p + 2 * lane), v.scale, false);
            acc[0] = fmaf(w, unpack_lo<TIO>(p2), acc[0]);
            acc[1] = fmaf(w, unpack_hi<TIO>(p2), acc[1]);
          }
        }
      }
    }
}

// GR groups of NW waves own the same rows and take every GR-th chunk each; their results are joined at the end, through LDS.
// F8 (pages, GR = 1): keys and values in 8 bits.  A chunk comes through registers, becomes 16-bit numbers there, once for all rows of the workgroup, and lies in LDS as the
// copies of a 16-bit chunk do; from there on nothing differs.
template <typename TIO, int D, int NP, int CK, int NW, int GR, bool PAGED, int PAD, int F8 = 0>
__global__ __launch_bounds__(64 * NW * GR, NW * GR == 4 ? 2 : 1) void band_fwd_kernel(const typename BandArgsOf<F8>::type a) {
  static_assert(F8 == 0 || (PAGED && GR == 1), "8-bit numbers: pages, one group of waves");
  dlt_kernargs_in<sizeof(typename BandArgsOf<F8>::type)>();
  typedef BandBuf<D, CK> B;
  extern __shared__ __align__(16) char smem[];
  constexpr int KC = band_kc(D, PAD), VB = 2 * KC, NKB = CK / 32, OWN = 16 * NP * NW;
  constexpr int NBUF = band_nbuf(B::BUF, GR), AHEAD = NBUF - 1;
  constexpr int NG = CK / NW / 16;                              // groups of 16 tokens that a wave copies
  static_assert(NG >= 1 && NG * NW * 16 == CK, "whole groups of 16 tokens per wave");
  constexpr int PER_CHUNK = 2 * NG * BandStage<D>::NI;

  const int tid = threadIdx.x;
  const int lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave_all = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = GR == 1 ? 0 : wave_all / NW, wave = wave_all - grp * NW;   // group of the wave, wave of the group

  const int lin = xcd_remap(blockIdx.x, gridDim.x);
  int b, h, blk, share;
  band_block(a, lin, true, b, h, blk, share);
  const int x0 = blk * OWN, bh = b * a.Hkv + h;
  const BandSeq sq = band_seq<PAGED>(a, b);
  const int n_rows = sq.n_q * a.G;                              // rows with a query; those behind get zeros
  const TIO* qb = reinterpret_cast<const TIO*>(a.q) + b * a.qs[0] + (int64_t)h * a.G * a.qs[1];
  typedef typename std::conditional<F8 != 0, uint8_t, TIO>::type TKV;
  const TKV* kh = reinterpret_cast<const TKV*>(a.k) + (PAGED ? 0 : b * a.ks[0]) + h * a.ks[1];
  const TKV* vh = reinterpret_cast<const TKV*>(a.v) + (PAGED ? 0 : b * a.vs[0]) + h * a.vs[1];
  const int32_t* pages = PAGED ? a.pg.table + b * a.pg.ts : nullptr;

  // chunks of the block and of this share of it
  BandWalk<CK> W;
  const int xl = dlt_imin(x0 + OWN, n_rows) - 1;
  const int first = sq.off + band_row(a, x0).tok, last = xl >= x0 ? dlt_imin(sq.off + band_row(a, dlt_imax(xl, 0)).tok, sq.n_k - 1) : -1;
  W.init(first, last, a.W, a.S);
  const int per = (W.n + a.shares - 1) / a.shares;
  const int i_beg = dlt_imin(share * per, W.n), i_end = dlt_imin(i_beg + per, W.n);

  BandStage<D> stk, stv;
  stk.init(lane, a.dk_, a.ks[2]);
  stv.init(lane, a.dv_, a.vs[2]);
  if constexpr (PAD && F8 == 0) {
#pragma unroll
    for (int i = 0; i < NBUF * GR; i++) {
      flashd_zero_pads<D>(smem + i * B::BUF, CK, a.dk_ >> 3, tid, 64 * NW * GR);
      flashd_zero_pads<D>(smem + i * B::BUF + B::REG, CK, a.dv_ >> 3, tid, 64 * NW * GR);
    }
  }
  char* const bufs = smem + grp * NBUF * B::BUF;   // of the group
  // page of each group of 16 tokens that the wave copies of a chunk (of any chunk: numbers behind the last one are taken back to it)
  struct Groups { int page[NG], in16[NG]; };
  auto lookup = [&](int i) __attribute__((always_inline)) {
    Groups x;
    if constexpr (PAGED) {
#pragma unroll
      for (int u = 0; u < NG; u++)
        x.page[u] = band_page(a.pg, pages, dlt_imax(0, dlt_imin(W.tok(CK * i + wave * 16 * NG + 16 * u), sq.n_k - 1)) >> 4, x.in16[u]);
    }
    return x;
  };
  auto issue = [&](int i, char* buf, const Groups& x) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NG; u++) {
      const int t0 = W.tok(CK * i + wave * 16 * NG + 16 * u);
      char* dst = buf + (wave * 16 * NG + 16 * u) * 2 * D;
      if constexpr (PAGED) {
        const int page = x.page[u];
        const int64_t row = 16 * x.in16[u];
        stk.template issue<PAD>(reinterpret_cast<const char*>(kh + (page * a.ks[0] + row * a.ks[2])), dst);
        stv.template issue<PAD>(reinterpret_cast<const char*>(vh + (page * a.vs[0] + row * a.vs[2])), dst + B::REG);
      } else {
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
    }
  };
  // Pages hold anything behind the last key: those value rows, which no row sees, are cleared by the wave that copied them
  auto settle = [&](int i, char* buf) __attribute__((always_inline)) {
    if constexpr (PAGED) {
#pragma unroll
      for (int u = 0; u < NG; u++) {
        const int t0 = W.tok(CK * i + wave * 16 * NG + 16 * u);
        if (t0 + 16 > sq.n_k) {
          keep_branch();
          char* v = buf + B::REG + (wave * 16 * NG + 16 * u) * 2 * D;
          for (int s = lane; s < 16 * D / 8; s += 64)
            if (t0 + s / (D / 8) >= sq.n_k) lds_write16(v + 16 * s, u32x4{0u, 0u, 0u, 0u});
        }
      }
    }
  };
  // 8-bit numbers: the wave's 16 tokens of the chunk behind the next one are on their way in registers.  Pages of 64 chunks are looked up at once, a lane each: a load of one
  // page a chunk, scalar or not, is a trip to memory that waits in the products end on.
  typedef BandStage8<D, F8 == 2 ? DLT_INT8 : DLT_FP8_E4M3, TIO> S8;
  static_assert(F8 == 0 || NG == 1, "16 tokens of a chunk a wave");
  S8 stk8, stv8;
  u32x4 rk[S8::NI], rv[S8::NI];
  int ek, ev, page64;
  // (tokens behind the last one are taken back to it; the table has a column for position 0)
  auto fetch8 = [&](int i) __attribute__((always_inline)) {
    if constexpr (F8 != 0) {
      auto group = [&](int c) __attribute__((always_inline)) { return dlt_imax(0, dlt_imin(W.tok(CK * c + wave * 16), sq.n_k - 1)) >> 4; };
      const int u = (i - i_beg) & 63;
      if (u == 0) page64 = pages[dlt_fastdiv((uint32_t)group(i + lane), a.pg.m16, a.pg.s16)];
      const int t16 = group(i), in16 = t16 - (int)dlt_fastdiv((uint32_t)t16, a.pg.m16, a.pg.s16) * a.pg.p16, blk = (int)dlt_fastdiv((uint32_t)in16, a.mB, a.sB);
      const int page = dlt_imax(0, dlt_imin(__builtin_amdgcn_readlane(page64, u), a.pg.n_pages - 1));
      const int64_t row = 16 * in16;
      stk8.fetch(reinterpret_cast<const char*>(kh) + (page * a.ks[0] + row * a.ks[2]), rk);
      stv8.fetch(reinterpret_cast<const char*>(vh) + (page * a.vs[0] + row * a.vs[2]), rv);
      ek = a.k_sc[page * a.kss[0] + h * a.kss[1] + blk * a.kss[2]];
      ev = a.v_sc[page * a.vss[0] + h * a.vss[1] + blk * a.vss[2]];
    }
  };
  // before chunk i goes to LDS: pages hold anything behind the last token; those values, which no row sees, are cleared, and so are scales of blocks of nothing else
  auto settle8 = [&](int i) __attribute__((always_inline)) {
    const int live = sq.n_k - W.tok(CK * i + wave * 16);
    if (live < 16) {
      keep_branch();
      stv8.clear(rv, live);
      if (live <= 0) ev = 127;
    }
  };
  constexpr int PUTS = F8 != 0 ? 4 * S8::NI : 0;   // 16-byte writes of a wave
  auto put8 = [&](char* buf, auto jc) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value;
    char* dst = buf + wave * 16 * 2 * D;
    // (one scale for the wave: formed by the scalar unit; 512 tokens over 8192, int8 / e4m3 108.5 / 99.8 -> 105.6 / 95 us)
    if constexpr (j < 2 * S8::NI) stk8.template put<j>(dst, rk, cvt8_scale(__builtin_amdgcn_readfirstlane(ek)));
    else stv8.template put<j - 2 * S8::NI>(dst + B::REG, rv, cvt8_scale(__builtin_amdgcn_readfirstlane(ev)));
  };
  if constexpr (F8 != 0) {
    stk8.init(lane, a.dk_, a.ks[2]);
    stv8.init(lane, a.dv_, a.vs[2]);
    if (i_beg < i_end) {
      fetch8(i_beg);
      settle8(i_beg);
      swa2_for<0, PUTS>([&](auto jc) __attribute__((always_inline)) { put8(bufs, jc); });
      if (i_beg + 1 < i_end) fetch8(i_beg + 1);
    }
  } else if constexpr (PAGED) {
    // Pages of the first chunks are looked up together: one trip to memory, not one a chunk (a token each of 8 sequences of up to 900, d = 64: 10.7 -> 10.1 us;
    // one sequence of 5000, d = 128: 10.1 -> 8.7; large grids alike).  Looked up behind the last chunk too: the table has a column for position 0.
    Groups x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; i++) x[i] = lookup(i_beg + i * GR + grp);
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
      if (i_beg + i * GR + grp < i_end) issue(i_beg + i * GR + grp, bufs + i * B::BUF, x[i]);
  } else {
#pragma unroll 1
    for (int i = 0; i < AHEAD; i++)
      if (i_beg + i * GR + grp < i_end) issue(i_beg + i * GR + grp, bufs + i * B::BUF, Groups{});
  }

  const int wq0 = x0 + wave * 16 * NP;
  u32x4 qf[NP][KC];
  int hi[NP], lo[NP];   // the row sees places lo < y <= hi, and the sinks
#pragma unroll
  for (int p = 0; p < NP; p++) {
    const int r = wq0 + 16 * p + n;
    const bool on = r < n_rows;
    const int pos = sq.off + band_row(a, on ? r : 0).tok;
    hi[p] = on ? dlt_imin(pos, sq.n_k - 1) - W.jump : -1;
    lo[p] = pos - a.W - W.jump;
    band_load_own<KC>(qf[p], band_row_ptr(qb, a.qs, a, on ? r : 0), on, a.dk_, g);
  }
  // places of the wave's first and last row
  const int wl = dlt_imin(wq0 + 16 * NP, n_rows) - 1;
  const int pa = wl >= wq0 ? sq.off + band_row(a, wq0).tok - W.jump : 0, pb = wl >= wq0 ? sq.off + band_row(a, wl).tok - W.jump : -1;

  float m_run[NP];
  f32x4 acc[NP][VB], acc_l[NP];
#pragma unroll
  for (int p = 0; p < NP; p++) {
    m_run[p] = -INFINITY;
    acc_l[p] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < VB; d++) acc[p][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float scale = a.scale_log2;
  const unsigned one2 = pack2<TIO>(1.f, 1.f);
  const u32x4 row_of_ones = n == 0 ? u32x4{one2, one2, one2, one2} : u32x4{0u, 0u, 0u, 0u};
  FlashDLane<D> lanes;
  flashd_lane_init(lanes, n, g);

  if constexpr (F8 == 0) swa2_wait_copies();
  pin_loaded(qf);
#pragma unroll
  for (int i = 0; i < AHEAD; i++)
    if (F8 == 0 && i_beg + i * GR + grp < i_end) settle(i_beg + i * GR + grp, bufs + i * B::BUF);
  __syncthreads();

  // beside(k): what runs beside the k-th operand's products
  auto consume = [&](const int x, Swa2Lds __restrict__ cur, auto mask_tag, auto beside) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    Swa2Lds sK = cur, sV = cur + B::REG;
    constexpr int N1 = NKB * 2 * KC, NT = N1 + NKB * VB;
    constexpr int RD = 1;   // LDS reads ahead of the matrix instruction (2 to 6: no faster)
    u32x4 ring[RD + 1];
    // 8-bit numbers under way take registers that places in LDS would fill: those are formed from one, a[c] = a[0] ^ 64 c and tr[d] = tr[0] ^ 32 d, and so is the row of ones
    FlashDLane<D> L = lanes;
    u32x4 ones = row_of_ones;
    if constexpr (F8 != 0) {
      int a0 = lanes.a[0], t0 = lanes.tr[0];
      unsigned o = row_of_ones[0];
      asm volatile("" : "+v"(a0), "+v"(t0), "+v"(o));
#pragma unroll
      for (int c = 0; c < D / 32; c++) L.a[c] = a0 ^ 64 * c;
#pragma unroll
      for (int d = 0; d < D / 16; d++) L.tr[d] = t0 ^ 32 * d;
      ones = u32x4{o, o, o, o};
    }
    auto rd = [&](auto kc) __attribute__((always_inline)) {
      constexpr int k = decltype(kc)::value;
      if constexpr (k < N1) {
        constexpr int kb = k / (2 * KC), mb = (k / KC) % 2, r = k % KC;
        ring[k % (RD + 1)] = swa2_lds16(sK + (32 * kb + 16 * mb) * FlashDRow<D>::ROW + L.a[r]);
      } else {
        constexpr int kb = (k - N1) / VB, d = (k - N1) % VB;
        ring[k % (RD + 1)] = flashd_read_tr<D, 32 * kb>(sV, L, d);
      }
    };
    swa2_for<0, RD>([&](auto kc) __attribute__((always_inline)) { rd(kc); });
    BandEdge edge[NP];
    if constexpr (MASK) {
#pragma unroll
      for (int p = 0; p < NP; p++) edge[p] = band_edge(hi[p], lo[p], a.S, x, g);
    }
    float t[NP][NKB][8];
    u32x4 pb_[NP][NKB];
    f32x4 s[NP];
    swa2_for<0, NT>([&](auto kc) __attribute__((always_inline)) {
      constexpr int k = decltype(kc)::value;
      if constexpr (k + RD < NT) rd(std::integral_constant<int, k + RD>{});
      __builtin_amdgcn_sched_barrier(0);
      const u32x4 op = ring[k % (RD + 1)];
      if constexpr (k < N1) {
        constexpr int kb = k / (2 * KC), mb = (k / KC) % 2, r = k % KC;
#pragma unroll
        for (int p = 0; p < NP; p++) s[p] = Mma<TIO>::mfma(op, qf[p][r], r == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[p]);
        beside(kc);
        if constexpr (r == KC - 1) {
#pragma unroll
          for (int p = 0; p < NP; p++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              float v = s[p][i];
              if constexpr (MASK) v = band_edge_sees(edge[p], 32 * kb + 16 * mb + i) ? v : -INFINITY;
              t[p][kb][4 * mb + i] = v;
            }
        }
        if constexpr (k == N1 - 1) {
#pragma unroll
          for (int p = 0; p < NP; p++) {
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int kb2 = 0; kb2 < NKB; kb2++)
#pragma unroll
              for (int i = 0; i < 4; i++) mx[i] = fmaxf(fmaxf(mx[i], t[p][kb2][2 * i]), t[p][kb2][2 * i + 1]);
            const float mloc = wave_max4(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
            // the reference maximum moves only when a score exceeds it by more than 2^8 after scaling: P stays below 2^8, its sum in
            // 32 bits below 2^8 times the keys.  In masked chunks, where rows of few keys lie, it moves with the maximum: the largest P is then 1, and not
            // rounded
            if (__builtin_amdgcn_ballot_w64((mloc - m_run[p]) * scale > (MASK ? 0.f : 8.f))) {
              keep_branch();
              const float m_new = fmaxf(m_run[p], mloc);
              const float alpha = fast_exp2((m_run[p] - m_new) * scale);
              m_run[p] = m_new;
              const float al = m_new == -INFINITY ? 1.f : alpha;
#pragma unroll
              for (int d = 0; d < VB; d++) acc[p][d] *= al;
              acc_l[p] *= al;
            }
            const float neg_m2 = m_run[p] == -INFINITY ? 0.f : -m_run[p] * scale;
#pragma unroll
            for (int kb2 = 0; kb2 < NKB; kb2++) {
#pragma unroll
              for (int i = 0; i < 8; i++) t[p][kb2][i] = fast_exp2(fmaf(t[p][kb2][i], scale, neg_m2));
              if constexpr (MASK) {   // rows of few keys lie in masked chunks: the sum of what is rounded afterwards, in 32 bits
                float l[4];
#pragma unroll
                for (int i = 0; i < 4; i++) l[i] = t[p][kb2][i] + t[p][kb2][4 + i];
                acc_l[p][0] += (l[0] + l[1]) + (l[2] + l[3]);
              }
              pb_[p][kb2] = pack8<TIO>(t[p][kb2]);
            }
          }
        }
      } else {
        constexpr int kb = (k - N1) / VB, d = (k - N1) % VB;
#pragma unroll
        for (int p = 0; p < NP; p++) acc[p][d] = Mma<TIO>::mfma(op, pb_[p][kb], acc[p][d]);
        if constexpr (d == VB - 1 && !MASK) {   // elsewhere the sum of the rounded P, a row of ones in the matrix product
#pragma unroll
          for (int p = 0; p < NP; p++) acc_l[p] = Mma<TIO>::mfma(ones, pb_[p][kb], acc_l[p]);
        }
      }
    });
  };
  auto chunk = [&](int i, char* buf, auto mask_tag, auto beside) __attribute__((always_inline)) {
    const int x = CK * i;
    if (decltype(mask_tag)::value && (x > pb || (x + CK - 1 <= pa - a.W && x >= a.S))) return;   // no row of the wave sees any of it
    consume(x, (Swa2Lds)buf, mask_tag, beside);
  };
  int f0, f1;
  W.whole(first, last, a.W, i_beg, i_end, f0, f1);
  // loops of their own: BandWalk::whole
  const int rounds = (i_end - i_beg + GR - 1) / GR, r0 = (f0 - i_beg + GR - 1) / GR, r1 = (f1 - i_beg) / GR;
  int bi = 0, it = 0, stop = dlt_imin(r0, rounds);
  auto buf_of = [&](int i) { return bufs + (i >= NBUF ? i - NBUF : i) * B::BUF; };
  auto step = [&](auto mask_tag) __attribute__((always_inline)) {
    const int i = i_beg + it * GR + grp;
    if constexpr (F8 != 0) {
      // The next chunk goes to LDS, where the last one was, beside the products of S, which leave the vector units idle; in masked chunks before them (beside them the compiler
      // runs out of registers: whole-number caches 115 -> 135 us).  Behind the last chunk nothing reads what is written.  512 tokens over 8192, 32 heads on 8, d = 128, all
      // pieces ahead of the products -> this: 110 -> 98 us (int8 115 -> 108), 2048 tokens 330 -> 275.
      settle8(i + 1);
      char* const next = buf_of(bi + 1);
      if constexpr (decltype(mask_tag)::value) {
        swa2_for<0, PUTS>([&](auto jc) __attribute__((always_inline)) { put8(next, jc); });
        chunk(i, buf_of(bi), mask_tag, [](auto) __attribute__((always_inline)) {});
      } else {
        chunk(i, buf_of(bi), mask_tag, [&](auto kc) __attribute__((always_inline)) {
          constexpr int k = decltype(kc)::value, every = NKB * 2 * KC / PUTS;
          if constexpr (k % every == every - 1 && k / every < PUTS) put8(next, std::integral_constant<int, k / every>{});
        });
      }
      if (i + 2 < i_end) fetch8(i + 2);
      bi = bi + 1 == NBUF ? 0 : bi + 1;
      it++;
      __syncthreads();
      return;
    }
    const bool more = i + AHEAD * GR < i_end;
    if (more) issue(i + AHEAD * GR, buf_of(bi + AHEAD), lookup(i + AHEAD * GR));
    if (GR == 1 || !decltype(mask_tag)::value || i < i_end) chunk(i, buf_of(bi), mask_tag, [](auto) __attribute__((always_inline)) {});
    if (more) flashd_wait_copies<(AHEAD - 1) * PER_CHUNK>();
    else swa2_wait_copies();
    bi = bi + 1 == NBUF ? 0 : bi + 1;
    it++;
    if (i + GR < i_end) settle(i + GR, buf_of(bi));
    if constexpr (NW > 1) __syncthreads();   // a group of one wave has its buffers to itself
  };
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    while (it < stop) step(std::true_type{});
    if (it >= rounds) break;
#pragma unroll 1
    while (it < r1) step(std::false_type{});
    stop = rounds;
  }

  // ---- epilogue
  float lt[NP], inv[NP];
  unsigned odd[NP];   // rows of the wave to be taken again
#pragma unroll
  for (int p = 0; p < NP; p++) lt[p] = wave_sum4(acc_l[p][0]);
  if constexpr (GR > 1) {
    // every lane of the other groups leaves its registers for the same lane of group 0
    constexpr int PER = NP * (VB * 16 + 8) * 64;   // bytes of a wave
    __syncthreads();
    char* mine = smem + ((grp - 1) * NW + wave) * PER + 16 * lane;
    if (grp > 0) {
#pragma unroll
      for (int p = 0; p < NP; p++) {
#pragma unroll
        for (int d = 0; d < VB; d++) *reinterpret_cast<f32x4*>(mine + (p * VB + d) * 1024) = acc[p][d];
        *reinterpret_cast<float2*>(smem + ((grp - 1) * NW + wave) * PER + NP * VB * 1024 + p * 512 + 8 * lane) = float2{m_run[p], lt[p]};
      }
    }
    __syncthreads();
    if (grp == 0) {
#pragma unroll 1
      for (int o = 0; o < GR - 1; o++) {
        const char* theirs = smem + (o * NW + wave) * PER;
#pragma unroll
        for (int p = 0; p < NP; p++) {
          const float2 x = *reinterpret_cast<const float2*>(theirs + NP * VB * 1024 + p * 512 + 8 * lane);
          float f1, f2;
          flash_merge(m_run[p], x.x, scale, f1, f2);
          lt[p] = flash_add(lt[p], f1, x.y, f2);
#pragma unroll
          for (int d = 0; d < VB; d++) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(theirs + (p * VB + d) * 1024 + 16 * lane);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[p][d][i] = flash_add(acc[p][d][i], f1, v[i], f2);
          }
        }
      }
    }
  }
#pragma unroll
  for (int p = 0; p < NP; p++) {
    const int r = wq0 + 16 * p + n;   // rows behind the last query: zeros
    inv[p] = r < n_rows ? band_inverse(lt[p], sq.off + band_row(a, r).tok) : 0.f;
    // these (pages) went through the products with P = 0 or 1: what an infinite or NaN key or value left there a factor of 0 would not clear
    if constexpr (PAGED)
#pragma unroll
      for (int d = 0; d < VB; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[p][d][i] = r < n_rows ? acc[p][d][i] : 0.f;
    const uint64_t bad = __builtin_amdgcn_ballot_w64(grp == 0 && wq0 + 16 * p + n < n_rows && (band_odd_row(acc, p) || band_odd(lt[p])));
    odd[p] = (unsigned)((bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffff);
  }
  const int64_t row0 = (int64_t)bh * a.rows;
  if (a.shares > 1) {
    if (grp != 0) return;
    const int64_t at = ((int64_t)bh * a.shares + share) * a.rows;
    float* part = a.part + at * a.dv_;
    float* ml = a.part + (int64_t)a.B * a.Hkv * a.shares * a.rows * a.dv_ + 2 * at;
    flash_share_put<NP>(part, acc, a.dv_, wq0 + n, n_rows, g);
#pragma unroll
    for (int p = 0; p < NP; p++)
      if (g == 0 && wq0 + 16 * p + n < n_rows) *reinterpret_cast<float2*>(ml + 2 * (wq0 + 16 * p + n)) = float2{m_run[p] * scale, lt[p]};
#pragma unroll 1
    for (int p = 0; p < NP; p++)
      for (unsigned todo = odd[p]; todo != 0; todo &= todo - 1) {
        const int r = wq0 + 16 * p + __builtin_ctz(todo);
        float m, l, o2[2];
        band_fwd_exact<TIO, PAGED, CK, F8>(a, h, band_row_ptr(qb, a.qs, a, r), reinterpret_cast<const TIO*>(kh), reinterpret_cast<const TIO*>(vh), pages, W, i_beg, i_end, sq.off + band_row(a, r).tok, sq.n_k, lane, m, l, o2);
        __threadfence();   // behind the wave's own stores of the row
        if (2 * lane < a.dv_) *reinterpret_cast<float2*>(part + (int64_t)r * a.dv_ + 2 * lane) = float2{o2[0], o2[1]};
        if (lane == 0) *reinterpret_cast<float2*>(ml + 2 * r) = float2{m, l};
      }
    return;
  }
  if (a.lse != nullptr) {
#pragma unroll
    for (int p = 0; p < NP; p++) {
      const int r = wq0 + 16 * p + n;
      if (grp == 0 && g == 0 && r < n_rows && (odd[p] >> n & 1) == 0) store_stream4(a.lse + row0 + r, m_run[p] * scale + fast_log2(lt[p]));
    }
  }
  __syncthreads();
  TIO* ob = reinterpret_cast<TIO*>(a.out) + b * a.os[0] + (int64_t)h * a.G * a.os[1];
  constexpr int PT = D * 2 + 16;
  // odd rows of the wave once more: o, or (`low`) what its rounding drops
  auto again = [&](bool low) __attribute__((always_inline)) {
#pragma unroll 1
    for (int p = 0; p < NP; p++)
      for (unsigned todo = odd[p]; todo != 0; todo &= todo - 1) {
        const int w = 16 * p + __builtin_ctz(todo), r = wq0 + w;
        float m, l, o2[2];
        band_fwd_exact<TIO, PAGED, CK, F8>(a, h, band_row_ptr(qb, a.qs, a, r), reinterpret_cast<const TIO*>(kh), reinterpret_cast<const TIO*>(vh), pages, W, i_beg, i_end, sq.off + band_row(a, r).tok, sq.n_k, lane, m, l, o2);
        const float f = band_inverse(l, sq.off + band_row(a, r).tok);
#pragma unroll
        for (int j = 0; j < 2; j++) o2[j] = low ? band_dropped<TIO>(o2[j] * f) : o2[j] * f;
        if (2 * lane < D) *reinterpret_cast<unsigned*>(smem + (wave * 16 * NP + w) * PT + 4 * lane) = pack2<TIO>(o2[0], o2[1]);
        if (lane == 0 && !low && a.lse != nullptr) a.lse[row0 + r] = m + fast_log2(l);
      }
  };
  band_store_rows<D, NP, TIO>(smem, acc, inv, NW, GR, grp == 0, a.dv_, wave, n, g, tid,
                              [&](int row) -> TIO* { return x0 + row < a.rows ? band_row_ptr(ob, a.os, a, x0 + row) : nullptr; }, [&]() { again(false); });
  if (!PAGED && a.low != nullptr && x0 < a.low_rows)
    band_store_rows<D, NP, TIO, true>(smem, acc, inv, NW, GR, grp == 0, a.dv_, wave, n, g, tid,
                                      [&](int row) -> TIO* { return x0 + row < a.rows ? band_low<TIO>(a, b, h, x0 + row) : nullptr; }, [&]() { again(true); });
}
