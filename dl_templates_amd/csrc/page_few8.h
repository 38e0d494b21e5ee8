// Attention of few rows (a decode step: the G heads of a group times up to a few tokens, at most 32) over a cache of pages in 8 bits, for gfx950.
//
// Bound by the cache's bytes.  A wave takes tiles of 32 tokens (64 at D = 64) by itself: K and V go from memory to its registers, the next tile while this one is
// worked on, and nothing passes through LDS or waits for another wave.  S^T = K Q^T: a lane's 8-bit numbers are a run of a token's dims, which become an operand as they are
// converted (the order of the dims is free as long as q has it too).  P^T leaves that product as the operand of the next one, O^T += V^T P^T, whose other operand wants the
// tokens of a dim side by side: a lane fetches the same few dims of 8 tokens, and 4 x 4 bytes are turned with 8 byte permutes.  Conversions are a tenth of the vector issue
// slots that the bytes' time leaves.
// P enters its product in two parts, its rounding and the rest, which costs 8 matrix instructions of 24 that nothing waits for: the only rounding to 16 bits is the
// output's (relative error 0.0024 -> 0.0017 in bf16, that of the output's rounding).
//
// Work is cut by what the lengths say, on the device: a step is a tile for each of a workgroup's four waves, the steps of all sequences and heads form one row, and every
// workgroup takes an equal run of it.  A run may end a head, hold some and begin another; heads that one run holds whole are finished there, parts of the others are
// added by a second launch.  Runs, parts and sums follow from the lengths alone: equal calls give equal bits.
#pragma once
#include "band_fwd_kernel.h"
#include "page_few8_shapes.h"

template <int D>
struct Few8 {
  static constexpr int NT = D == 128 ? 1 : 2, TK = 32 * NT, NG = 2 * NT;   // 32-token products, tokens and 16-token groups of a tile
  static constexpr int VB = D / 16, KC = D / 32, VW = D / 64;              // blocks of 16 output dims, of 32 head dims; dwords of a lane's V per token
  static constexpr int BATCH = 64 / NG;                                    // tiles whose pages a wave looks up at once
  static constexpr int WAVE_LDS = VB * 1024 + 256;                         // results of 16 rows of a wave: sums of products; {maximum, sum}
};
// chunks of a sequence that its rows see
template <int TK>
DLT_DEV void few8_walk(const Band8Args& a, const BandSeq& sq, BandWalk<TK>& W, int& first, int& last) {
  const int rows = sq.n_q * a.G;
  first = sq.off;
  last = rows > 0 ? dlt_imin(sq.off + band_row(a, rows - 1).tok, sq.n_k - 1) : -1;
  W.init(first, last, a.W, a.S);
}
template <int TK>
DLT_DEV int few8_steps(const Band8Args& a, int b) {
  BandWalk<TK> W;
  int first, last;
  few8_walk(a, band_seq<true>(a, b), W, first, last);
  return dlt_imax((W.n + 3) >> 2, 1);
}

// bytes (i, j) of 4 dwords -> (j, i)
DLT_DEV void few8_turn(const unsigned (&r)[4], unsigned (&t)[4]) {
  const unsigned x0 = __builtin_amdgcn_perm(r[1], r[0], 0x05010400), x1 = __builtin_amdgcn_perm(r[1], r[0], 0x07030602);
  const unsigned y0 = __builtin_amdgcn_perm(r[3], r[2], 0x05010400), y1 = __builtin_amdgcn_perm(r[3], r[2], 0x07030602);
  t[0] = __builtin_amdgcn_perm(y0, x0, 0x05040100);
  t[1] = __builtin_amdgcn_perm(y0, x0, 0x07060302);
  t[2] = __builtin_amdgcn_perm(y1, x1, 0x05040100);
  t[3] = __builtin_amdgcn_perm(y1, x1, 0x07060302);
}

// A tile on its way or there
template <int D>
struct Few8Tile {
  typedef Few8<D> F;
  unsigned k[F::NG][D / 16], v[F::NG][4][F::VW];
  int ek[F::NG], ev[F::NG], tok[F::NG];   // wave-uniform: scales, first token of each group
};

// FULL: both tensors have D dims, K's rows lie at multiples of 16 bytes.  BAL: workgroups take runs of all steps, else one (batch, kv head) each.
template <typename TIO, int D, int NP, int FMT, bool FULL, bool BAL>
__global__ __launch_bounds__(256, NP == 1 ? 2 : 1) void few8_kernel(const Few8Args a) {
  dlt_kernargs_in<sizeof(Few8Args)>();
  typedef Few8<D> F;
  constexpr int NG = F::NG, VB = F::VB, KC = F::KC, VW = F::VW, TK = F::TK;
  extern __shared__ __align__(16) char smem[];   // results of the waves; BAL: behind them the steps in front of each sequence
  __shared__ unsigned odd_rows[NP];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // the run of steps of this workgroup
  int u0 = 0, u1 = 1, per = 1, rem = 0;
  int32_t* before = reinterpret_cast<int32_t*>(smem + 4 * NP * F::WAVE_LDS);
  if constexpr (BAL) {
    __shared__ int part[4];
    const int each = (a.B + 255) >> 8, b0 = dlt_imin(tid * each, a.B), b1 = dlt_imin(b0 + each, a.B);
    int x = 0;
    for (int b = b0; b < b1; b++) {
      const int s = few8_steps<TK>(a, b);
      before[b] = s;
      x += s;
    }
    int sum = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(sum, d);
      if (lane >= d) sum += y;
    }
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    int total = 0, base = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      if (w < wave) base += part[w];
      total += part[w];
    }
    base += sum - x;
    for (int b = b0; b < b1; b++) {
      const int s = before[b];
      before[b] = base;
      base += s;
    }
    if (tid == 0) before[a.B] = total;
    __syncthreads();
    total *= a.Hkv;
    const int wgs = dlt_imax(1, dlt_imin((int)gridDim.x, total / a.least));
    if ((int)blockIdx.x >= wgs) return;
    per = total / wgs;
    rem = total - per * wgs;
    u0 = blockIdx.x * per + dlt_imin(blockIdx.x, rem);
    u1 = u0 + per + ((int)blockIdx.x < rem ? 1 : 0);
  }

  const float scale = a.scale_log2;
  const unsigned one2 = pack2<TIO>(1.f, 1.f);
  const u32x4 ones = n == 0 ? u32x4{one2, one2, one2, one2} : u32x4{0u, 0u, 0u, 0u};

#pragma unroll 1
  for (int u = u0; u < u1;) {
    // (batch, kv head) and its steps [s0, s1) of `steps`
    int bh = blockIdx.x, b, h, s0 = 0, s1, steps;
    if constexpr (BAL) {
      int lo = 0, hi = a.B;
      const int q = u;   // the last b whose steps begin at or before u
      while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (before[m] * a.Hkv <= q) lo = m;
        else hi = m;
      }
      b = __builtin_amdgcn_readfirstlane(lo);
      const int first_u = __builtin_amdgcn_readfirstlane(before[b]) * a.Hkv;
      steps = __builtin_amdgcn_readfirstlane(before[b + 1]) - __builtin_amdgcn_readfirstlane(before[b]);
      h = (u - first_u) / steps;
      s0 = u - first_u - h * steps;
      s1 = dlt_imin(steps, s0 + u1 - u);
      bh = b * a.Hkv + h;
    } else {
      b = band_div(bh, a.by_heads);
      h = bh - b * a.Hkv;
      steps = s1 = 1;
    }
    const BandSeq sq = band_seq<true>(a, b);
    BandWalk<TK> W;
    int first, last;
    few8_walk(a, sq, W, first, last);
    const int t0 = BAL ? 4 * s0 : 0, t1 = BAL ? dlt_imin(4 * s1, W.n) : W.n;
    const int n_rows = sq.n_q * a.G;
    const int32_t* pages = a.pg.table + b * a.pg.ts;
    const uint8_t* kh = reinterpret_cast<const uint8_t*>(a.k) + h * a.ks[1];
    const uint8_t* vh = reinterpret_cast<const uint8_t*>(a.v) + h * a.vs[1];
    const uint8_t *ksc = a.k_sc + h * a.kss[1], *vsc = a.v_sc + h * a.vss[1];
    const TIO* qb = reinterpret_cast<const TIO*>(a.q) + b * a.qs[0] + (int64_t)h * a.G * a.qs[1];

    // pages and scales of the wave's next BATCH tiles: a group of 16 tokens to a lane
    int pg_l = 0, in_l = 0, ek_l = 127, ev_l = 127;
    auto look = [&](int tile) __attribute__((always_inline)) {   // `tile`: the first of them
      const int t = tile + 4 * (lane / NG);
      const int tok = dlt_imin(W.tok(TK * dlt_imin(t, dlt_imax(W.n - 1, 0)) + 16 * (lane % NG)), sq.n_k - 1);
      pg_l = band_page(a.pg, pages, dlt_imax(tok, 0) >> 4, in_l);
      const int blk = (int)dlt_fastdiv((uint32_t)in_l, a.mB, a.sB);
      ek_l = ksc[pg_l * a.kss[0] + blk * a.kss[2]];
      ev_l = vsc[pg_l * a.vss[0] + blk * a.vss[2]];
    };
    const uint32_t ko = FULL ? (uint32_t)n * (uint32_t)a.ks[2] + 16u * g : (uint32_t)n * (uint32_t)a.ks[2] + 8u * g;
    const uint32_t vo = (uint32_t)(4 * g) * (uint32_t)a.vs[2] + (uint32_t)(4 * VW) * n;
    auto fetch = [&](Few8Tile<D>& x, int tile, int at) __attribute__((always_inline)) {   // the at-th of the batch
#pragma unroll
      for (int u2 = 0; u2 < NG; u2++) {
        const int l = at * NG + u2;
        const int page = __builtin_amdgcn_readlane(pg_l, l), row = 16 * __builtin_amdgcn_readlane(in_l, l);
        x.ek[u2] = __builtin_amdgcn_readlane(ek_l, l);
        x.ev[u2] = __builtin_amdgcn_readlane(ev_l, l);
        x.tok[u2] = W.tok(TK * tile + 16 * u2);
        const uint8_t* kp = kh + (page * a.ks[0] + row * a.ks[2]);
        const uint8_t* vp = vh + (page * a.vs[0] + row * a.vs[2]);
        if constexpr (FULL) {
#pragma unroll
          for (int c = 0; c < D / 64; c++) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(kp + (ko + 64u * c));
#pragma unroll
            for (int i = 0; i < 4; i++) x.k[u2][4 * c + i] = w[i];
          }
        } else {
#pragma unroll
          for (int c = 0; c < D / 32; c++) {
            u32x2 w = {0u, 0u};
            if (32 * c + 8 * g < a.dk_) w = *reinterpret_cast<const u32x2*>(kp + (ko + 32u * c));
            x.k[u2][2 * c] = w[0];
            x.k[u2][2 * c + 1] = w[1];
          }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint8_t* p = vp + j * a.vs[2];
          if constexpr (VW == 2) {
            u32x2 w = {0u, 0u};
            if (FULL || 8 * n < a.dv_) w = *reinterpret_cast<const u32x2*>(p + vo);
            x.v[u2][j][0] = w[0];
            x.v[u2][j][VW - 1] = w[1];
          } else {
            x.v[u2][j][0] = 0u;
            if (FULL || 4 * n < a.dv_) x.v[u2][j][0] = *reinterpret_cast<const unsigned*>(p + vo);
          }
        }
      }
    };

    Few8Tile<D> xa, xb;
    const int tw = t0 + wave, tiles = tw < t1 ? (t1 - tw + 3) >> 2 : 0;   // the wave's tiles: tw, tw + 4, ..
    if (tiles > 0) {
      look(tw);
      fetch(xa, tw, 0);
    }
    u32x4 qf[NP][KC];
    int hi[NP], lo[NP];   // the row sees tokens lo < x <= hi, and the sinks
#pragma unroll
    for (int p = 0; p < NP; p++) {
      const int r = 16 * p + n;
      const bool on = r < n_rows;
      const int pos = sq.off + band_row(a, on ? r : 0).tok;
      hi[p] = on ? dlt_imin(pos, sq.n_k - 1) : -1;
      lo[p] = pos - a.W;
      const TIO* row = band_row_ptr(qb, a.qs, a, on ? r : 0);
#pragma unroll
      for (int c = 0; c < KC; c++) {
        const int d = FULL ? 16 * (g + 4 * (c >> 1)) + 8 * (c & 1) : 32 * c + 8 * g;
        qf[p][c] = u32x4{0u, 0u, 0u, 0u};
        if (on && (FULL || d < a.dk_)) qf[p][c] = *reinterpret_cast<const u32x4*>(row + d);
      }
    }
    float m_run[NP];
    f32x4 acc[NP][VB], acc_l[NP];
#pragma unroll
    for (int p = 0; p < NP; p++) {
      m_run[p] = -INFINITY;
      acc_l[p] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < VB; d++) acc[p][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    auto consume = [&](Few8Tile<D>& x, auto mask_tag) __attribute__((always_inline)) {
      constexpr bool MASK = decltype(mask_tag)::value;
      float t[NP][NG][4];
#pragma unroll
      for (int u2 = 0; u2 < NG; u2++) {
        f32x4 s[NP];
        const float sc = cvt8_scale(x.ek[u2]);
#pragma unroll
        for (int c = 0; c < KC; c++) {
          const u32x4 op = cvt8_eight<FMT, TIO>(x.k[u2][2 * c], x.k[u2][2 * c + 1], sc);
#pragma unroll
          for (int p = 0; p < NP; p++) s[p] = Mma<TIO>::mfma(op, qf[p][c], c == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[p]);
        }
#pragma unroll
        for (int p = 0; p < NP; p++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int at = x.tok[u2] + 4 * g + i;
            t[p][u2][i] = !MASK || (at <= hi[p] && (at > lo[p] || at < a.S)) ? s[p][i] : -INFINITY;
          }
      }
      u32x4 ph[NP][F::NT], pl[NP][F::NT];
#pragma unroll
      for (int p = 0; p < NP; p++) {
        float mx = -INFINITY;
#pragma unroll
        for (int u2 = 0; u2 < NG; u2++)
#pragma unroll
          for (int i = 0; i < 4; i++) mx = fmaxf(mx, t[p][u2][i]);
        mx = wave_max4(mx);
        // the reference maximum moves when a score exceeds it by more than 2^8 after scaling: P stays below 2^8
        if (__builtin_amdgcn_ballot_w64((mx - m_run[p]) * scale > 8.f)) {
          keep_branch();
          const float m_new = fmaxf(m_run[p], mx);
          const float alpha = m_run[p] == -INFINITY ? 0.f : fast_exp2((m_run[p] - m_new) * scale);
          const float al = m_new == -INFINITY ? 1.f : alpha;
          m_run[p] = m_new;
#pragma unroll
          for (int d = 0; d < VB; d++) acc[p][d] *= al;
          acc_l[p] *= al;
        }
        const float neg = m_run[p] == -INFINITY ? 0.f : -m_run[p] * scale;
#pragma unroll
        for (int kb = 0; kb < F::NT; kb++) {
          float e[8], r[8];
#pragma unroll
          for (int i = 0; i < 8; i++) e[i] = fast_exp2(fmaf(t[p][2 * kb + (i >> 2)][i & 3], scale, neg));
          ph[p][kb] = pack8<TIO>(e);
          unpack8<TIO>(ph[p][kb], r);
#pragma unroll
          for (int i = 0; i < 8; i++) r[i] = e[i] - r[i];
          pl[p][kb] = pack8<TIO>(r);
          acc_l[p] = Mma<TIO>::mfma(ones, ph[p][kb], acc_l[p]);
          acc_l[p] = Mma<TIO>::mfma(ones, pl[p][kb], acc_l[p]);
        }
      }
      if constexpr (MASK) {   // pages hold anything behind the last key: those values, which no row sees, are cleared, and so are scales of blocks of nothing else
#pragma unroll
        for (int u2 = 0; u2 < NG; u2++) {
          if (x.tok[u2] >= sq.n_k) x.ev[u2] = 127;
#pragma unroll
          for (int j = 0; j < 4; j++)
#pragma unroll
            for (int w = 0; w < VW; w++) x.v[u2][j][w] = x.tok[u2] + 4 * g + j < sq.n_k ? x.v[u2][j][w] : 0u;
        }
      }
#pragma unroll
      for (int kb = 0; kb < F::NT; kb++)
#pragma unroll
        for (int w = 0; w < VW; w++) {
          unsigned r0[4], r1[4], c0[4], c1[4];
#pragma unroll
          for (int j = 0; j < 4; j++) { r0[j] = x.v[2 * kb][j][w]; r1[j] = x.v[2 * kb + 1][j][w]; }
          few8_turn(r0, c0);
          few8_turn(r1, c1);
          const float sc0 = cvt8_scale(x.ev[2 * kb]), sc1 = cvt8_scale(x.ev[2 * kb + 1]);
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const u32x4 op = u32x4{cvt8_pair<FMT, TIO>(c0[c], sc0, false), cvt8_pair<FMT, TIO>(c0[c], sc0, true), cvt8_pair<FMT, TIO>(c1[c], sc1, false),
                                   cvt8_pair<FMT, TIO>(c1[c], sc1, true)};
#pragma unroll
            for (int p = 0; p < NP; p++) {
              acc[p][4 * w + c] = Mma<TIO>::mfma(op, ph[p][kb], acc[p][4 * w + c]);
              acc[p][4 * w + c] = Mma<TIO>::mfma(op, pl[p][kb], acc[p][4 * w + c]);
            }
          }
        }
    };
    // every row sees the whole tile
    auto whole = [&](const Few8Tile<D>& x) __attribute__((always_inline)) {
      const int end = x.tok[NG - 1] + 15;
      return end <= first && (x.tok[0] > last - a.W || end < a.S);
    };
    auto work = [&](Few8Tile<D>& x) __attribute__((always_inline)) {
      if (whole(x)) consume(x, std::false_type{});
      else consume(x, std::true_type{});
    };
    int at = 0;   // of the batch, of the tile that is fetched last
#pragma unroll 1
    for (int i = 0; i < tiles; i += 2) {
      auto next = [&](Few8Tile<D>& y, int k) __attribute__((always_inline)) {
        if (k >= tiles) return;
        at++;
        if (at == F::BATCH) {
          at = 0;
          look(tw + 4 * k);
        }
        fetch(y, tw + 4 * k, at);
      };
      next(xb, i + 1);
      __builtin_amdgcn_sched_barrier(0);
      work(xa);
      if (i + 1 >= tiles) break;
      next(xa, i + 2);
      __builtin_amdgcn_sched_barrier(0);
      work(xb);
    }

    // ---- the four waves' results, joined: each takes a quarter of the blocks of output dims
    if (tid < NP) odd_rows[tid] = 0u;
#pragma unroll
    for (int p = 0; p < NP; p++) {
      char* mine = smem + (wave * NP + p) * F::WAVE_LDS;
#pragma unroll
      for (int d = 0; d < VB; d++) *reinterpret_cast<f32x4*>(mine + 1024 * d + 16 * lane) = acc[p][d];
      const float l = wave_sum4(acc_l[p][0]);
      if (g == 0) *reinterpret_cast<float2*>(mine + 1024 * VB + 8 * n) = float2{m_run[p] * scale, l};
    }
    __syncthreads();
    constexpr int OB = VB / 4;
    f32x4 o[NP][OB];
    float om[NP], ol[NP];
#pragma unroll
    for (int p = 0; p < NP; p++) {
      float2 x[4];
      om[p] = -INFINITY;
      ol[p] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; w++) {
        x[w] = *reinterpret_cast<const float2*>(smem + (w * NP + p) * F::WAVE_LDS + 1024 * VB + 8 * n);
        om[p] = fmaxf(om[p], x[w].x);
      }
#pragma unroll
      for (int d = 0; d < OB; d++) o[p][d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; w++) {
        const float f = x[w].x == -INFINITY ? (x[w].y == 0.f ? 0.f : 1.f) : fast_exp2(x[w].x - om[p]);
        ol[p] = fmaf(x[w].y, f, ol[p]);
#pragma unroll
        for (int d = 0; d < OB; d++) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(smem + (w * NP + p) * F::WAVE_LDS + 1024 * (OB * wave + d) + 16 * lane);
#pragma unroll
          for (int i = 0; i < 4; i++) o[p][d][i] = fmaf(v[i], f, o[p][d][i]);
        }
      }
      bool bad = band_odd(ol[p]);
#pragma unroll
      for (int d = 0; d < OB; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) bad = bad || band_odd(o[p][d][i]);
      const uint64_t ball = __builtin_amdgcn_ballot_w64(bad && 16 * p + n < n_rows);
      const unsigned bits = (unsigned)((ball | ball >> 16 | ball >> 32 | ball >> 48) & 0xffff);
      if (lane == 0 && bits != 0) atomicOr(&odd_rows[p], bits);
    }
    __syncthreads();
    unsigned odd[NP];
#pragma unroll
    for (int p = 0; p < NP; p++) odd[p] = __builtin_amdgcn_readfirstlane(odd_rows[p]);

    const bool all = !BAL || (s0 == 0 && s1 == steps);
    // block d of the wave holds, of row n, dims VSTEP (4 g + i) + OB wave + d
    constexpr int VSTEP = 4 * VW;
    if (all) {
      TIO* ob = reinterpret_cast<TIO*>(a.out) + b * a.os[0] + (int64_t)h * a.G * a.os[1];
#pragma unroll
      for (int p = 0; p < NP; p++) {
        const int r = 16 * p + n;
        if (r >= a.rows || (odd[p] >> n & 1) != 0) continue;
        const float inv = r < n_rows ? band_inverse(ol[p], hi[p]) : 0.f;
        TIO* row = band_row_ptr(ob, a.os, a, r);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int d0 = VSTEP * (4 * g + i) + OB * wave;
          if (d0 >= a.dv_) continue;
          if constexpr (OB == 2) {
            const float v0 = r < n_rows ? o[p][0][i] * inv : 0.f, v1 = r < n_rows ? o[p][OB - 1][i] * inv : 0.f;
            *reinterpret_cast<unsigned*>(row + d0) = pack2<TIO>(v0, v1);
          } else {
            row[d0] = (TIO)(r < n_rows ? o[p][0][i] * inv : 0.f);
          }
        }
      }
    }
    float* part = nullptr;
    float2* ml = nullptr;
    if constexpr (BAL) {
      // a run's first head may have begun in an earlier run (slot 2 w), its last one may go on (slot 2 w + 1)
      const int64_t slot = 2 * (int64_t)blockIdx.x + (s0 == 0 ? 1 : 0);
      part = a.part + slot * a.rows * a.dv_;
      ml = reinterpret_cast<float2*>(a.part + 2 * (int64_t)gridDim.x * a.rows * a.dv_) + slot * a.rows;
      if (s0 == 0 && tid == 0) {
        const int e = u + steps - 1, big = rem * (per + 1);   // the last step of the head, and its workgroup
        const int w = e < big ? e / (per + 1) : rem + (e - big) / per;
        *reinterpret_cast<int2*>(a.meta + 2 * bh) = int2{(int)blockIdx.x, w - (int)blockIdx.x + 1};
      }
      if (!all) {
#pragma unroll
        for (int p = 0; p < NP; p++) {
          const int r = 16 * p + n;
          if (r >= n_rows || (odd[p] >> n & 1) != 0) continue;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int d0 = VSTEP * (4 * g + i) + OB * wave;
            if (d0 >= a.dv_) continue;
            if constexpr (OB == 2) *reinterpret_cast<float2*>(part + (int64_t)r * a.dv_ + d0) = float2{o[p][0][i], o[p][OB - 1][i]};
            else part[(int64_t)r * a.dv_ + d0] = o[p][0][i];
          }
          if (wave == 0 && g == 0) ml[r] = float2{om[p], ol[p]};
        }
      }
    }
    // rows whose sums came out infinite or NaN, once more over the keys that each sees, a wave to a row
#pragma unroll 1
    for (int p = 0; p < NP; p++)
      for (unsigned todo = odd[p]; todo != 0; todo &= todo - 1) {
        const int r = 16 * p + __builtin_ctz(todo);
        if ((r & 3) != wave) continue;
        const int pos = sq.off + band_row(a, r).tok;
        float m, l, o2[2];
        band_fwd_exact<TIO, true, TK, FMT + 1>(a, h, band_row_ptr(qb, a.qs, a, r), reinterpret_cast<const TIO*>(kh), reinterpret_cast<const TIO*>(vh), pages, W, t0, t1, pos,
                                               sq.n_k, lane, m, l, o2);
        if (2 * lane < a.dv_) {
          if (all) {
            const float f = band_inverse(l, pos);
            TIO* row = band_row_ptr(reinterpret_cast<TIO*>(a.out) + b * a.os[0] + (int64_t)h * a.G * a.os[1], a.os, a, r);
            *reinterpret_cast<unsigned*>(row + 2 * lane) = pack2<TIO>(o2[0] * f, o2[1] * f);
          } else {
            *reinterpret_cast<float2*>(part + (int64_t)r * a.dv_ + 2 * lane) = float2{o2[0], o2[1]};
          }
        }
        if (!all && lane == 0) ml[r] = float2{m, l};
      }
    u += s1 - s0;
    if (BAL && u < u1) __syncthreads();   // the waves' results have been read
  }
}

// Rows of heads that several runs hold: their parts, in order.  A workgroup to a row: every wave takes every fourth part.
template <typename TIO>
__global__ __launch_bounds__(256) void few8_join_kernel(const Few8Args a) {
  dlt_kernargs_in<sizeof(Few8Args)>();
  __shared__ float sum[4][128], big[4], len[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int bh = blockIdx.y, r = blockIdx.x, b = band_div(bh, a.by_heads), h = bh - b * a.Hkv;
  const int2 who = *reinterpret_cast<const int2*>(a.meta + 2 * bh);
  if (who.y <= 1) return;
  const BandSeq sq = band_seq<true>(a, b);
  const bool on = r < sq.n_q * a.G;
  const int64_t first = 2 * (int64_t)who.x + 1;   // slots first, first + 1, first + 3, first + 5, ..
  auto slot = [&](int i) { return first + (i == 0 ? 0 : 2 * i - 1); };
  const float2* ml = reinterpret_cast<const float2*>(a.part + 2 * (int64_t)a.wgs * a.rows * a.dv_);
  float m = -INFINITY;
  if (on)
    for (int i = threadIdx.x; i < who.y; i += 256) m = fmaxf(m, ml[slot(i) * a.rows + r].x);
  m = band_wave_max(m);
  if (lane == 0) big[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3]));
  float l = 0.f, o0 = 0.f, o1 = 0.f;
  if (on) {
    const int d = 2 * dlt_imin(lane, a.dv_ / 2 - 1);
    for (int i0 = wave; i0 < who.y; i0 += 32) {
      float2 v[8], x[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int64_t s = slot(dlt_imin(i0 + 4 * k, who.y - 1));
        x[k] = ml[s * a.rows + r];
        v[k] = *reinterpret_cast<const float2*>(a.part + (s * a.rows + r) * a.dv_ + d);
      }
#pragma unroll
      for (int k = 0; k < 8; k++) {
        if (i0 + 4 * k >= who.y) break;
        // with a weight of 0 too: an infinite or NaN part holds such a value of a key that the row sees
        const float f = x[k].x == -INFINITY ? (x[k].y == 0.f ? 0.f : 1.f) : fast_exp2(x[k].x - m);
        l = fmaf(x[k].y, f, l);
        o0 = fmaf(v[k].x, f, o0);
        o1 = fmaf(v[k].y, f, o1);
      }
    }
  }
  sum[wave][2 * lane] = o0;
  sum[wave][2 * lane + 1] = o1;
  if (lane == 0) len[wave] = l;
  __syncthreads();
  if (wave != 0) return;
  l = ((len[0] + len[1]) + len[2]) + len[3];
  o0 = ((sum[0][2 * lane] + sum[1][2 * lane]) + sum[2][2 * lane]) + sum[3][2 * lane];
  o1 = ((sum[0][2 * lane + 1] + sum[1][2 * lane + 1]) + sum[2][2 * lane + 1]) + sum[3][2 * lane + 1];
  const float f = on ? band_inverse(l, dlt_imin(sq.off + band_row(a, r).tok, sq.n_k - 1)) : 0.f;
  TIO* p = band_row_ptr(reinterpret_cast<TIO*>(a.out) + b * a.os[0] + (int64_t)h * a.G * a.os[1], a.os, a, r);
  if (2 * lane < a.dv_) *reinterpret_cast<unsigned*>(p + 2 * lane) = on ? pack2<TIO>(o0 * f, o1 * f) : 0u;
}
