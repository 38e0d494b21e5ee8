// Attention of few rows (a decode step: the G heads of a group times up to a few tokens, at most 32) over a cache of pages in 8 bits, for gfx950.
//
// Bound by the cache's bytes.  A wave takes tiles of 32 tokens (64 at D = 64) by itself: K and V go from memory to its registers, the next tile while this one is
// worked on, and nothing passes through LDS or waits for another wave.  S^T = K Q^T: a lane's 8-bit numbers are a run of a token's dims, which become an operand as they are
// converted (the order of the dims is free as long as q has it too).  P^T leaves that product as the operand of the next one, O^T += V^T P^T, whose other operand wants the
// tokens of a dim side by side: a lane fetches the same few dims of 8 tokens, and 4 x 4 bytes are turned with 8 byte permutes.  A tile is 12 loads of a lane, 24 matrix
// instructions and about 250 vector ones at D = 128, a third of the time that its 8 KB take at the rate of memory.
// P enters its product in two parts, its rounding and the rest, which costs 8 matrix instructions of 24 that nothing waits for: the only rounding to 16 bits is the
// output's (relative error 0.0024 -> 0.0017 in bf16, that of the output's rounding).
//
// Work is cut by what the lengths say, on the device: a step is a tile for each of a workgroup's four waves, and every (batch, kv head) is taken by as many workgroups as it
// has runs of `target` steps, so that all sequences together make about as many runs as the chip wants.  Heads of one run are finished there; parts of the others are
// added by a second launch.  Every wave finds its workgroup's run from the lengths by itself, in registers.  Runs, parts and sums follow from the lengths alone: equal calls
// give equal bits.
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
DLT_DEV int few8_steps(const Band8Args& a, const BandSeq& sq) {
  BandWalk<TK> W;
  int first, last;
  few8_walk(a, sq, W, first, last);
  return dlt_imax((W.n + 3) >> 2, 1);
}
DLT_DEV int few8_ceil(int n, int d) { return (n + d - 1) / d; }
DLT_DEV int few8_scan(int x, int lane) {   // inclusive sums over the wave
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}
// Run `wg` of all: the heads of a sequence one behind the other, the runs of a head.  A lane has `each` sequences in a row; false: there are fewer runs.
template <int TK>
DLT_DEV bool few8_run(const Few8Args& a, int wg, int lane, int& b, int& h, int& run, int& runs, int& s0, int& s1, BandSeq& sq) {
  const int each = (a.B + 63) >> 6, b0 = dlt_imin(lane * each, a.B), b1 = dlt_imin(b0 + each, a.B);
  BandSeq mine = band_seq<true>(a, dlt_imin(b0, a.B - 1));
  int x = b0 < b1 ? few8_steps<TK>(a, mine) : 0;
  const int one = x;
#pragma unroll 1
  for (int i = b0 + 1; i < b1; i++) x += few8_steps<TK>(a, band_seq<true>(a, i));
  const int total = __builtin_amdgcn_readlane(few8_scan(x, lane), 63) * a.Hkv;
  const int target = few8_ceil(total, total < 5 * a.want ? a.want_few : a.want);
  int y = b0 < b1 ? few8_ceil(one, target) : 0;
#pragma unroll 1
  for (int i = b0 + 1; i < b1; i++) y += few8_ceil(few8_steps<TK>(a, band_seq<true>(a, i)), target);
  int upto = few8_scan(y, lane) * a.Hkv;   // runs of the lane's sequences and those before
  uint64_t behind = __builtin_amdgcn_ballot_w64(upto > wg);
  if (behind == 0) return false;
  int at = __builtin_ctzll(behind), base = __builtin_amdgcn_readlane(upto - y * a.Hkv, at);
  b = at;
  if (each > 1) {   // which of that lane's sequences, one to a lane
    const int c0 = at * each, c = c0 + lane;
    mine = band_seq<true>(a, dlt_imin(c, a.B - 1));
    x = lane < each && c < a.B ? few8_steps<TK>(a, mine) : 0;
    y = few8_ceil(x, target);
    upto = base + few8_scan(y, lane) * a.Hkv;
    behind = __builtin_amdgcn_ballot_w64(upto > wg);
    at = __builtin_ctzll(behind);
    base = __builtin_amdgcn_readlane(upto - y * a.Hkv, at);
    b = c0 + at;
  }
  sq.off = __builtin_amdgcn_readlane(mine.off, at);
  sq.n_q = __builtin_amdgcn_readlane(mine.n_q, at);
  sq.n_k = __builtin_amdgcn_readlane(mine.n_k, at);
  const int steps = __builtin_amdgcn_readlane(x, at);
  runs = __builtin_amdgcn_readlane(y, at);
  h = (wg - base) / runs;
  run = wg - base - h * runs;
  // the first steps % runs of them have one step more
  const int len = steps / runs, more = steps - len * runs;
  s0 = run * len + dlt_imin(run, more);
  s1 = s0 + len + (run < more ? 1 : 0);
  return true;
}

// weight of a part with {maximum, sum} beside others, m: the largest maximum.  One that held no key of the row has (-inf, 0); a sum that is infinite or NaN goes through
DLT_DEV float few8_weight(const float2& x, float m) { return x.x == -INFINITY ? (x.y == 0.f ? 0.f : 1.f) : fast_exp2(x.x - m); }

// bytes (i, j) of 4 dwords -> (j, i)
DLT_DEV void few8_turn(const unsigned (&r)[4], unsigned (&t)[4]) {
  const unsigned x0 = __builtin_amdgcn_perm(r[1], r[0], 0x05010400), x1 = __builtin_amdgcn_perm(r[1], r[0], 0x07030602);
  const unsigned y0 = __builtin_amdgcn_perm(r[3], r[2], 0x05010400), y1 = __builtin_amdgcn_perm(r[3], r[2], 0x07030602);
  t[0] = __builtin_amdgcn_perm(y0, x0, 0x05040100);
  t[1] = __builtin_amdgcn_perm(y0, x0, 0x07060302);
  t[2] = __builtin_amdgcn_perm(y1, x1, 0x05040100);
  t[3] = __builtin_amdgcn_perm(y1, x1, 0x07060302);
}

// Whole numbers: P times the scale of its key's values enters its product in bfloat16, whose least numbers are 2^-133; scales go down to 2^-127, and a key's share of a sum to
// far less than its P of 1.  So P is taken times 2^32, and the sums times 2^-32 when they are done: at the least scale a P of 2^-38 still counts.  From scales of about 2^80 on that
// does not fit 32 bits any more: those rows come out infinite or NaN and are formed again one by one, without it.
constexpr int FEW8_LIFT = 32;
DLT_DEV float few8_lifted(int e) { return __uint_as_float((unsigned)dlt_imin(e + FEW8_LIFT, 255) << 23); }   // 255 and beyond the exponents: infinite

// Operands of 8 numbers.  e4m3: one instruction for two, which also takes the scale.  Whole numbers enter the products as they are, exact in both types, and their scales
// multiply scores and P instead; values, and P, enter as bfloat16 whatever q's type is, whose exponents hold every scale (P's two parts keep 16 bits of it).
DLT_DEV unsigned few8_ints_bf16(unsigned w, bool hi) {   // whole numbers in 32 bits have no bits set below bfloat16's
  const float x = (float)(int8_t)(hi ? w >> 16 : w), y = (float)(int8_t)(hi ? w >> 24 : w >> 8);
  return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302);
}
DLT_DEV unsigned few8_ints_f16(unsigned biased, bool hi) {   // bytes + 128 behind the exponent of 1024
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const unsigned x = __builtin_amdgcn_perm(0x64646464u, biased, hi ? 0x07030702 : 0x07010700);
  return __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, x) - f16x2{(_Float16)1152.f, (_Float16)1152.f});
}
template <int FMT, typename TIO>
DLT_DEV u32x4 few8_keys(unsigned a, unsigned b, float scale) {
  if constexpr (FMT == DLT_FP8_E4M3) return cvt8_eight<FMT, TIO>(a, b, scale);
  else if constexpr (std::is_same<TIO, f16_t>::value) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    return u32x4{few8_ints_f16(a, false), few8_ints_f16(a, true), few8_ints_f16(b, false), few8_ints_f16(b, true)};
  } else return u32x4{few8_ints_bf16(a, false), few8_ints_bf16(a, true), few8_ints_bf16(b, false), few8_ints_bf16(b, true)};
}
template <int FMT, typename TIO>
DLT_DEV u32x4 few8_values(unsigned a, unsigned b, float scale_a, float scale_b) {
  if constexpr (FMT == DLT_FP8_E4M3)
    return u32x4{cvt8_pair<FMT, TIO>(a, scale_a, false), cvt8_pair<FMT, TIO>(a, scale_a, true), cvt8_pair<FMT, TIO>(b, scale_b, false), cvt8_pair<FMT, TIO>(b, scale_b, true)};
  else return u32x4{few8_ints_bf16(a, false), few8_ints_bf16(a, true), few8_ints_bf16(b, false), few8_ints_bf16(b, true)};
}

// FULL: both tensors have D dims, K's rows lie at multiples of 16 bytes.  BAL: a run of steps to a workgroup, else a (batch, kv head).
template <typename TIO, int D, int NP, int FMT, bool FULL, int NW, bool BAL>
__global__ __launch_bounds__(64 * NW, NW > 4 ? 4 : NP == 1 ? 3 : 2) void few8_kernel(const Few8Args a) {
  static_assert(NW == 4 || !BAL, "a step is four tiles");
  dlt_kernargs_in<sizeof(Few8Args)>();
  typedef Few8<D> F;
  constexpr int NG = F::NG, VB = F::VB, KC = F::KC, VW = F::VW, TK = F::TK;
  extern __shared__ __align__(16) char smem[];   // results of the waves
  __shared__ unsigned odd_rows[NP];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // (batch, kv head), the run of it, how many it has, its steps [s0, s1)
  int b, h, run = 0, runs = 1, s0 = 0, s1 = 0;
  BandSeq sq;
  if constexpr (BAL) {
    if (!few8_run<TK>(a, (int)blockIdx.x, lane, b, h, run, runs, s0, s1, sq)) return;
  } else {
    b = band_div((int)blockIdx.x, a.by_heads);
    h = (int)blockIdx.x - b * a.Hkv;
    sq = band_seq<true>(a, b);
  }
  const float scale = a.scale_log2;
  typedef typename std::conditional<FMT == DLT_INT8, bf16_t, TIO>::type PT;   // of P and the values

  {
    const int32_t* pages = a.pg.table + b * a.pg.ts;
    const uint8_t* kh = reinterpret_cast<const uint8_t*>(a.k) + h * a.ks[1];
    const uint8_t* vh = reinterpret_cast<const uint8_t*>(a.v) + h * a.vs[1];
    const uint8_t *ksc = a.k_sc + h * a.kss[1], *vsc = a.v_sc + h * a.vss[1];
    const TIO* qb = reinterpret_cast<const TIO*>(a.q) + b * a.qs[0] + (int64_t)h * a.G * a.qs[1];

    // pages and scales of the wave's next BATCH tiles: a group of 16 tokens to a lane
    int64_t ka_l = 0, va_l = 0;
    int ek_l = 127, ev_l = 127;
    auto look_at = [&](int tok) __attribute__((always_inline)) {
      int in16;
      const int page = band_page(a.pg, pages, dlt_imax(tok, 0) >> 4, in16);
      const int blk = (int)dlt_fastdiv((uint32_t)in16, a.mB, a.sB);
      ka_l = page * a.ks[0] + 16 * in16 * a.ks[2];
      va_l = page * a.vs[0] + 16 * in16 * a.vs[2];
      ek_l = ksc[page * a.kss[0] + blk * a.kss[2]];
      ev_l = vsc[page * a.vss[0] + blk * a.vss[2]];
    };
    // A tile: 8-bit numbers as they come.  The next tile's take their places as soon as these are converted.
    unsigned kr[NG][D / 16], vr[NG][4][VW];
    auto from = [&](const uint8_t* base, int64_t at_l, int l) __attribute__((always_inline)) {
      const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)at_l, l), hi = __builtin_amdgcn_readlane((int)(at_l >> 32), l);
      return base + (int64_t)((uint64_t)hi << 32 | lo);
    };
    auto fetch_k = [&](int at) __attribute__((always_inline)) {   // the at-th of the batch
      uint32_t o = FULL ? (uint32_t)n * (uint32_t)a.ks[2] + 16u * g : (uint32_t)n * (uint32_t)a.ks[2] + 8u * g;
      asm volatile("" : "+v"(o));   // 32-bit offsets beside a wave-uniform address, not 64-bit ones for every load
#pragma unroll
      for (int u = 0; u < NG; u++) {
        const uint8_t* base = from(kh, ka_l, at * NG + u);
        if constexpr (FULL) {
#pragma unroll
          for (int c = 0; c < D / 64; c++) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(base + o + 64 * c);
#pragma unroll
            for (int i = 0; i < 4; i++) kr[u][4 * c + i] = w[i];
          }
        } else {
#pragma unroll
          for (int c = 0; c < D / 32; c++) {
            u32x2 w = {0u, 0u};
            if (32 * c + 8 * g < a.dk_) w = *reinterpret_cast<const u32x2*>(base + o + 32 * c);
            kr[u][2 * c] = w[0];
            kr[u][2 * c + 1] = w[1];
          }
        }
      }
    };
    auto fetch_v = [&](int at) __attribute__((always_inline)) {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        o[j] = (uint32_t)(4 * g + j) * (uint32_t)a.vs[2] + (uint32_t)(4 * VW) * n;
        asm volatile("" : "+v"(o[j]));
      }
#pragma unroll
      for (int u = 0; u < NG; u++) {
        const uint8_t* base = from(vh, va_l, at * NG + u);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if constexpr (VW == 2) {
            u32x2 w = {0u, 0u};
            if (FULL || 8 * n < a.dv_) w = *reinterpret_cast<const u32x2*>(base + o[j]);
            vr[u][j][0] = w[0];
            vr[u][j][VW - 1] = w[1];
          } else {
            vr[u][j][0] = 0u;
            if (FULL || 4 * n < a.dv_) vr[u][j][0] = *reinterpret_cast<const unsigned*>(base + o[j]);
          }
        }
      }
    };

    // Where no window leaves tokens out, the places of the first tiles do not wait for the sequence's length: what lies behind it is some page's, and masked
    const bool early = !BAL && a.W >= a.Lk;
    if (early) {
      look_at(dlt_imin(TK * (wave + NW * (lane / NG)) + 16 * (lane % NG), a.Lk - 1));
      fetch_k(0);
      fetch_v(0);
    }
    u32x4 qf[NP][KC];
#pragma unroll
    for (int p = 0; p < NP; p++) {
      const int r = 16 * p + n;
      const TIO* row = band_row_ptr(qb, a.qs, a, r < a.rows ? r : 0);   // (rows of padding too: nothing of theirs reaches another row)
#pragma unroll
      for (int c = 0; c < KC; c++) {
        const int d = FULL ? 16 * (g + 4 * (c >> 1)) + 8 * (c & 1) : 32 * c + 8 * g;
        qf[p][c] = u32x4{0u, 0u, 0u, 0u};
        if (r < a.rows && (FULL || d < a.dk_)) qf[p][c] = *reinterpret_cast<const u32x4*>(row + d);
      }
    }
    BandWalk<TK> W;
    int first, last;
    few8_walk(a, sq, W, first, last);
    const int n_rows = sq.n_q * a.G;
    const int t0 = 4 * s0, t1 = BAL ? dlt_imin(4 * s1, W.n) : W.n;
    auto look = [&](int tile) __attribute__((always_inline)) {   // `tile`: the first of the batch
      const int t = tile + NW * (lane / NG);
      look_at(dlt_imin(W.tok(TK * dlt_imin(t, dlt_imax(W.n - 1, 0)) + 16 * (lane % NG)), sq.n_k - 1));
    };
    const int tw = t0 + wave, tiles = tw < t1 ? (t1 - tw + NW - 1) / NW : 0;   // the wave's tiles: tw, tw + NW, ..
    if (!early && tiles > 0) {
      look(tw);
      fetch_k(0);
      fetch_v(0);
    }
    int hi[NP], lo[NP];   // the row sees tokens lo < x <= hi, and the sinks
#pragma unroll
    for (int p = 0; p < NP; p++) {
      const int r = 16 * p + n;
      const bool on = r < n_rows;
      const int pos = sq.off + band_row(a, on ? r : 0).tok;
      hi[p] = on ? dlt_imin(pos, sq.n_k - 1) : -1;
      lo[p] = pos - a.W;
    }
    float m_run[NP], l_run[NP];
    f32x4 acc[NP][VB];
#pragma unroll
    for (int p = 0; p < NP; p++) {
      m_run[p] = -INFINITY;
      l_run[p] = 0.f;
#pragma unroll
      for (int d = 0; d < VB; d++) acc[p][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    int at = 0;   // the tile's place in its batch
#pragma unroll 1
    for (int i = 0; i < tiles; i++) {
      const int tile = tw + NW * i;
      int tok[NG], ek[NG], ev[NG];
#pragma unroll
      for (int u = 0; u < NG; u++) {
        tok[u] = W.tok(TK * tile + 16 * u);
        ek[u] = __builtin_amdgcn_readlane(ek_l, at * NG + u);
        const int e = __builtin_amdgcn_readlane(ev_l, at * NG + u);
        ev[u] = tok[u] < sq.n_k ? e : 127;   // of a block of nothing that the sequence holds: anything
      }
      float t[NP][NG][4];
#pragma unroll
      for (int u = 0; u < NG; u++) {
        f32x4 s[NP];
        const float sc = cvt8_scale(ek[u]);
#pragma unroll
        for (int c = 0; c < KC; c++) {
          const u32x4 op = few8_keys<FMT, TIO>(kr[u][2 * c], kr[u][2 * c + 1], sc);
#pragma unroll
          for (int p = 0; p < NP; p++) s[p] = Mma<TIO>::mfma(op, qf[p][c], c == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[p]);
        }
#pragma unroll
        for (int p = 0; p < NP; p++)
#pragma unroll
          for (int j = 0; j < 4; j++) t[p][u][j] = FMT == DLT_INT8 ? s[p][j] * sc : s[p][j];
      }
      __builtin_amdgcn_sched_barrier(0);
      const bool more = i + 1 < tiles;
      if (more) {
        if (++at == F::BATCH) {
          at = 0;
          look(tile + NW);
        }
        fetch_k(at);
      }
      __builtin_amdgcn_sched_barrier(0);
      // unless every row sees the whole tile
      const bool edge = tok[NG - 1] + 15 > first || (tok[0] <= last - a.W && tok[NG - 1] + 15 >= a.S);
      if (edge) {
        keep_branch();
#pragma unroll
        for (int p = 0; p < NP; p++)
#pragma unroll
          for (int u = 0; u < NG; u++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const int x = tok[u] + 4 * g + j;
              t[p][u][j] = x <= hi[p] && (x > lo[p] || x < a.S) ? t[p][u][j] : -INFINITY;
            }
      }
      u32x4 ph[NP][F::NT], pl[NP][F::NT];
#pragma unroll
      for (int p = 0; p < NP; p++) {
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < NG; u++)
#pragma unroll
          for (int j = 0; j < 4; j++) mx = fmaxf(mx, t[p][u][j]);
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
          l_run[p] *= al;
        }
        const float neg = m_run[p] == -INFINITY ? 0.f : -m_run[p] * scale;
#pragma unroll
        for (int kb = 0; kb < F::NT; kb++) {
          float e[8], r[8];
#pragma unroll
          for (int j = 0; j < 8; j++) e[j] = fast_exp2(fmaf(t[p][2 * kb + (j >> 2)][j & 3], scale, neg));
          l_run[p] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
          if constexpr (FMT == DLT_INT8) {
            // values enter as whole numbers, their scales here: a block of 16 tokens has one
#pragma unroll
            for (int j = 0; j < 8; j++) e[j] *= few8_lifted(ev[2 * kb + (j >> 2)]);
          }
          ph[p][kb] = pack8<PT>(e);
          unpack8<PT>(ph[p][kb], r);
#pragma unroll
          for (int j = 0; j < 8; j++) r[j] = e[j] - r[j];
          pl[p][kb] = pack8<PT>(r);
        }
      }
      if (tok[NG - 1] + 16 > sq.n_k) {   // pages hold anything behind the last key: those values, which no row sees, are cleared
        keep_branch();
#pragma unroll
        for (int u = 0; u < NG; u++)
#pragma unroll
          for (int j = 0; j < 4; j++)
#pragma unroll
            for (int w = 0; w < VW; w++) vr[u][j][w] = tok[u] + 4 * g + j < sq.n_k ? vr[u][j][w] : 0u;
      }
#pragma unroll
      for (int kb = 0; kb < F::NT; kb++)
#pragma unroll
        for (int w = 0; w < VW; w++) {
          unsigned r0[4], r1[4], c0[4], c1[4];
#pragma unroll
          for (int j = 0; j < 4; j++) { r0[j] = vr[2 * kb][j][w]; r1[j] = vr[2 * kb + 1][j][w]; }
          few8_turn(r0, c0);
          few8_turn(r1, c1);
          const float sc0 = cvt8_scale(ev[2 * kb]), sc1 = cvt8_scale(ev[2 * kb + 1]);
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const u32x4 op = few8_values<FMT, TIO>(c0[c], c1[c], sc0, sc1);
#pragma unroll
            for (int p = 0; p < NP; p++) {
              acc[p][4 * w + c] = Mma<PT>::mfma(op, ph[p][kb], acc[p][4 * w + c]);
              acc[p][4 * w + c] = Mma<PT>::mfma(op, pl[p][kb], acc[p][4 * w + c]);
            }
          }
        }
      __builtin_amdgcn_sched_barrier(0);
      if (more) fetch_v(at);
      __builtin_amdgcn_sched_barrier(0);
    }

    // Whole-number keys meet q without their scales.  From 2^114 on (inputs of bfloat16 only) such a sum of up to 128 products of up to 2^7 each can leave 32 bits, and an infinity
    // with the sign of a small probability would not be seen in the sums: rows with such an element of q are formed again, from keys with their scales.
    bool huge[NP];
#pragma unroll
    for (int p = 0; p < NP; p++) {
      huge[p] = false;
      if constexpr (FMT == DLT_INT8 && std::is_same<TIO, bf16_t>::value) {
        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
        u16x2 most = {0, 0};
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
          for (int i = 0; i < 4; i++) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, qf[p][c][i] & 0x7fff7fffu));
        constexpr unsigned short limit = (127 + 114) << 7;
        huge[p] = most[0] >= limit || most[1] >= limit;
      }
    }

    // ---- the waves' results, joined: four waves take a quarter of the blocks of output dims each
    if (tid < NP) odd_rows[tid] = 0u;
#pragma unroll
    for (int p = 0; p < NP; p++) {
      char* mine = smem + (wave * NP + p) * F::WAVE_LDS;
#pragma unroll
      for (int d = 0; d < VB; d++) {
        f32x4 x = acc[p][d];
        if constexpr (FMT == DLT_INT8) x *= __uint_as_float((unsigned)(127 - FEW8_LIFT) << 23);
        *reinterpret_cast<f32x4*>(mine + 1024 * d + 16 * lane) = x;
      }
      const float l = wave_sum4(l_run[p]);
      if (g == 0) *reinterpret_cast<float2*>(mine + 1024 * VB + 8 * n) = float2{m_run[p] * scale, l};
    }
    __syncthreads();
    constexpr int OB = VB / 4;
    const int quarter = wave & 3;
    const bool joins = NW == 4 || wave < 4;
    f32x4 o[NP][OB];
    float om[NP], ol[NP];
#pragma unroll
    for (int p = 0; p < NP; p++) {
      if (!joins) continue;
      float2 x[NW];
      om[p] = -INFINITY;
      ol[p] = 0.f;
#pragma unroll
      for (int w = 0; w < NW; w++) {
        x[w] = *reinterpret_cast<const float2*>(smem + (w * NP + p) * F::WAVE_LDS + 1024 * VB + 8 * n);
        om[p] = fmaxf(om[p], x[w].x);
      }
#pragma unroll
      for (int d = 0; d < OB; d++) o[p][d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; w++) {
        const float f = few8_weight(x[w], om[p]);
        ol[p] = fmaf(x[w].y, f, ol[p]);
#pragma unroll
        for (int d = 0; d < OB; d++) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(smem + (w * NP + p) * F::WAVE_LDS + 1024 * (OB * quarter + d) + 16 * lane);
#pragma unroll
          for (int i = 0; i < 4; i++) o[p][d][i] = fmaf(v[i], f, o[p][d][i]);
        }
      }
      bool bad = band_odd(ol[p]) || huge[p];
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

    const bool all = !BAL || runs == 1;
    // block d of the wave holds, of row n, dims VSTEP (4 g + i) + OB wave + d
    constexpr int VSTEP = 4 * VW;
    if (all && joins) {
      TIO* ob = reinterpret_cast<TIO*>(a.out) + b * a.os[0] + (int64_t)h * a.G * a.os[1];
#pragma unroll
      for (int p = 0; p < NP; p++) {
        const int r = 16 * p + n;
        if (r >= a.rows || (odd[p] >> n & 1) != 0) continue;
        const float inv = r < n_rows ? band_inverse(ol[p], hi[p]) : 0.f;
        TIO* row = band_row_ptr(ob, a.os, a, r);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int d0 = VSTEP * (4 * g + i) + OB * quarter;
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
      part = a.part + (int64_t)blockIdx.x * a.rows * a.dv_;
      ml = reinterpret_cast<float2*>(a.part + (int64_t)a.wgs * a.rows * a.dv_) + (int64_t)blockIdx.x * a.rows;
      if (run == 0 && tid == 0) *reinterpret_cast<int2*>(a.meta + 2 * (b * a.Hkv + h)) = int2{(int)blockIdx.x, runs};
      if (!all) {
#pragma unroll
        for (int p = 0; p < NP; p++) {
          const int r = 16 * p + n;
          if (r >= n_rows || (odd[p] >> n & 1) != 0) continue;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int d0 = VSTEP * (4 * g + i) + OB * quarter;
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
        if ((r & (NW - 1)) != wave) continue;
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
  }
}

// Rows of heads that several runs hold: their parts, in order.  WG: a workgroup to a row, every wave takes every fourth part; else a wave to a row.
template <typename TIO, bool WG>
__global__ __launch_bounds__(256) void few8_join_kernel(const Few8Args a) {
  dlt_kernargs_in<sizeof(Few8Args)>();
  __shared__ float sum[WG ? 4 : 1][128];
  __shared__ float2 ends[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int bh = blockIdx.y, r = WG ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave, b = band_div(bh, a.by_heads), h = bh - b * a.Hkv;
  const int2 who = *reinterpret_cast<const int2*>(a.meta + 2 * bh);
  const BandSeq sq = band_seq<true>(a, b);   // (asked for beside it)
  asm volatile("" ::"v"(sq.n_q), "v"(sq.n_k));
  if (who.y <= 1 || r >= a.rows) return;
  const bool on = r < sq.n_q * a.G;
  const float2* ml = reinterpret_cast<const float2*>(a.part + (int64_t)a.wgs * a.rows * a.dv_);
  constexpr int EACH = WG ? 4 : 1, TOGETHER = WG ? 16 : 8;   // parts on their way together
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  const int d = 2 * dlt_imin(lane, a.dv_ / 2 - 1);
  if (on)
    for (int i0 = WG ? wave : 0; i0 < who.y; i0 += EACH * TOGETHER) {
      float2 v[TOGETHER], x[TOGETHER];
#pragma unroll
      for (int k = 0; k < TOGETHER; k++) {
        const int64_t s = (int64_t)(who.x + dlt_imin(i0 + EACH * k, who.y - 1)) * a.rows + r;
        x[k] = ml[s];
        v[k] = *reinterpret_cast<const float2*>(a.part + s * a.dv_ + d);
      }
      __builtin_amdgcn_sched_barrier(0);
      float m_new = m;
#pragma unroll
      for (int k = 0; k < TOGETHER; k++) m_new = fmaxf(m_new, x[k].x);   // the last part again behind it
      const float al = m == -INFINITY ? 1.f : fast_exp2(m - m_new);
      l *= al; o0 *= al; o1 *= al;
      m = m_new;
#pragma unroll
      for (int k = 0; k < TOGETHER; k++) {
        // with a weight of 0 too: an infinite or NaN part holds such a value of a key that the row sees.  The last part again is left out, not given a weight of 0: it may be
        // infinite.  (No branch around it: the loads would be moved behind it, one after the other.)
        const bool one = i0 + EACH * k < who.y;
        const float f = few8_weight(x[k], m);
        l = one ? fmaf(x[k].y, f, l) : l;
        o0 = one ? fmaf(v[k].x, f, o0) : o0;
        o1 = one ? fmaf(v[k].y, f, o1) : o1;
      }
    }
  if constexpr (WG) {
    sum[wave][2 * lane] = o0;
    sum[wave][2 * lane + 1] = o1;
    if (lane == 0) ends[wave] = float2{m, l};
    __syncthreads();
    if (wave != 0) return;
    m = fmaxf(fmaxf(ends[0].x, ends[1].x), fmaxf(ends[2].x, ends[3].x));
    l = o0 = o1 = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float f = few8_weight(ends[w], m);
      l = fmaf(ends[w].y, f, l);
      o0 = fmaf(sum[w][2 * lane], f, o0);
      o1 = fmaf(sum[w][2 * lane + 1], f, o1);
    }
  }
  const float f = on ? band_inverse(l, dlt_imin(sq.off + band_row(a, r).tok, sq.n_k - 1)) : 0.f;
  TIO* p = band_row_ptr(reinterpret_cast<TIO*>(a.out) + b * a.os[0] + (int64_t)h * a.G * a.os[1], a.os, a, r);
  if (2 * lane < a.dv_) *reinterpret_cast<unsigned*>(p + 2 * lane) = on ? pack2<TIO>(o0 * f, o1 * f) : 0u;
}
