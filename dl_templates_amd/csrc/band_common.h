// Attention over a 1D window with first tokens that stay visible (sinks), heads of q in groups that share one head of k and v:
// what the forward, backward and paged kernels share.
//
// Query token i of a sequence stands at position p = off + i (off = Lk - Lq, paged: length - new tokens) and sees key j iff
//   j <= p  and  (p - j < W  or  j < S).
// The G query heads of a group read the same keys, so they are rows of one tile: row r = i G + (head in the group).  A tile of 128 rows
// then spans 128 / G tokens: the keys that only some of its rows see shrink with G, and a key is fetched once for the whole group.
// lse2 and delta are contiguous [B, Hkv, Lq G] in that row order.
#pragma once
#include "flash_dma_kernel.hpp"
#include "kernargs.h"

struct BandPages {          // keys and values in pages (paged calls); strides in elements
  const int32_t* table;     // [B, cols] page numbers
  const int32_t* seq;       // [B] tokens of a sequence, the new ones included
  const int32_t* n_new;     // [B] new tokens, or NULL: T of every sequence
  int64_t ts;               // row stride of the table
  int32_t cols, n_pages;
  int32_t p16;              // 16-token groups of a page
  uint32_t m16, s16;        // division by p16
};

struct BandDiv { uint32_t m, s; };   // division of 31-bit numbers (dlt_fastdiv)
struct BandArgs {
  const void *q, *k, *v, *o, *d_o;
  void *out, *dq, *dk, *dv;
  float *lse, *delta, *part;
  void* low;                // what the rounding of o left, [B, H, low tokens, dv] (see band_low)
  int64_t qs[3], ks[3], vs[3], os[3], dos[3], dqs[3], dks[3], dvs[3];   // batch (pages: page), head, token; head dims are contiguous
  int32_t B, Hkv, G, Lq, Lk, dk_, dv_;
  uint32_t mG, sG;          // division by G
  int32_t W, S, off, rows;  // W <= Lk; rows = Lq G
  int32_t nblk, group;      // own blocks of a (batch, kv head); heads interleaved at launch (band_block)
  int32_t units;            // nblk * shares
  BandDiv by_group_units, by_group, by_last, by_shares, by_heads;   // workgroups of a group of heads; heads of a group, of the last one; shares; kv heads
  int32_t shares;           // workgroups that share the keys (forward) or rows (dK / dV) of an own block
  int32_t far, far_groups;  // dK / dV: workgroups that share the far rows of a group of sinks, such groups (band_bwd_kernel.h); 0: none
  int32_t part_keys;        // keys of a (batch, kv head) with partial sums
  int32_t cycle;            // dK / dV: chunks of rows that see a block of keys
  int32_t low_rows;         // rows of a (batch, kv head) with low parts
  int32_t q16;              // 16 is a multiple of G: 16 rows are whole tokens
  float scale_log2, grad_scale;   // grad_scale: of dQ and dK; 0 where every row sees one key, whose dS are zero but for roundings
  BandPages pg;
};

DLT_HD int64_t dlt_imin64(int64_t a, int64_t b) { return a < b ? a : b; }
DLT_HD int64_t dlt_imax64(int64_t a, int64_t b) { return a > b ? a : b; }

// Partial sums of the dK / dV kernel in `part`: dK rows [bh][share][keys], far dK rows [bh][far share, wave][far_keys], then the same of dV
struct BandParts {
  int64_t keys, far_keys, far_at, v_at, v_far_at, floats;   // far_at from the start, v_far_at from v_at on
  DLT_HD BandParts(const BandArgs& a) {
    const int64_t bh = (int64_t)a.B * a.Hkv;
    keys = a.part_keys;
    far_keys = (int64_t)a.far_groups * 16;
    far_at = bh * a.shares * keys * a.dk_;
    v_at = far_at + bh * a.far * 4 * far_keys * a.dk_;
    v_far_at = bh * a.shares * keys * a.dv_;
    floats = v_at + v_far_at + bh * a.far * 4 * far_keys * a.dv_;
  }
};

// Workgroup -> (batch, kv head), own block and share of it: `group` heads at a time are interleaved, as flash_block_causal has it, the blocks from the last on
// (`rev`: own = queries, whose first blocks may see less) or from the first.  Divisions are products: four divisions were a third of the instructions in front
// of the first copy.
DLT_DEV int band_div(int n, const BandDiv& d) { return (int)dlt_fastdiv((uint32_t)n, d.m, d.s); }
DLT_DEV void band_block(const BandArgs& a, int lin, bool rev, int& b, int& h, int& blk, int& share) {
  const int grp = band_div(lin, a.by_group_units), rem = lin - grp * (a.group * a.units);
  const int left = a.B * a.Hkv - grp * a.group;
  const bool last = left < a.group;
  const int gc = last ? left : a.group, rank = band_div(rem, last ? a.by_last : a.by_group);
  const int bh = grp * a.group + (rem - rank * gc);
  const int unit = rev ? a.units - 1 - rank : rank;
  blk = band_div(unit, a.by_shares);
  share = unit - blk * a.shares;
  b = band_div(bh, a.by_heads);
  h = bh - b * a.Hkv;
}

// Of the rows of a tile: token and head in the group
struct BandRow { int tok, head; };
DLT_DEV BandRow band_row(const BandArgs& a, int r) {
  const int t = (int)dlt_fastdiv((uint32_t)r, a.mG, a.sG);
  return BandRow{t, r - t * a.G};
}
// delta = dO . o is subtracted from every dP of a row; where a row sees few keys these cancel, and the rounding of o is what is left of it: with two keys dQ
// and dK are off by 2.3 times what their own rounding is, with 16 by 1.5, at most 1.5 in any case with o unrounded (the roundings of dS remain).  Rows that see
// up to 16 keys, those of short windows and of the first 16 positions, therefore keep the part of o that its rounding drops.
template <typename TIO>
DLT_DEV TIO* band_low(const BandArgs& a, int b, int h, int r) {
  if (r >= a.low_rows) return nullptr;
  const BandRow w = band_row(a, r);
  const int tokens = a.low_rows / a.G;
  return reinterpret_cast<TIO*>(a.low) + (((int64_t)b * a.Hkv + h) * a.G + w.head) * tokens * a.dv_ + (int64_t)w.tok * a.dv_;
}
// v less its rounding (0 where that is no number)
template <typename TIO>
DLT_DEV float band_dropped(float v) {
  const float d = v - (float)(TIO)v;
  return fabsf(d) < INFINITY ? d : 0.f;
}

template <typename T>
DLT_DEV T* band_row_ptr(T* base, const int64_t (&st)[3], const BandArgs& a, int r) {
  const BandRow w = band_row(a, r);
  return base + (w.tok * st[2] + w.head * st[1]);
}

// Keys that the rows of a block at positions [first, last] see, in groups of 16: those with sinks, then those of the window.  Places y count them without the
// gap between (token y, from 16 sink groups on token y + jump); chunk i holds places CK i .. + CK - 1, so sinks share a chunk with the window's first keys.
// With bounds less the jump a row's rule is the same for places as for tokens: no token below the window's first group is in any row's window, and none behind
// the sinks' groups is a sink.  us, against sinks in chunks of their own and a window that starts at a multiple
// of CK: 8 x 8 kv heads of 4 query heads, 1111 tokens, window 300, 5 sinks, forward / dQ, d = 64 69 / 70 -> 60 / 62, d = 128 109 / 149 -> 96 / 137; 4 of 8192,
// window 1024, d = 128 111 / 138 -> 106 / 136.  Without sinks a start at multiples of 16 changes nothing or loses up to 3 %: neighbouring blocks' chunks then
// are not the same.
template <int CK>
struct BandWalk {
  int sinks, jump, n;   // places with sinks, when there is a gap behind them; tokens left out; chunks
  DLT_DEV void init(int first, int last, int W, int S) {
    sinks = jump = n = 0;
    if (last < 0) return;
    const int w0 = dlt_imax(first - W + 1, 0) & (S > 0 ? ~15 : ~(CK - 1)), end = (dlt_imin(S, last + 1) + 15) & ~15;
    if (w0 > end) { sinks = end; jump = w0 - end; }
    n = (last - jump) / CK + 1;
  }
  DLT_DEV int tok(int y) const { return y + (y >= sinks ? jump : 0); }
  // Of chunks [beg, end) those that every one of the rows sees whole (sinks not counted): [f0, f1).  These and the others, at an edge of the window, run in
  // loops of their own: with both bodies in one loop the compiler copies the accumulators from one set of registers to another, twice a chunk (72 vector
  // instructions next to 210).
  DLT_DEV void whole(int first, int last, int W, int beg, int end, int& f0, int& f1) const {
    const int behind = last - jump - W + 1;                   // the last row's window starts there
    const int lo = behind > 0 ? (behind + CK - 1) / CK : 0;
    const int hi = first - jump >= 0 ? (first - jump + 1) / CK : 0;
    f0 = dlt_imin(dlt_imax(beg, lo), end);
    f1 = dlt_imax(f0, dlt_imin(end, hi));
  }
};

// Blocks of 32 head dims that take part.  PAD 0: both tensors have D dims; 1: fewer; 2 (D = 128): at most 96 (2 x 8 kv heads of 4 query heads, 4096 tokens,
// window 500, forward / dQ / dK and dV, us: d = 96 105 / 127 / 143, d = 112, where all blocks take part, 124 / 172 / 165)
constexpr int band_kc(int d, int pad) { return pad == 2 ? 3 : d / 32; }

// Own rows as B operands: lane (n, g) holds head dims 32 c + 8 g .. + 7 of row n; r < 0: no row
template <int KC, typename TIO>
DLT_DEV void band_load_own(u32x4 (&f)[KC], const TIO* row, bool on, int dims, int g) {
#pragma unroll
  for (int c = 0; c < KC; c++) {
    f[c] = u32x4{0u, 0u, 0u, 0u};
    if (on && 8 * (4 * c + g) < dims) f[c] = *reinterpret_cast<const u32x4*>(row + 8 * (4 * c + g));
  }
}

// Copies of 16 bytes a lane to `lds` + OA, + OB (and + OC, + OD) + 16 lane, as dlt_copy16_to_lds (swa2_common.hpp) with one set-up of M0 for all: the offset
// field of the instruction counts for the memory address too, so `voff` of a copy is its lane's offset less that.  (A set-up for each copy was a sixth of a
// chunk's instructions.)
template <int OA, int OB>
DLT_DEV void band_copy2(const char* base, uint32_t va, uint32_t vb, char* lds) {
  const uint32_t m = (uint32_t)(uintptr_t)(DLT_LDS char*)lds;
  uint32_t saved;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %1 offset:%5\n\t"
               "global_load_lds_dwordx4 %3, %1 offset:%6\n\ts_mov_b32 m0, %0"
               : "=&s"(saved) : "s"(base), "v"(va), "v"(vb), "s"(m), "n"(OA), "n"(OB) : "memory");
}
DLT_DEV void band_copy4(const char* base, const uint32_t (&v)[4], char* lds) {
  const uint32_t m = (uint32_t)(uintptr_t)(DLT_LDS char*)lds;
  uint32_t saved;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %6\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %1\n\tglobal_load_lds_dwordx4 %3, %1 offset:%7\n\t"
               "global_load_lds_dwordx4 %4, %1 offset:%8\n\tglobal_load_lds_dwordx4 %5, %1 offset:%9\n\ts_mov_b32 m0, %0"
               : "=&s"(saved) : "s"(base), "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "s"(m), "n"(1024), "n"(2 * 1024), "n"(3 * 1024) : "memory");
}
// All copies of a group of 16 tokens: copy i goes to `lds` + 1024 i; v[i] = the lane's offset + band_bias - 1024 i, taken from base - band_bias.  Under PAD
// lanes of pieces that do not exist copy nothing; copies two apart move the same piece (8 tokens apart).
template <int NI> constexpr int band_bias = 1024 * (NI - 1);
template <int NI, int PAD>
DLT_DEV void band_copy_group(const char* base, const uint32_t (&v)[NI], bool on0, bool on1, char* lds) {
  static_assert(NI == 2 || NI == 4, "head dim 64 or 128");
  const char* b = base - band_bias<NI>;
  if constexpr (NI == 2) {
    if (!PAD || on0) band_copy2<0, 1024>(b, v[0], v[1], lds);
  } else if constexpr (!PAD) {
    band_copy4(b, v, lds);
  } else {
    if (on0) band_copy2<0, 2 * 1024>(b, v[0], v[2], lds);
    if (on1) band_copy2<1024, 3 * 1024>(b, v[1], v[3], lds);
  }
}

// Copies of keys or values HBM -> LDS, 16 tokens at a time (one wave): token t of the group, piece c of its row lies at piece
// c ^ swz(t) (FlashDRow).  The place of the group is wave-uniform, a lane's offset inside it is kept in registers.
template <int D>
struct BandStage {
  typedef FlashDRow<D> R;
  static constexpr int NI = 16 / R::TPI;                    // copy instructions per 16 tokens
  uint32_t off[NI];
  int t0, lp, npieces;
  uint32_t sn2;
  DLT_DEV uint32_t piece(int i) const { return (uint32_t)(lp ^ R::swz(t0 + R::TPI * i)); }
  DLT_DEV void init(int lane, int dims, int64_t sn) {
    t0 = lane / R::PIECES;
    lp = lane % R::PIECES;
    npieces = dims >> 3;
    sn2 = (uint32_t)sn * 2u;
#pragma unroll
    for (int i = 0; i < NI; i++) off[i] = (uint32_t)(t0 + R::TPI * i) * sn2 + 16u * piece(i) + (uint32_t)(band_bias<NI> - 1024 * i);
  }
  template <int PAD>
  DLT_DEV void issue(const char* base, char* dst) const {   // all 16 tokens are there
    band_copy_group<NI, PAD>(base, off, (int)piece(0) < npieces, (int)piece(1) < npieces, dst);
  }
  template <int PAD>
  DLT_DEV void issue_clamped(const char* base, int last, char* dst) const {   // tokens behind `last` repeat it
#pragma unroll 1
    for (int i = 0; i < NI; i++)
      if (!PAD || (int)piece(i) < npieces) dlt_copy16_to_lds(base, (uint32_t)dlt_imin(t0 + R::TPI * i, last) * sn2 + 16u * piece(i), dst + R::TPI * i * R::ROW);
  }
};

// Rows r0 .. r0 + 15 of a query-side tensor -> LDS (dK / dV kernel).  `base`: of the (batch, kv head).
template <int D>
struct BandStageRows {
  typedef FlashDRow<D> R;
  static constexpr int NI = 16 / R::TPI;
  uint32_t off[NI];   // q16: of the lane's row inside a group of 16 that starts with a token
  int t0, lp, npieces;
  DLT_DEV uint32_t piece(int i) const { return (uint32_t)(lp ^ R::swz(t0 + R::TPI * i)); }
  DLT_DEV void init(const BandArgs& a, int lane, int dims, const int64_t (&st)[3]) {
    t0 = lane / R::PIECES;
    lp = lane % R::PIECES;
    npieces = dims >> 3;
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const BandRow w = band_row(a, t0 + R::TPI * i);
      off[i] = (uint32_t)(w.tok * (int)st[2] + w.head * (int)st[1]) * 2u + 16u * piece(i) + (uint32_t)(band_bias<NI> - 1024 * i);
    }
  }
  // rows behind `last` repeat it
  template <int PAD>
  DLT_DEV void issue(const BandArgs& a, const char* base, const int64_t (&st)[3], int r0, int last, char* dst) const {
    const int f0 = dlt_imin(r0, last);
    const int tk = (int)dlt_fastdiv((uint32_t)f0, a.mG, a.sG);
    const char* b = base + (int64_t)tk * st[2] * 2;   // wave-uniform
    if (a.q16 != 0 && r0 + 15 <= last) {
      band_copy_group<NI, PAD>(b, off, (int)piece(0) < npieces, (int)piece(1) < npieces, dst);
    } else {
      keep_branch();
#pragma unroll 1
      for (int i = 0; i < NI; i++) {
        const BandRow w = band_row(a, dlt_imin(r0 + t0 + R::TPI * i, last));
        const uint32_t o = (uint32_t)((w.tok - tk) * (int)st[2] + w.head * (int)st[1]) * 2u + 16u * piece(i);
        if (!PAD || (int)piece(i) < npieces) dlt_copy16_to_lds(b, o, dst + R::TPI * i * R::ROW);
      }
    }
  }
};

// bytes of a chunk of CK tokens of both streamed tensors, and of the scalars of CK rows (dK / dV kernel)
template <int D, int CK>
struct BandBuf {
  static constexpr int REG = CK * 2 * D;
  static constexpr int BUF = 2 * REG;
  static constexpr int BUF_KV = 2 * REG + 2 * CK * 4;
};

// chunk buffers of a workgroup: as many as leave a CU two workgroups and more (one more at d = 128, with one block of rows per wave: 155 -> 186 us for the
// decode step of 64 sequences, 18 -> 29 for 3 x 6 heads of 1111 tokens)
constexpr int band_nbuf(int buf, int groups = 1) { return 4 * buf <= 65536 && 3 * groups * buf <= 131072 ? 3 : 2; }

// Accumulators in C layout (lane (n, g): dims 16 d + 4 g .. + 3 of own row n, times mul[p]) -> LDS tile of 16-bit values -> rows.
// `ptr(row)`: the row's place or NULL.  The tile takes the chunk buffers' LDS.
// `again()`: the wave writes rows of its own part of the tile once more (see below).  LOW: what the rounding drops instead of what it leaves.
template <int D, int NP, typename TIO, bool LOW = false, int NA, typename PtrFn, typename AgainFn>
DLT_DEV void band_store_rows(char* sT, const f32x4 (&acc)[NP][NA], const float (&mul)[NP], int nw, int groups, bool write, int dims, int wave, int n, int g,
                             int tid, PtrFn ptr, AgainFn again) {
  constexpr int PT = D * 2 + 16;
  // `write`: the wave's group writes the tile; the waves of all groups store it
#pragma unroll
  for (int p = 0; write && p < NP; p++) {
    char* row = sT + (wave * 16 * NP + 16 * p + n) * PT + 8 * g;
#pragma unroll
    for (int d = 0; d < NA; d++) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = LOW ? band_dropped<TIO>(acc[p][d][i] * mul[p]) : acc[p][d][i] * mul[p];
      u32x2 w;
      w.x = pack2<TIO>(v[0], v[1]);
      w.y = pack2<TIO>(v[2], v[3]);
      *reinterpret_cast<u32x2*>(row + 32 * d) = w;
    }
  }
  again();
  __syncthreads();
  int tw = tid;   // opaque copy: keeps the addresses out of the registers that live across the chunk loop
  asm volatile("" : "+v"(tw));
  constexpr int CH = D / 8;
  const int c = tw % CH;
  if (8 * c < dims)
    for (int row = tw / CH; row < 16 * NP * nw; row += 64 * nw * groups / CH) {
      TIO* p = ptr(row);
      if (p == nullptr) continue;
      const u32x4 v = lds_read16(sT + row * PT + 16 * c);
      store_stream16(p + 8 * c, v);
    }
  __syncthreads();
}

// 1 / sum of a row at position `pos` (< 0: it sees nothing, and gives zeros).  A sum of 0 otherwise means that every score that the row sees is -inf: the
// softmax of those is NaN.
DLT_DEV float band_inverse(float sum, int pos) { return sum != 0.f ? fast_rcp(sum) : pos < 0 ? 0.f : NAN; }
DLT_DEV bool band_odd(float v) { return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u; }   // infinite or NaN
template <int NP, int NA>
DLT_DEV bool band_odd_row(const f32x4 (&acc)[NP][NA], int p) {
  bool odd = false;
#pragma unroll
  for (int d = 0; d < NA; d++)
#pragma unroll
    for (int i = 0; i < 4; i++) odd = odd || band_odd(acc[p][d][i]);
  return odd;
}

// Hidden pairs of a chunk at the edge.  Key x + 4 g + c of own row p (c a constant of the unrolled code) is seen iff c <= h && (c > l || c < s).  The
// bounds are formed here, per chunk, from a value the compiler cannot look through: left to itself it keeps one register for each c, in kernels that have none
// left.
struct BandEdge { int h, l, s; };
DLT_DEV BandEdge band_edge(int hi, int lo, int S, int x, int g) {
  int at = x + 4 * g;
  asm volatile("" : "+v"(at));
  return BandEdge{hi - at, lo - at, S - at};
}
DLT_DEV bool band_edge_sees(const BandEdge& e, int c) { return c <= e.h && (c > e.l || c < e.s); }
// a value formed for every lane, hidden pairs too (where it is an exponential the compiler would otherwise branch around it)
DLT_DEV float band_formed(float v) {
  asm volatile("" : "+v"(v));
  return v;
}

// ---- rows whose sums came out infinite or NaN ------------------------------------------------------------------------------------
// The matrix products of a chunk at the edge of a window multiply hidden pairs by 0, and 0 times an infinity or a NaN is NaN: a hidden key
// (in the backward pass a hidden query) with such values would reach rows that do not see it.  Every kernel therefore looks at its sums once,
// at the end, and takes rows with such a value again, one wave a row, over the pairs that see each other alone.  Ordinary data never
// comes here.
template <typename TIO>
DLT_DEV float band_dot(const TIO* x, const TIO* y, int dims) {
  float s = 0.f;
  for (int d = 0; d < dims; d += 8) {
    float fx[8], fy[8];
    unpack8<TIO>(*reinterpret_cast<const u32x4*>(x + d), fx);
    unpack8<TIO>(*reinterpret_cast<const u32x4*>(y + d), fy);
#pragma unroll
    for (int j = 0; j < 8; j++) s = fmaf(fx[j], fy[j], s);
  }
  return s;
}
DLT_DEV float band_lane(float v, int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); }
DLT_DEV float band_wave_max(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}
// acc[2] += w * (dims 2 lane, 2 lane + 1 of x)
template <typename TIO>
DLT_DEV void band_axpy(float (&acc)[2], float w, const TIO* x, int dims, int lane) {
  if (2 * lane < dims) {
    acc[0] = fmaf(w, (float)x[2 * lane], acc[0]);
    acc[1] = fmaf(w, (float)x[2 * lane + 1], acc[1]);
  }
}
DLT_DEV bool band_sees(int p, int j, int W, int S) { return j <= p && (p - j < W || j < S); }
