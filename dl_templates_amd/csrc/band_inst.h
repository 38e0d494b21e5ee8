// Included by band_{fwd,paged,paged8,dq,dkv}_<D>.hip with DLT_BAND_D (padded head dim) and DLT_BAND_PART (0: forward, 1: forward on pages, 2: dQ, 3: dK / dV,
// 4: forward on pages in 8 bits)
// defined: kernels for one class of head dims, translation units of their own since they take long to compile.
#if DLT_BAND_PART == 2 || DLT_BAND_PART == 3
#include "band_bwd_kernel.h"
#else
#include "band_fwd_kernel.h"
#endif
#include "band_shapes.h"

#define DLT_BCAT_(a, b) a##b
#define DLT_BCAT(a, b) DLT_BCAT_(a, b)

namespace {
constexpr int D = DLT_BAND_D;
constexpr int band_lds(int bufs, int rows) { return bufs > rows * (2 * D + 16) ? bufs : rows * (2 * D + 16); }

template <typename KernT, typename ArgsT>
int band_go(KernT kern, const ArgsT& a, int64_t grid, int threads, int lds, int record, const char* who, hipStream_t stream) {
  const int rc = dlt_ensure_lds(reinterpret_cast<const void*>(kern), lds);
  if (rc != DLT_OK) return rc;
  dlt_timing_before(record, stream);
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(threads), lds, stream, a);
  dlt_timing_after(stream);
  DLT_CHECK_LAUNCH(who);
  return DLT_OK;
}
constexpr int FEWER = D == 128 ? 2 : 1;
inline int band_pad(const BandArgs& a) { return a.dk_ == D && a.dv_ == D ? 0 : dlt_imax(a.dk_, a.dv_) <= 96 ? FEWER : 1; }
template <typename KernT>
KernT band_pick(const BandArgs& a, KernT whole, KernT fewer, KernT less) { const int pad = band_pad(a); return pad == 0 ? whole : pad == FEWER ? fewer : less; }

#if DLT_BAND_PART < 2
template <typename TIO, int NP, int CK, int NW, int GR>
int band_fwd(const BandArgs& a, hipStream_t stream) {
  constexpr bool PG = DLT_BAND_PART == 1;
  constexpr int join = (GR - 1) * NW * NP * (D + 8) * 64, bufs = GR * band_nbuf(BandBuf<D, CK>::BUF, GR) * BandBuf<D, CK>::BUF;
  constexpr int lds = band_lds(bufs > join ? bufs : join, 16 * NP * NW);
  return band_go(band_pick(a, band_fwd_kernel<TIO, D, NP, CK, NW, GR, PG, 0>, band_fwd_kernel<TIO, D, NP, CK, NW, GR, PG, FEWER>,
                           band_fwd_kernel<TIO, D, NP, CK, NW, GR, PG, 1>), a, (int64_t)a.B * a.Hkv * a.nblk * a.shares,
                 64 * NW * GR, lds, DLT_K_FWD, "window forward launch", stream);
}
template <typename TIO>
int band_fwd_np(const BandArgs& a, int kind, hipStream_t stream) {
  switch (kind) {
    case BAND_FEW: return band_fwd<TIO, 1, 32, 1, 4>(a, stream);
    case BAND_HALVES: return band_fwd<TIO, 1, 64, 4, 2>(a, stream);
    case BAND_ONE: return band_fwd<TIO, 1, 64, 4, 1>(a, stream);
    default: return band_fwd<TIO, 2, 64, 4, 1>(a, stream);
  }
}
}  // namespace
#if DLT_BAND_PART == 0
int DLT_BCAT(dlt_band_fwd_, DLT_BAND_D)(const BandArgs& a, int dtype, int kind, hipStream_t stream) {
#else
int DLT_BCAT(dlt_band_paged_, DLT_BAND_D)(const BandArgs& a, int dtype, int kind, hipStream_t stream) {
#endif
  return dtype == DLT_BF16 ? band_fwd_np<bf16_t>(a, kind, stream) : band_fwd_np<f16_t>(a, kind, stream);
}
#elif DLT_BAND_PART == 4
template <typename TIO, int NP, int F8>
int band_fwd8(const Band8Args& a, hipStream_t stream) {
  constexpr int lds = band_lds(band_nbuf(BandBuf<D, 64>::BUF) * BandBuf<D, 64>::BUF, 64 * NP);
  // (pieces that do not exist are written as zeros: no kernel of its own for them but that of fewer blocks of head dims)
  return band_go(D == 128 && dlt_imax(a.dk_, a.dv_) <= 96 ? band_fwd_kernel<TIO, D, NP, 64, 4, 1, true, D == 128 ? 2 : 0, F8> : band_fwd_kernel<TIO, D, NP, 64, 4, 1, true, 0, F8>,
                 a, (int64_t)a.B * a.Hkv * a.nblk * a.shares, 256, lds, DLT_K_FWD, "paged8 forward launch", stream);
}
template <typename TIO>
int band_fwd8_kind(const Band8Args& a, int format, int kind, hipStream_t stream) {
  if (format == DLT_FP8_E4M3) return kind == BAND_TWO ? band_fwd8<TIO, 2, 1>(a, stream) : band_fwd8<TIO, 1, 1>(a, stream);
  return kind == BAND_TWO ? band_fwd8<TIO, 2, 2>(a, stream) : band_fwd8<TIO, 1, 2>(a, stream);
}
}  // namespace
int DLT_BCAT(dlt_band_paged8_, DLT_BAND_D)(const Band8Args& a, int dtype, int format, int kind, hipStream_t stream) {
  return dtype == DLT_BF16 ? band_fwd8_kind<bf16_t>(a, format, kind, stream) : band_fwd8_kind<f16_t>(a, format, kind, stream);
}
#elif DLT_BAND_PART == 2
template <typename TIO, int NP>
int band_bwd_q(const BandArgs& a, hipStream_t stream) {
  constexpr int lds = band_lds(band_nbuf(BandBuf<D, 64>::BUF) * BandBuf<D, 64>::BUF, 64 * NP);
  return band_go(band_pick(a, band_bwd_q_kernel<TIO, D, NP, 64, 4, 0>, band_bwd_q_kernel<TIO, D, NP, 64, 4, FEWER>, band_bwd_q_kernel<TIO, D, NP, 64, 4, 1>), a,
                 (int64_t)a.B * a.Hkv * a.nblk * a.shares, 256, lds, DLT_K_BWD_Q, "window dQ launch", stream);
}
template <typename TIO>
int band_bwd_q_np(const BandArgs& a, int kind, hipStream_t stream) { return kind != BAND_TWO ? band_bwd_q<TIO, 1>(a, stream) : band_bwd_q<TIO, 2>(a, stream); }
}  // namespace
int DLT_BCAT(dlt_band_bwd_q_, DLT_BAND_D)(const BandArgs& a, int dtype, int kind, hipStream_t stream) {
  return dtype == DLT_BF16 ? band_bwd_q_np<bf16_t>(a, kind, stream) : band_bwd_q_np<f16_t>(a, kind, stream);
}
#else
template <typename TIO>
int band_bwd_kv(const BandArgs& a, hipStream_t stream) {
  constexpr int lds = band_lds(band_nbuf(BandBuf<D, 64>::BUF) * BandBuf<D, 64>::BUF_KV, 64);
  return band_go(band_pick(a, band_bwd_kv_kernel<TIO, D, 0>, band_bwd_kv_kernel<TIO, D, FEWER>, band_bwd_kv_kernel<TIO, D, 1>), a,
                 (int64_t)a.B * a.Hkv * ((int64_t)a.nblk * a.shares + a.far * a.far_groups), 256, lds, DLT_K_BWD_KV, "window dK/dV launch", stream);
}
}  // namespace
int DLT_BCAT(dlt_band_bwd_kv_, DLT_BAND_D)(const BandArgs& a, int dtype, hipStream_t stream) {
  return dtype == DLT_BF16 ? band_bwd_kv<bf16_t>(a, stream) : band_bwd_kv<f16_t>(a, stream);
}
#endif
