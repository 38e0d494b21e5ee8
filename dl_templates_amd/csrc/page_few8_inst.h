// Included by page_few8_<D>.hip with DLT_FEW8_D (padded head dim) defined.
#include "page_few8.h"

#define DLT_FCAT_(a, b) a##b
#define DLT_FCAT(a, b) DLT_FCAT_(a, b)

namespace {
constexpr int D = DLT_FEW8_D;
// Up to so many rows of a call are joined by a workgroup each, if a head has 8 runs or more; others by a wave each.  us, wave / workgroup: 96 rows, 64 runs a head (2 sequences
// of 100000, 4 kv heads) 44 / 37; 32 rows, 64 runs 13.6 / 11.5; 512 rows, 16 runs (4 of 20000, 4 tokens, 8 kv heads) 26.5 / 25.7; 512 rows, 4 runs (16 of up to 4000) 22.5 / 24.0;
// 1024 rows, 2 runs 40.4 / 43.1.
constexpr int FEW8_JOIN_WGS = 1024;

template <typename KernT>
int few8_go(KernT kern, const Few8Args& a, int64_t grid, int waves, int lds, hipStream_t stream) {
  const int rc = dlt_ensure_lds(reinterpret_cast<const void*>(kern), lds);
  if (rc != DLT_OK) return rc;
  dlt_timing_before(DLT_K_FWD, stream);
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * waves), lds, stream, a);
  dlt_timing_after(stream);
  DLT_CHECK_LAUNCH("paged8 launch");
  return DLT_OK;
}
template <typename TIO, int NP, int FMT, int NW, bool BAL>
int few8_nw(const Few8Args& a, bool full, int64_t grid, hipStream_t stream) {
  const int lds = NW * NP * Few8<D>::WAVE_LDS;
  return full ? few8_go(few8_kernel<TIO, D, NP, FMT, true, NW, BAL>, a, grid, NW, lds, stream) : few8_go(few8_kernel<TIO, D, NP, FMT, false, NW, BAL>, a, grid, NW, lds, stream);
}
template <typename TIO, int NP, int FMT>
int few8_np(const Few8Args& a, bool full, hipStream_t stream) {
  if constexpr (NP == 1)
    if (a.wgs == 0 && a.waves == 8) return few8_nw<TIO, NP, FMT, 8, false>(a, full, (int64_t)a.B * a.Hkv, stream);
  if (a.wgs == 0) return few8_nw<TIO, NP, FMT, 4, false>(a, full, (int64_t)a.B * a.Hkv, stream);
  const int rc = few8_nw<TIO, NP, FMT, 4, true>(a, full, a.wgs, stream);
  if (rc != DLT_OK) return rc;
  dlt_timing_before(DLT_K_FWD, stream);
  const unsigned bh = (unsigned)(a.B * a.Hkv);
  if ((int64_t)bh * a.rows <= FEW8_JOIN_WGS && 8 * bh <= a.want) hipLaunchKernelGGL((few8_join_kernel<TIO, true>), dim3((unsigned)a.rows, bh), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((few8_join_kernel<TIO, false>), dim3((unsigned)(a.rows + 3) / 4, bh), dim3(256), 0, stream, a);
  dlt_timing_after(stream);
  DLT_CHECK_LAUNCH("paged8 sum launch");
  return DLT_OK;
}
template <typename TIO>
int few8_t(const Few8Args& a, int format, bool full, hipStream_t stream) {
  if (format == DLT_FP8_E4M3) return a.rows <= 16 ? few8_np<TIO, 1, DLT_FP8_E4M3>(a, full, stream) : few8_np<TIO, 2, DLT_FP8_E4M3>(a, full, stream);
  return a.rows <= 16 ? few8_np<TIO, 1, DLT_INT8>(a, full, stream) : few8_np<TIO, 2, DLT_INT8>(a, full, stream);
}
}  // namespace

int DLT_FCAT(dlt_few8_, DLT_FEW8_D)(const Few8Args& a, int dtype, int format, bool full, hipStream_t stream) {
  return dtype == DLT_BF16 ? few8_t<bf16_t>(a, format, full, stream) : few8_t<f16_t>(a, format, full, stream);
}
