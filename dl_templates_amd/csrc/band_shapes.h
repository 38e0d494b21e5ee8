// Launchers of the kernels of band_*.hip, by padded head dim, and how a call is cut into workgroups.
#pragma once
#include "dlt_internal.hpp"

struct BandArgs;
constexpr int band_class(int dk, int dv) { return dk > 64 || dv > 64 ? 128 : 64; }
// How a forward workgroup is made up: one wave's 16 rows, their keys over 4 waves; 64 rows, one block a wave, their keys over two groups of 4 waves; 64 rows on 4 waves;
// 128 rows, two blocks a wave.  (The dQ kernel: BAND_ONE and BAND_TWO.)
enum { BAND_FEW = 0, BAND_HALVES = 1, BAND_ONE = 2, BAND_TWO = 3 };
int dlt_band_fwd_64(const BandArgs& a, int dtype, int kind, hipStream_t stream);
int dlt_band_fwd_128(const BandArgs& a, int dtype, int kind, hipStream_t stream);
int dlt_band_paged_64(const BandArgs& a, int dtype, int kind, hipStream_t stream);
int dlt_band_paged_128(const BandArgs& a, int dtype, int kind, hipStream_t stream);
int dlt_band_bwd_q_64(const BandArgs& a, int dtype, int kind, hipStream_t stream);
int dlt_band_bwd_q_128(const BandArgs& a, int dtype, int kind, hipStream_t stream);
int dlt_band_bwd_kv_64(const BandArgs& a, int dtype, hipStream_t stream);
int dlt_band_bwd_kv_128(const BandArgs& a, int dtype, hipStream_t stream);
constexpr int BAND_SHARES_MAX = 128;   // workgroups that share the keys of a block of rows (forward)
// keys of a workgroup of the dK / dV kernel
// (128 at d = 128 leave one wave a SIMD: 187 -> 198 us for 16 heads on 4, 8192 tokens, window 1024)
constexpr int band_kv_own(int d) { return d <= 64 ? 128 : 64; }
// ... and of one of its workgroups for far rows
constexpr int band_kv_group(int d) { return band_kv_own(d) / 4; }
