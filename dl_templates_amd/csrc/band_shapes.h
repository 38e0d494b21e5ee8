// Launchers of the kernels of band_*.hip, by padded head dim, and how a call is cut into workgroups.
#pragma once
#include "dlt_internal.hpp"

struct BandArgs;
constexpr int band_class(int dk, int dv) { return dk > 64 || dv > 64 ? 128 : 64; }
// np: 16-row blocks per wave, 4 waves (own rows or keys of a workgroup: 64 np)
int dlt_band_fwd_64(const BandArgs& a, int dtype, int np, hipStream_t stream);
int dlt_band_fwd_128(const BandArgs& a, int dtype, int np, hipStream_t stream);
int dlt_band_paged_64(const BandArgs& a, int dtype, int np, hipStream_t stream);
int dlt_band_paged_128(const BandArgs& a, int dtype, int np, hipStream_t stream);
int dlt_band_bwd_q_64(const BandArgs& a, int dtype, int np, hipStream_t stream);
int dlt_band_bwd_q_128(const BandArgs& a, int dtype, int np, hipStream_t stream);
int dlt_band_bwd_kv_64(const BandArgs& a, int dtype, hipStream_t stream);
int dlt_band_bwd_kv_128(const BandArgs& a, int dtype, hipStream_t stream);
constexpr int BAND_SHARES_MAX = 128;   // workgroups that share the keys of a block of rows (forward)
// keys of a workgroup of the dK / dV kernel
#ifndef BAND_KV128
#define BAND_KV128 64
#endif
constexpr int band_kv_own(int d) { return d <= 64 ? 128 : BAND_KV128; }
// ... and of one of its workgroups for far rows
constexpr int band_kv_group(int d) { return band_kv_own(d) / 4; }
