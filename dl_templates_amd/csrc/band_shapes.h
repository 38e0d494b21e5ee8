// Launchers of the kernels of band_*.hip, by padded head dim, and how a call is cut into workgroups.
#pragma once
#include "dlt_internal.hpp"

struct BandArgs;
constexpr int band_class(int dk, int dv) { return dk > 64 || dv > 64 ? 128 : 64; }
// How a forward workgroup is made up: one wave's 16 rows, their keys over 4 waves; 64 rows, one block a wave, their keys over two groups of 4 waves; 64 rows on
// 4 waves; 128 rows, two blocks a wave.  (The dQ kernel: BAND_ONE and BAND_TWO.)
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
// Keys of a dK / dV workgroup, 16 a wave.  128 (32 a wave) read half as much from LDS for a product, and that is not what these kernels lack: with as many
// workgroups on a CU, 8 x 8 kv heads of 4 query heads, 1111 tokens, window 300, d = 64: 112 us against 81; 4 x 8, 2048 tokens, window 500: 101 / 99; 4 heads,
// 8192 tokens, window 1024: 131 / 100, d = 128: 198 / 187.  So did 128 keys on 8 waves with the values in LDS, d = 128: 189.
constexpr int BAND_KV_OWN = 64;
