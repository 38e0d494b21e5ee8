// Arguments and launchers of the kernels of page_few8.h, by padded head dim.
#pragma once
#include "band_common.h"

struct Few8Args : Band8Args {
  int32_t wgs;          // workgroups, at least one a run; 0: a (batch, kv head) each
  int32_t waves;        // of a workgroup that has a (batch, kv head) to itself
  int32_t want, want_few;   // runs that the steps are cut into, but for what rounding adds (up to one a head); where those would have fewer than 5 steps
  int32_t* meta;        // of each (batch, kv head): first workgroup, how many
};
constexpr int FEW8_B_MAX = 4096;   // sequences: 64 to a lane
// full: both tensors have that many dims and K's rows lie at multiples of 16 bytes
int dlt_few8_64(const Few8Args& a, int dtype, int format, bool full, hipStream_t stream);
int dlt_few8_128(const Few8Args& a, int dtype, int format, bool full, hipStream_t stream);
