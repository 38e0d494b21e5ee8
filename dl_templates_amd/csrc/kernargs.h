// A kernel's arguments into the scalar cache, for kernels whose arguments span several cache lines.
#pragma once
#include <hip/hip_runtime.h>

// The compiler loads each argument where it is first used; every first touch of a cache line is then a trip to memory of its own, one after the other, before
// the kernel has asked for any data.  Here one word of each line is loaded, all at once.  Rotation of 256 tokens 7.1 -> 6.4 us, append of one token to 64
// sequences 6.6 -> 6.0, decode step on 300 keys 7.8 -> 7.4.
template <int BYTES>
__device__ __attribute__((always_inline)) inline void dlt_kernargs_in() {
  constexpr int N = (BYTES + 63) / 64;
  static_assert(N <= 14, "one word a line in registers");
  const __attribute__((address_space(4))) unsigned* p = (const __attribute__((address_space(4))) unsigned*)__builtin_amdgcn_kernarg_segment_ptr();
  unsigned v[14];
#pragma unroll
  for (int i = 0; i < 14; i++) v[i] = p[16 * (i < N ? i : 0)];
  asm volatile("" ::"s"(v[0]), "s"(v[1]), "s"(v[2]), "s"(v[3]), "s"(v[4]), "s"(v[5]), "s"(v[6]), "s"(v[7]), "s"(v[8]), "s"(v[9]), "s"(v[10]), "s"(v[11]), "s"(v[12]), "s"(v[13]));
}
