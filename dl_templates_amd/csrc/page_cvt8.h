// 8-bit numbers and their scales (powers of two), and the conversions to and from them.
//
// e4m3: 448 = 1.75 2^8 is the largest number, 2^-9 the smallest, 0x7f NaN.  int8: whole numbers -127 .. 127.  A scale is a byte e, 2^(e - 127), 255 NaN.
#pragma once
#include "attn_common.hpp"

typedef float f32x2 __attribute__((ext_vector_type(2)));
int dlt_scales8_check(const char* who, const dlt_scales8_t* s, int page);

constexpr int CVT8_LEAST = 127 - 100;   // of the exponents that an append gives
// 1 / 2^(e - 127); a scale that is NaN: 0
DLT_DEV float cvt8_inverse(int e) { return e >= 254 ? (e == 254 ? 0x1p-127f : 0.f) : __uint_as_float((unsigned)(254 - e) << 23); }
// least biased exponent at which the magnitude with these bits fits
template <int FMT>
DLT_DEV int cvt8_exponent(unsigned bits) {
  const int x = (int)(bits >> 23);
  const unsigned m = bits & 0x7fffffu;
  const int e = FMT == DLT_FP8_E4M3 ? x - 8 + (m > 0x600000u) : x - 6 + (m > 0x7e0000u);   // 1.75 2^8, 1.984375 2^6
  return dlt_imax(e, CVT8_LEAST);
}
template <int FMT>
DLT_DEV constexpr float cvt8_most() { return FMT == DLT_FP8_E4M3 ? 448.f : 127.f; }
// the largest number whose value at scale e is finite in fp16 (65504 and below)
template <int FMT>
DLT_DEV float cvt8_most_f16(int e) {
  const float inv = cvt8_inverse(e);
  return FMT == DLT_FP8_E4M3 ? fminf(448.f, 61440.f * inv) : fminf(127.f, floorf(65504.f * inv));
}

// 8 numbers -> 32 bits
template <int FMT>
DLT_DEV void cvt8_get8(u32x2 w, float (&f)[8]) {
  if constexpr (FMT == DLT_FP8_E4M3) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
      f[4 * i] = lo[0]; f[4 * i + 1] = lo[1]; f[4 * i + 2] = hi[0]; f[4 * i + 3] = hi[1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = (float)(int8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
}
// 8 values in units of their scale, rounded to nearest, bounded by `most`; no number: NaN (int8: 0)
template <int FMT>
DLT_DEV u32x2 cvt8_put8(const float (&v)[8], float most) {
  u32x2 w;
  if constexpr (FMT == DLT_FP8_E4M3) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = fabsf(v[i]) < INFINITY ? fminf(fmaxf(v[i], -most), most) : __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      int x = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
      w[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], x, true);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      unsigned x = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float f = v[4 * i + j], r = fabsf(f) < INFINITY ? fminf(fmaxf(__builtin_rintf(f), -most), most) : 0.f;
        x |= ((unsigned)(int)r & 0xffu) << (8 * j);
      }
      w[i] = x;
    }
  }
  return w;
}

// Two neighbouring 8-bit numbers (the low two bytes, or the high two) times the scale with biased exponent e as a pair of 16-bit values.  e4m3: one instruction, which takes
// the scale's exponent.  int8: a whole number to 32 bits, times the scale, packed; exact.
// (both ends of a byte need the bit below the exponent's: 0 is 2^-127, a subnormal number, 255 NaN)
DLT_DEV float cvt8_scale(int e) { return __uint_as_float((unsigned)e << 23 | ((e + 1 & 0xfe) == 0 ? 0x400000u : 0u)); }
template <int FMT, typename TIO>
DLT_DEV unsigned cvt8_pair(unsigned w, float scale, bool hi);
template <> DLT_DEV unsigned cvt8_pair<DLT_FP8_E4M3, bf16_t>(unsigned w, float scale, bool hi) {
  return hi ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))
            : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}
template <> DLT_DEV unsigned cvt8_pair<DLT_FP8_E4M3, f16_t>(unsigned w, float scale, bool hi) {
  return hi ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true))
            : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
}
template <> DLT_DEV unsigned cvt8_pair<DLT_INT8, bf16_t>(unsigned w, float scale, bool hi) {
  return pack2<bf16_t>((float)(int8_t)(hi ? w >> 16 : w) * scale, (float)(int8_t)(hi ? w >> 24 : w >> 8) * scale);
}
template <> DLT_DEV unsigned cvt8_pair<DLT_INT8, f16_t>(unsigned w, float scale, bool hi) {
  return pack2<f16_t>((float)(int8_t)(hi ? w >> 16 : w) * scale, (float)(int8_t)(hi ? w >> 24 : w >> 8) * scale);
}
template <int FMT, typename TIO>
DLT_DEV u32x4 cvt8_eight(unsigned a, unsigned b, float scale) {
  return u32x4{cvt8_pair<FMT, TIO>(a, scale, false), cvt8_pair<FMT, TIO>(a, scale, true), cvt8_pair<FMT, TIO>(b, scale, false), cvt8_pair<FMT, TIO>(b, scale, true)};
}
