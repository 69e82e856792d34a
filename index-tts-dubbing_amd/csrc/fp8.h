// Block-scaled e4m3: a block of values shares one power-of-two scale 2^(byte - 127), and each value is held as an
// OCP e4m3 code (1-4-3, largest 448, one NaN per sign, no infinity).  The scale is the smallest power of two that
// brings the block's largest finite magnitude within 448, so x / scale is exact (f32 keeps every bit of it) and
// the codes are defined bit for bit: the rounding to 8 bits is the only one.  Values that are not finite become
// the NaN code and do not count for the scale; a block without a nonzero finite value has the byte 127.
#pragma once
#include "common.h"

namespace itts {

// scale byte of a block whose largest finite magnitude is a: E = min { e : a <= 1.75 * 2^(8 + e) }, e >= -126
__device__ __forceinline__ int e4m3_scale_byte(float a) {
  const uint32_t u = __float_as_uint(a);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return u == 0 ? 127 : (e < 1 ? 1 : e);
}
// 1 / scale, exact: bytes are 1 .. 247
__device__ __forceinline__ float e4m3_inv_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }
__device__ __forceinline__ float e4m3_scale(int byte) { return __uint_as_float((uint32_t)byte << 23); }

// four codes (round to nearest even) of four values already divided by the scale
__device__ __forceinline__ uint32_t e4m3_pack4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// The magnitudes' maximum is taken on their bits: as integers they order like the values, and what is not finite comes out
// above every finite value, so one test per block finds it and the ordinary path tests no value.  max_bits: of f32 values
// or of pairs of bf16 (dwords), the result in f32's bits.
constexpr uint32_t kInfBits = 0x7F800000u;
__device__ __forceinline__ uint32_t max_bits(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return m;
}

// scale byte of N values' block and the values divided by the scale, given the block's largest magnitude's bits
// (`top`); `reduce`: a value's maximum over the block's lanes.  Values that are not finite become NaN.
template <int N, typename R>
__device__ __forceinline__ int e4m3_scaled(float (&v)[N], uint32_t top, R reduce) {
  if (__any(top >= kInfBits)) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
      m = max(m, b < kInfBits ? b : 0u);
      v[i] = b < kInfBits ? v[i] : __builtin_nanf("");
    }
    top = reduce(m);
  }
  const int byte = e4m3_scale_byte(__uint_as_float(top));
  const float inv = e4m3_inv_scale(byte);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] *= inv;
  return byte;
}

}  // namespace itts
