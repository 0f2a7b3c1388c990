// The 8-bit row format of the block-scaled linear layers (OCP microscaling,
// MXFP8 with e4m3 elements): every 32 values of a row share one power-of-two
// scale, held as its biased exponent (E8M0, 2^(code - 127)).
//
// The scale is the smallest power of two, at least 2^-127, with which no finite
// value of the block passes 448 = 1.75 * 2^8, so no value is ever clipped and each
// is rounded once, to within half an e4m3 step.  (The OCP text's floor rule
// would clip values between 1.75 and 2 times the block's power of two.)
// A value that is not finite becomes NaN in its place and does not count in
// the block's maximum.
#pragma once

#include "ltx_common.h"

namespace ltx {

constexpr int kMxBlock = LTX_MX_BLOCK;

// The largest finite magnitude of N values.  A maximum passes over NaN by itself;
// only one that is infinite is taken again without the infinities.
template <int N>
__device__ __forceinline__ float mx_top(const float (&v)[N]) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i += 2) top = fmaxf(top, fmaxf(fabsf(v[i]), fabsf(v[i + 1])));
  if (top == __builtin_inff()) {
    top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(v[i]) < __builtin_inff() ? fabsf(v[i]) : 0.0f);
  }
  return top;
}

// The E8M0 code of a block with maximum `top` (finite, >= 0): the exponent of
// top / 256, one more where top's mantissa is over 1.75.
__device__ __forceinline__ uint32_t mx_scale_code(float top) {
  const int bits = (int)__float_as_uint(top);
  const int e = (bits + 0x1FFFFF) >> 23;  // one more for a mantissa over 0x600000
  return (uint32_t)(e > 8 ? e - 8 : 0);
}

// 2^(127 - code), what the block's values are multiplied with (exact: a power
// of two; code is at most 247).
__device__ __forceinline__ float mx_inverse(uint32_t code) { return __uint_as_float((254u - code) << 23); }

// Four values, already divided by the scale, as e4m3 codes (byte i = value i),
// to nearest even; NaN and infinities give NaN.
__device__ __forceinline__ uint32_t mx_pack4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

}  // namespace ltx
