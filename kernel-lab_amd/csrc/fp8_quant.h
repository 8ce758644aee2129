// Rounding to OCP FP8 E4M3 with an fp32 scale, for the kernels that write 8 bits.
#pragma once

#include "hip_common.h"
#include "packs.h"

namespace kl {

constexpr float kE4M3Max = 448.0f;        // largest finite code
constexpr float kMinScale = 0x1p-126f;    // smallest scale: its reciprocal is finite, and 0 / scale is 0

// |v| where v is finite, else 0: what counts towards a scale.
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a < INFINITY ? a : 0.0f;  // false for NaN
}

// The scale that takes a largest magnitude to the largest code.
__device__ __forceinline__ float e4m3_scale(float most) { return fmaxf(most / kE4M3Max, kMinScale); }

// Two values rounded to nearest even, the first in the low byte of the low (or,
// HI, the high) half of `old`. What rounds past 448 and what is not finite
// becomes NaN: callers divide by a scale that leaves finite values at 448 at most.
template <bool HI>
__device__ __forceinline__ uint32_t e4m3x2(float a, float b, uint32_t old) {
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(a, b, static_cast<int>(old), HI));
}

__device__ __forceinline__ uint8_t e4m3(float v) { return static_cast<uint8_t>(e4m3x2<false>(v, 0.0f, 0) & 0xffu); }

// Four codes, the first in the lowest byte.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2<true>(c, d, e4m3x2<false>(a, b, 0));
}

// The value of byte N of a word of codes.
template <int N>
__device__ __forceinline__ float e4m3_value_at(uint32_t word) {
  return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), N);
}

// The value of a code.
__device__ __forceinline__ float e4m3_value(uint32_t code) { return e4m3_value_at<0>(code); }

// The codes of VEC values.
template <bool ALIGNED, int VEC>
__device__ __forceinline__ void store_codes(uint8_t* row, int off, const float (&c)[VEC]) {
  static_assert(VEC == 4 || VEC == 8, "a pack is four or eight elements");
  if constexpr (VEC == 8) {
    const u32x2 v = {e4m3x4(c[0], c[1], c[2], c[3]), e4m3x4(c[4], c[5], c[6], c[7])};
    store_at<ALIGNED>(row, off, v);
  } else {
    const uint32_t v = e4m3x4(c[0], c[1], c[2], c[3]);
    store_at<ALIGNED>(row, off, v);
  }
}

}  // namespace kl
