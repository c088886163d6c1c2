// Element types of the expert kernels and the 4-bit conversions.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/ponni_hip.h"

namespace ponni_hip {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// Calls f(element of the type) for a ponni_dtype of 16 or 32 bits; false for any other.
template <class F> inline bool with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case PONNI_F32: f(float{}); return true;
    case PONNI_F16: f(_Float16{}); return true;
    case PONNI_BF16: f(__bf16{}); return true;
    default: return false;
  }
}

// The scale of a block whose largest magnitude is `amax`, as the exponent biased
// by 127: floor(log2 amax) - 2 (6 is the largest magnitude of a 4-bit element,
// 2^2 its binade), at least -127.  255 marks a block that holds NaN or an
// infinity.  (The exponent field of a float below its normal range is 0; such
// blocks take the smallest scale.)
__device__ inline unsigned mx4_scale(float amax) {
  unsigned const e = (__builtin_bit_cast(unsigned, amax) >> 23) & 255u;
  return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}
// 2^(127 - scale): exact, also for scale 0 (2^127); 0 for a NaN block.
__device__ inline float mx4_inverse(unsigned scale) {
  return scale == 255u ? 0.0f : __builtin_bit_cast(float, (254u - scale) << 23);
}
// Sign and 3 bits of v = x * 2^(127 - scale), to nearest, ties to the even code,
// at most 6: the values are 0, 0.5, ..., 2 in steps of 0.5, to 4 in steps of 1, 6.
__device__ inline unsigned mx4_code(float v) {
  float const s = __builtin_fabsf(v);
  float const c = s < 2.0f ? __builtin_rintf(2.0f * s) : s < 4.0f ? 2.0f + __builtin_rintf(s)
                                                                  : 4.0f + __builtin_rintf(0.5f * s);
  unsigned const m = unsigned(c < 7.0f ? c : 7.0f);
  return m | ((__builtin_bit_cast(unsigned, v) >> 31) << 3);
}
// Value of a 4-bit element: its three bits are the last exponent and first
// mantissa bits of a float 2^126 times smaller (also below the binades: 0.5).
__device__ inline float mx4_value(unsigned code) {
  unsigned const bits = ((code & 7u) << 22) | ((code & 8u) << 28);
  return __builtin_bit_cast(float, bits) * 0x1p126f;
}
__device__ inline float mx4_scale_value(unsigned scale) {
  return __builtin_bit_cast(float, scale == 255u ? 0x7fc00000u : scale == 0u ? 0x00400000u : scale << 23);
}

}  // namespace ponni_hip
