// Element types of the expert kernels and the 4-bit conversions.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

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
// Two elements into byte AT of `word`: a, b over scale_value, a power of two, to
// nearest, ties to the even code, at most 6, by the hardware's conversion.
template <int AT, class S> __device__ inline unsigned mx4_pair(unsigned word, S a, S b, float scale_value) {
  typedef S S2 __attribute__((ext_vector_type(2)));
  if constexpr (std::is_same_v<S, float>) return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, a, b, scale_value, AT);
  else if constexpr (std::is_same_v<S, _Float16>)
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, S2{a, b}, scale_value, AT);
  else return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, S2{a, b}, scale_value, AT);
}
// Eight elements, element(i) the i-th, as a word.
template <class F> __device__ inline unsigned mx4_word(float scale_value, F&& element) {
  unsigned w = 0;
  w = mx4_pair<0>(w, element(0), element(1), scale_value);
  w = mx4_pair<1>(w, element(2), element(3), scale_value);
  w = mx4_pair<2>(w, element(4), element(5), scale_value);
  return mx4_pair<3>(w, element(6), element(7), scale_value);
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
