// Activations on accumulators (kernels_layered.hip, kernels_experts.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "pointwise.h"

namespace ponni_hip {

// The usual activations of fp32 plans on the accumulators.  The hardware forms
// of the generated kernels (pointwise.h) are off by up to an ulp of one near
// zero (tanh) and by |x| / 2 ulp (sigmoid and SiLU of negative x), which libm's
// (GENERIC's) are not: largest relative errors, libm / hardware forms / these,
// tanh on -2..-0.55 1.5e-7 / 3.5e-7 / 2.0e-7, sigmoid on -40..-12 1.8e-7 /
// 1.9e-6 / 2.0e-7.  64-1024-1024-64 tanh, 65,536 columns: 1302 us with the
// hardware forms, 1307 with these, 1325 with libm's; 40-700-30 sigmoid 129, 132, 170.
// e^v: 2^(v log2 e) with the rounding error of the product carried along.
__device__ inline float exp_f32(float v) {
  constexpr float kLog2eRest = 1.9259630e-8f, kLn2 = 0.69314718f;
  float const t = v * kLog2e;
  float const rest = fmaf(v, kLog2eRest, fmaf(v, kLog2e, -t));
  float const e = __builtin_amdgcn_exp2f(t);
  return __builtin_fabsf(t) < 128.0f ? fmaf(e, rest * kLn2, e) : e;
}
// x / (1 + e): the hardware's reciprocal and one correction of the quotient.
__device__ inline float over_one_plus(float x, float e) {
  float const d = 1.0f + e, r = __builtin_amdgcn_rcpf(d), q = x * r;
  return __builtin_amdgcn_div_fixupf(fmaf(fmaf(-d, q, x), r, q), d, x);
}
__device__ inline float sigmoid_f32(float x) { return over_one_plus(1.0f, exp_f32(-x)); }
__device__ inline float silu_f32(float x) { return over_one_plus(x, exp_f32(-x)); }
// ponni_Gelu.h:48-53: x sigmoid(2u), u = sqrt(2/pi) (x + 0.044715 x^3)
__device__ inline float gelu_tanh_f32(float x) {
  constexpr float c = -2.0f * 0.79788456080286535588f;
  return over_one_plus(x, exp_f32(x * fmaf(0.044715f * c, x * x, c)));
}
// 1 - 2 e / (1 + e) of |x|, e = e^(-2|x|); near zero, where that cancels, x p(x^2)
// with p a Chebyshev fit of tanh(x) / x (4.5e-9 on |x| <= 0.55).
__device__ inline float tanh_f32(float x) {
  float const s = x * x;
  float q = fmaf(s, -0.00623885f, 0.02104217f);
  q = fmaf(s, q, -0.05384337f);
  q = fmaf(s, q, 0.13332468f);
  q = fmaf(s, q, -0.33333311f);
  float const a = __builtin_fabsf(x);
  float const e = __builtin_amdgcn_exp2f(-2.0f * kLog2e * a);
  float const r = a <= 0.55f ? fmaf(a * s, q, a) : 1.0f + over_one_plus(-2.0f * e, e);
  return __builtin_copysignf(r, x);
}
// 16-bit plans: the hardware form, and x itself where that is closer than the
// type resolves (below 2^-7 tanh(x) is x to 2e-5; the form's error there is an
// ulp of fp32's one, more than an ulp of a small fp16 result, and all of a bf16 one at 1e-8).  fp16
// 24-1100-200, 40,000 columns: 84 us without, 87 with; a chain of expert layers 64-256-256-256-64,
// 1,000,000 columns: 489 and 510.
__device__ inline float tanh_half(float x) { return __builtin_fabsf(x) < 0.0078125f ? x : act_tanh_fast(x); }

}  // namespace ponni_hip
