// exp of arguments up to zero, as softmax terms and gates need it, and what is made of it.
#pragma once

#include "common.h"

namespace hpd {

// exp(x) for x <= 0 (NaN stays NaN): 2^(x log2 e) on the transcendental unit,
// with the rounding error of the product x log2 e, which would grow with |x|,
// and the constant's own put back to first order, 2^(t + d) = 2^t (1 + d ln 2).
// Within 2 units in the last place in seven instructions, where the library
// function takes about fifteen. Results below 2^-126 are zero.
__device__ __forceinline__ float exp_down(float x) {
  constexpr float kLog2e = 0x1.715476p+0f, kLog2eRest = 0x1.4ae0cp-26f, kLn2 = 0x1.62e43p-1f;
  const float t = x * kLog2e;
  const float d = __builtin_fmaf(x, kLog2eRest, __builtin_fmaf(x, kLog2e, -t));
  const float r = __builtin_amdgcn_exp2f(t);
  return x < -87.3f ? 0.0f : __builtin_fmaf(r, d * kLn2, r);
}
__device__ __forceinline__ double exp_down(double x) { return exp(x); }

// 1 / x for x in [1, 3]: the hardware's estimate (1 ulp) and a Newton step.
__device__ __forceinline__ float inverse(float x) {
  const float r = __builtin_amdgcn_rcpf(x);
  return __builtin_fmaf(r, __builtin_fmaf(-x, r, 1.0f), r);
}
__device__ __forceinline__ double inverse(double x) { return 1.0 / x; }

// keep = sigmoid(g) and take = 1 - keep, each to full precision where it is a normal
// number: one of them is 1 / (1 + exp(-|g|)), the other exp(-|g|) times it. Of a float
// past 87.3 the smaller one is 0. Of a NaN both are NaN.
template <typename T>
__device__ __forceinline__ void gates(T g, T& keep, T& take) {
  const T small = exp_down(-__builtin_elementwise_abs(g));
  const T large = inverse(T(1) + small);
  keep = g >= T(0) ? large : small * large;
  take = g >= T(0) ? small * large : large;
}

// log(1 + exp(v)) and its derivative sigmoid(v), to full relative precision:
// max(v, 0) + log(1 + e) with e = exp(-|v|), log(1 + e) = 2 artanh(t), t = e / (2 + e) <= 1/3,
// by its series; the first term left out is below 2^-26 of it.
__device__ __forceinline__ float softplus(float v, float& slope) {
  const float e = exp_down(-__builtin_elementwise_abs(v));
  const float t = e * inverse(2.0f + e), p = t * t, large = inverse(1.0f + e);
  float r = 1.0f / 13;
#pragma unroll
  for (int k = 11; k > 0; k -= 2) r = __builtin_fmaf(r, p, 1.0f / k);
  const float tail = 2.0f * t * r;
  slope = v >= 0.0f ? large : e * large;
  return v > 0.0f ? v + tail : v <= 0.0f ? tail : v;
}
__device__ __forceinline__ double softplus(double v, double& slope) {
  const double e = exp(-__builtin_elementwise_abs(v)), tail = log1p(e), large = 1.0 / (1.0 + e);
  slope = v >= 0 ? large : e * large;
  return v > 0 ? v + tail : v <= 0 ? tail : v;
}

}  // namespace hpd
