// The activations of nn.FusedLinear and nn.GroupedLinear, and their slopes, in FP32.
//   relu  z > 0 ? z : 0 (what nn.Threshold(0, 0) gives, a NaN included)
//   gelu  z P(z), P the standard normal distribution's integral
//   silu  z / (1 + exp(-z))
#ifndef THC_NN_ACTIVATION_CUH
#define THC_NN_ACTIVATION_CUH

#include "thc_internal.h"

#include <type_traits>

namespace thc {

enum : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3, kActs = 4 };

#ifdef __CUDACC__
// P(z) = erfc(-z / sqrt 2) / 2.  For z < 0 the Chebyshev fit of Numerical Recipes (section 6.2, `erfcc`), erfc(a) = t exp(-a^2 + q(t)) with
// t = 1 / (1 + a / 2), whose relative error is below 1.2e-7 however small erfc is; for z > 0 one minus that of -z.  -a^2 is -z^2 / 2, rounded
// once with q(t).  No branch and some 20 instructions, which the epilogues below pay for every value (erfcf takes about three
// times that).
__device__ __forceinline__ float normal_below(float z) {
  const float t = __fdividef(1.f, fmaf(fabsf(z), 0.35355339059327376f, 1.f));
  float q = 0.17087277f;
  q = fmaf(t, q, -0.82215223f);
  q = fmaf(t, q, 1.48851587f);
  q = fmaf(t, q, -1.13520398f);
  q = fmaf(t, q, 0.27886807f);
  q = fmaf(t, q, -0.18628806f);
  q = fmaf(t, q, 0.09678418f);
  q = fmaf(t, q, 0.37409196f);
  q = fmaf(t, q, 1.00002368f);
  q = fmaf(t, q, -1.26551223f);
  const float p = 0.5f * t * __expf(fmaf(-0.5f * z, z, q));
  return z > 0.f ? 1.f - p : p;
}
template <int ACT> __device__ __forceinline__ float activation(float z) {
  if constexpr (ACT == kActRelu) return z > 0.f ? z : 0.f;
  else if constexpr (ACT == kActGelu) return z * normal_below(z);
  else if constexpr (ACT == kActSilu) return z / (1.f + expf(-z));
  else return z;
}
template <int ACT> __device__ __forceinline__ float activation_slope(float z) {
  if constexpr (ACT == kActRelu) return z > 0.f ? 1.f : 0.f;
  else if constexpr (ACT == kActGelu) return fmaf(z * 0.39894228040143268f, expf(-0.5f * z * z), normal_below(z));
  else if constexpr (ACT == kActSilu) {
    const float s = 1.f / (1.f + expf(-z));
    return s * fmaf(z, 1.f - s, 1.f);
  } else return 1.f;
}
#endif
// f(integral constant act)
template <class F> __host__ __device__ __forceinline__ void with_activation(int act, F f) {
  if (act == kActRelu) f(std::integral_constant<int, kActRelu>());
  else if (act == kActGelu) f(std::integral_constant<int, kActGelu>());
  else if (act == kActSilu) f(std::integral_constant<int, kActSilu>());
  else f(std::integral_constant<int, kActNone>());
}

}  // namespace thc

#endif
