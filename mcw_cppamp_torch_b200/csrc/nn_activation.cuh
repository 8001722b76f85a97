// The activations of nn.FusedLinear and nn.GroupedLinear, and their slopes, in FP32.
//   relu  z > 0 ? z : 0 (what nn.Threshold(0, 0) gives, a NaN included)
//   gelu  z P(z), P the standard normal distribution's integral: erfc(-z / sqrt 2) / 2, which keeps its bits where P is small
//   silu  z / (1 + exp(-z))
#ifndef THC_NN_ACTIVATION_CUH
#define THC_NN_ACTIVATION_CUH

#include "thc_internal.h"

namespace thc {

enum : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3, kActs = 4 };

#ifdef __CUDACC__
__device__ __forceinline__ float normal_below(float z) { return 0.5f * erfcf(z * -0.70710678118654752f); }
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
// f(integral constant act)
template <class F> void with_activation(int act, F f) {
  switch (act) {
    case kActRelu: f(std::integral_constant<int, kActRelu>()); return;
    case kActGelu: f(std::integral_constant<int, kActGelu>()); return;
    case kActSilu: f(std::integral_constant<int, kActSilu>()); return;
    default: f(std::integral_constant<int, kActNone>());
  }
}
#endif

}  // namespace thc

#endif
