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
// P(-a) = erfc(a / sqrt 2) / 2 for a >= 0 by the Chebyshev fit of Numerical Recipes (section 6.2, `erfcc`): erfc(x) = t exp(-x^2 + q(t)) with
// t = 1 / (1 + x / 2), whose own relative error is below 1.2e-7 however small erfc is.  Here in powers of two, with the half in q: its
// coefficients divided by ln 2, and one less.  The exponent is rounded to FP32, which its power multiplies by its size: gelu(-z) is off by 4e-7 of itself up to
// z = 1, by about (1 + z^2) 2^-24 beyond 4 (1.9e-6 at 6, 8e-6 at 13), as measured against 64 bits.  The epilogues of the products pay for every instruction 128
// times a thread: 15 of them, no branch (erfcf takes some three times that).
__device__ __forceinline__ float normal_tail(float a) {
  float t, e;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(a, 0.35355339059327376f, 1.f)));
  float q = 0.246517298f;
  q = fmaf(t, q, -1.186114945f);
  q = fmaf(t, q, 2.147474464f);
  q = fmaf(t, q, -1.637753152f);
  q = fmaf(t, q, 0.402321582f);
  q = fmaf(t, q, -0.268756860f);
  q = fmaf(t, q, 0.139630057f);
  q = fmaf(t, q, 0.539700616f);
  q = fmaf(t, q, 1.442729204f);
  q = fmaf(t, q, -2.825748218f);
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(-0.72134752044448170f * a, a, q)));
  return t * e;
}
__device__ __forceinline__ float normal_below(float z) {
  const float p = normal_tail(fabsf(z));
  return z > 0.f ? 1.f - p : p;
}
// z P(z) = max(z, 0) - |z| P(-|z|); beyond 30 the second term is zero, and an infinite z would make it none.
__device__ __forceinline__ float gelu(float z) {
  const float a = fminf(fabsf(z), 30.f);
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(z), "f"(0.f));
  return fmaf(-a, normal_tail(a), m);
}
// z / (1 + exp(-z)) through e = exp(-|z|), which does not overflow: z / (1 + e), and e times that for z < 0.  The exponent's product with log2 e
// is taken in two parts, so that e is as exact for large |z| as for small.
__device__ __forceinline__ float silu(float z) {
  const float a = fminf(fabsf(z), 128.f), s = a * -1.44269504f;
  const float rest = fmaf(a, -1.92596303e-8f, fmaf(a, -1.44269504f, -s));
  float e, t;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(s));
  e = fmaf(e, rest * 0.69314718f, e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(1.f + e));
  return z * (z < 0.f ? e * t : t);
}
template <int ACT> __device__ __forceinline__ float activation(float z) {
  if constexpr (ACT == kActRelu) return z > 0.f ? z : 0.f;
  else if constexpr (ACT == kActGelu) return gelu(z);
  else if constexpr (ACT == kActSilu) return silu(z);
  else return z;
}
template <int ACT> __device__ __forceinline__ float activation_slope(float z) {
  if constexpr (ACT == kActRelu) return z > 0.f ? 1.f : 0.f;
  else if constexpr (ACT == kActGelu) {          // P(z) + z exp(-z^2 / 2) / sqrt(2 pi)
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-0.72134752044448170f * z * z));
    return fmaf(z * 0.39894228040143268f, e, normal_below(z));
  } else if constexpr (ACT == kActSilu) {        // s (1 + z (1 - s)) with s = 1 / (1 + exp(-z)), neither s nor 1 - s a difference
    float e, t;
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(fminf(fabsf(z), 128.f) * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(1.f + e));
    const float u = e * t, s = z < 0.f ? u : t, rest = z < 0.f ? t : u;
    return s * fmaf(z, rest, 1.f);
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
