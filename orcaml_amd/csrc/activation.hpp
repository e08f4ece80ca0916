// The activations of the fused Linear (ORCA_HIP_ACT_*) and their derivatives, in fp32.
//
// They run in epilogues whose block then multiplies nothing (a 256 x 256 tile with the library's erfc
// took 45 us of a 640 us product), so each is a few arithmetic instructions around the hardware's
// exponential and reciprocal (both within an ulp): a few 2^-24 of 1 + |z|, below the product's own error.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/orca_hip.h"

namespace orca_hip {
namespace {

// exp2(inf) is infinity and its reciprocal 0: no NaN for finite x.
__device__ __forceinline__ float logistic(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

// 2 sqrt(2 / pi) (z + 0.044715 z^3): tanh(u) = 2 logistic(2 u) - 1, so gelu_tanh(z) = z logistic(2 u)
__device__ __forceinline__ float gelu_tanh_2u(float z) {
  return 1.5957691216057308f * z * (1.0f + 0.044715f * z * z);
}

// exp(-z^2 / 2)
__device__ __forceinline__ float gauss(float z) { return __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z); }

// Phi(z) = erfc(-z / sqrt 2) / 2, given gauss(z): the upper tail Q(|z|) is gauss(z) times a function that
// falls smoothly from 1/2, here t times a polynomial in t = 1 / (1 + 0.21 |z|).  Coefficients: a
// weighted least-squares fit of the scaled erfc, iterated towards equal relative errors on [0, 14]
// (2.4e-8; with constants and arithmetic in fp32 4.4e-7).  The tail is a product, so its error stays relative, where
// 1 + erf would cancel; it grows with gauss's, whose exponent is rounded: 2.5 * 2^-24 of z^2 / 2 (in all 2.0e-6 at
// z = -6, 7.8e-6 at -12.5), about what z's own rounding to fp32 does to Phi there (z^2 * 2^-24).
__device__ __forceinline__ float normal_cdf(float z, float g) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.21f, fabsf(z), 1.0f));
  float r = -0.07167498f;
  r = fmaf(r, t, 0.2836754620f);
  r = fmaf(r, t, -0.3304254413f);
  r = fmaf(r, t, 0.3495901823f);
  r = fmaf(r, t, -0.0940513834f);
  r = fmaf(r, t, 0.1249249429f);
  r = fmaf(r, t, 0.0691790804f);
  r = fmaf(r, t, 0.0850706771f);
  r = fmaf(r, t, 0.0837114677f);
  const float q = r * t * g;
  return z > 0.0f ? 1.0f - q : q;
}

// act(z) of N values.
template <int N, class V>
__device__ __forceinline__ void activations(int act, const V& z, V& y) {
  switch (act) {
    case ORCA_HIP_ACT_RELU:
#pragma unroll
      for (int j = 0; j < N; ++j) y[j] = z[j] > 0.0f ? z[j] : 0.0f;
      break;
    case ORCA_HIP_ACT_GELU:
#pragma unroll
      for (int j = 0; j < N; ++j) y[j] = z[j] * normal_cdf(z[j], gauss(z[j]));
      break;
    case ORCA_HIP_ACT_GELU_TANH:
#pragma unroll
      for (int j = 0; j < N; ++j) y[j] = z[j] * logistic(gelu_tanh_2u(z[j]));
      break;
    case ORCA_HIP_ACT_SILU:
#pragma unroll
      for (int j = 0; j < N; ++j) y[j] = z[j] * logistic(z[j]);
      break;
    default: y = z;
  }
}

// g * act'(z) of N values.
template <int N, class V>
__device__ __forceinline__ void activation_slopes(int act, const V& z, V& g) {
  switch (act) {
    case ORCA_HIP_ACT_RELU:
#pragma unroll
      for (int j = 0; j < N; ++j) g[j] = z[j] > 0.0f ? g[j] : 0.0f;
      break;
    case ORCA_HIP_ACT_GELU:
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float e = gauss(z[j]);
        g[j] = g[j] * (normal_cdf(z[j], e) + z[j] * (0.39894228040143268f * e));
      }
      break;
    case ORCA_HIP_ACT_GELU_TANH:
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float s = logistic(gelu_tanh_2u(z[j])), t = s * (1.0f - s);
        // where the logistic is 0 or 1 in fp32 the second term is below its last place, and z^2 may overflow
        g[j] = g[j] * (t == 0.0f ? s : s + z[j] * t * (1.5957691216057308f * (1.0f + 0.134145f * z[j] * z[j])));
      }
      break;
    case ORCA_HIP_ACT_SILU:
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float s = logistic(z[j]);
        g[j] = g[j] * (s * (1.0f + z[j] * (1.0f - s)));
      }
      break;
    default: break;
  }
}

}  // namespace
}  // namespace orca_hip
