// The activations of the fused Linear (ORCA_HIP_ACT_*) and their derivatives, in fp32.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/orca_hip.h"

namespace orca_hip {
namespace {

// exp(-x) overflows to infinity for very negative x and its reciprocal is then 0: no NaN.
__device__ __forceinline__ float logistic(float x) { return 1.0f / (1.0f + expf(-x)); }

// 2 sqrt(2 / pi) (z + 0.044715 z^3): tanh(u) = 2 logistic(2 u) - 1, so gelu_tanh(z) = z logistic(2 u)
__device__ __forceinline__ float gelu_tanh_2u(float z) {
  return 1.5957691216057308f * z * (1.0f + 0.044715f * z * z);
}

__device__ __forceinline__ float activation(int act, float z) {
  switch (act) {
    case ORCA_HIP_ACT_RELU: return z > 0.0f ? z : 0.0f;
    // the complementary error function keeps the tail's relative precision, where 1 + erf cancels
    case ORCA_HIP_ACT_GELU: return z * (0.5f * erfcf(-0.70710678118654752f * z));
    case ORCA_HIP_ACT_GELU_TANH: return z * logistic(gelu_tanh_2u(z));
    case ORCA_HIP_ACT_SILU: return z * logistic(z);
    default: return z;
  }
}

__device__ __forceinline__ float activation_slope(int act, float z) {
  switch (act) {
    case ORCA_HIP_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case ORCA_HIP_ACT_GELU:
      return 0.5f * erfcf(-0.70710678118654752f * z) + z * (0.39894228040143268f * expf(-0.5f * z * z));
    case ORCA_HIP_ACT_GELU_TANH: {
      const float s = logistic(gelu_tanh_2u(z)), t = s * (1.0f - s);
      // where the logistic is 0 or 1 in fp32 the second term is below its last place, and z^2 may overflow
      return t == 0.0f ? s : s + z * t * (1.5957691216057308f * (1.0f + 0.134145f * z * z));
    }
    case ORCA_HIP_ACT_SILU: {
      const float s = logistic(z);
      return s * (1.0f + z * (1.0f - s));
    }
    default: return 1.0f;
  }
}

}  // namespace
}  // namespace orca_hip
