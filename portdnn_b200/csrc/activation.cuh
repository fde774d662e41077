// The activations that the fused matrix product and the norms around a block apply, and their derivatives, as
// functions of the value they are applied to.
#pragma once

#include "common.cuh"

namespace pdnn {

inline bool known_activation(int act) {
  return (act >= PDNN_ACT_NONE && act <= PDNN_ACT_RELU6) || (act >= PDNN_ACT_GELU && act <= PDNN_ACT_SIGMOID);
}

// 1 / (1 + exp(-z)).  exp(-z) overflows to infinity below -88, and the quotient is then zero.
__device__ __forceinline__ float sigmoid_f32(float z) { return 1.f / (1.f + expf(-z)); }

// NaN stays NaN (fmaxf would drop it).
__device__ __forceinline__ float activate(int act, float z) {
  switch (act) {
    case PDNN_ACT_RELU: return z < 0.f ? 0.f : z;
    case PDNN_ACT_TANH: return tanhf(z);
    case PDNN_ACT_RELU6: return z < 0.f ? 0.f : z > 6.f ? 6.f : z;
    case PDNN_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678f));
    case PDNN_ACT_SILU: return z * sigmoid_f32(z);
    case PDNN_ACT_SIGMOID: return sigmoid_f32(z);
    default: return z;
  }
}

__device__ __forceinline__ float activation_slope(int act, float z) {
  switch (act) {
    case PDNN_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case PDNN_ACT_TANH: {
      const float t = tanhf(z);
      return 1.f - t * t;
    }
    case PDNN_ACT_RELU6: return z > 0.f && z < 6.f ? 1.f : 0.f;
    case PDNN_ACT_GELU:  // the normal distribution's function, plus z times its density
      return 0.5f * (1.f + erff(z * 0.70710678f)) + z * 0.39894228f * expf(-0.5f * z * z);
    case PDNN_ACT_SILU: {
      const float s = sigmoid_f32(z);
      return s * (1.f + z * (1.f - s));
    }
    case PDNN_ACT_SIGMOID: {
      const float s = sigmoid_f32(z);
      return s * (1.f - s);
    }
    default: return 1.f;
  }
}

}  // namespace pdnn
