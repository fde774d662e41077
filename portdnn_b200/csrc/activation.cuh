// The activations that the fused matrix product and the norms around a block apply, and their derivatives, as
// functions of the value they are applied to.
#pragma once

#include "common.cuh"

#include <type_traits>

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

// ---- for results of 16 bits, and with the activation known at compile time --------------------------------
__device__ __forceinline__ float reciprocal_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Phi(z), the normal distribution's function, for two z: a polynomial in t = 1 / (1 + p |x|) times e = exp(-x^2), x = z / sqrt(2)
// (Abramowitz and Stegun, 7.1.26, with half of their coefficients; off by 7.5e-8 at most, in the tail relative to e).
__device__ __forceinline__ float2 normal_cdf(float2 z, float2& e) {
  const float2 s = mul2(mul2(z, both(-0.72134752f)), z);  // -x^2 log2(e)
  e = make_float2(exp2_approx(s.x), exp2_approx(s.y));
  const float2 d = fma2(make_float2(fabsf(z.x), fabsf(z.y)), both(0.23164189f), both(1.f));
  const float2 t = make_float2(reciprocal_approx(d.x), reciprocal_approx(d.y));
  float2 q = fma2(t, both(0.5307027145f), both(-0.7265760135f));
  q = fma2(q, t, both(0.7107068705f));
  q = fma2(q, t, both(-0.142248368f));
  q = fma2(q, t, both(0.127414796f));
  q = mul2(mul2(q, t), e);  // Phi(-|z|)
  return make_float2(z.x >= 0.f ? 1.f - q.x : q.x, z.y >= 0.f ? 1.f - q.y : q.y);
}
// (the quotient is 0 where the exponential is beyond 2^126)
__device__ __forceinline__ float fast_sigmoid(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

// The activation ACT, and its slope, of two values for results of type T: the functions above for fp32, within 2^-20 of
// 1 + |z| for 16 bits.
template <int ACT, typename T>
__device__ __forceinline__ float2 value_of(float2 z) {
  if constexpr (sizeof(T) == 2 && ACT == PDNN_ACT_GELU) {
    float2 e;
    return mul2(z, normal_cdf(z, e));
  } else if constexpr (sizeof(T) == 2 && ACT == PDNN_ACT_SILU) {
    return make_float2(z.x * fast_sigmoid(z.x), z.y * fast_sigmoid(z.y));
  } else if constexpr (sizeof(T) == 2 && ACT == PDNN_ACT_SIGMOID) {
    return make_float2(fast_sigmoid(z.x), fast_sigmoid(z.y));
  } else {
    return make_float2(activate(ACT, z.x), activate(ACT, z.y));
  }
}
template <int ACT, typename T>
__device__ __forceinline__ float2 slope_of(float2 z) {
  if constexpr (sizeof(T) == 2 && ACT == PDNN_ACT_GELU) {
    float2 e;
    const float2 c = normal_cdf(z, e);
    return fma2(mul2(z, both(0.39894228f)), e, c);
  } else if constexpr (sizeof(T) == 2 && (ACT == PDNN_ACT_SILU || ACT == PDNN_ACT_SIGMOID)) {
    const float2 s = make_float2(fast_sigmoid(z.x), fast_sigmoid(z.y)), r = fma2(s, both(-1.f), both(1.f));
    return mul2(s, ACT == PDNN_ACT_SIGMOID ? r : fma2(z, r, both(1.f)));
  } else {
    return make_float2(activation_slope(ACT, z.x), activation_slope(ACT, z.y));
  }
}

template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  switch (act) {
    case PDNN_ACT_RELU: f(std::integral_constant<int, PDNN_ACT_RELU>{}); break;
    case PDNN_ACT_TANH: f(std::integral_constant<int, PDNN_ACT_TANH>{}); break;
    case PDNN_ACT_RELU6: f(std::integral_constant<int, PDNN_ACT_RELU6>{}); break;
    case PDNN_ACT_GELU: f(std::integral_constant<int, PDNN_ACT_GELU>{}); break;
    case PDNN_ACT_SILU: f(std::integral_constant<int, PDNN_ACT_SILU>{}); break;
    case PDNN_ACT_SIGMOID: f(std::integral_constant<int, PDNN_ACT_SIGMOID>{}); break;
    default: f(std::integral_constant<int, PDNN_ACT_NONE>{}); break;
  }
}

}  // namespace pdnn
