// glq_act.cuh -- activations of the feed-forward operators and their
// derivatives, in FP32, and the element types they are stored as.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "../../include/glq.h"

namespace glq {

template <typename T>
struct Elem16;

template <>
struct Elem16<__half> {
  static constexpr int kFormat = 0;  // tcgen05 kind::f16 operand format
  using Pair = __half2;
  __device__ static float to_f(__half v) { return __half2float(v); }
  __device__ static __half from_f(float v) { return __float2half_rn(v); }
  __device__ static float2 to_f2(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
  __device__ static uint32_t from_f2(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};

template <>
struct Elem16<__nv_bfloat16> {
  static constexpr int kFormat = 1;
  using Pair = __nv_bfloat162;
  __device__ static float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ static __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
  __device__ static float2 to_f2(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
  __device__ static uint32_t from_f2(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};

// sigmoid(x); exp(-x) overflows to infinity below -88, where the quotient is 0.
__device__ __forceinline__ float sigmoid_f(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

constexpr float kInvSqrt2 = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;  // density of the standard normal at 0
constexpr float kGeluC = 1.59576912160573071f;       // 2 sqrt(2 / pi): tanh(t) = 2 sigmoid(2 t) - 1
constexpr float kGeluCubic = 0.044715f;

// Phi(x) of the exact GELU from e = exp(-x^2 / 2), which its derivative needs
// anyway: erfc by formula 7.1.26 of Abramowitz and Stegun's Handbook of
// Mathematical Functions (absolute error below 1.5e-7, i.e. 7.5e-8 here; the
// 16-bit result's half-step is 2.4e-4 of it or more).  erff costs twice the
// instructions and bounded the backward kernel (4096 x 11008: 80 us).
__device__ __forceinline__ float normal_cdf(float x, float e) {
  const float t = __fdividef(1.0f, fmaf(0.3275911f * kInvSqrt2, fabsf(x), 1.0f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float tail = 0.5f * p * t * e;
  return x > 0.0f ? 1.0f - tail : tail;
}

// act(x).  ACT is a glq_activation; the callers switch on it once per tile.
template <int ACT>
__device__ __forceinline__ float act_f(float x) {
  if constexpr (ACT == GLQ_ACT_SILU) {
    return x * sigmoid_f(x);
  } else if constexpr (ACT == GLQ_ACT_GELU) {
    return x * normal_cdf(x, __expf(-0.5f * x * x));
  } else if constexpr (ACT == GLQ_ACT_GELU_TANH) {
    return x * sigmoid_f(kGeluC * x * (1.0f + kGeluCubic * x * x));
  } else if constexpr (ACT == GLQ_ACT_RELU) {
    return x > 0.0f || x != x ? x : 0.0f;  // NaN stays NaN
  } else {
    return x;
  }
}

// act(x) and act'(x).
template <int ACT>
__device__ __forceinline__ void act_grad_f(float x, float* value, float* slope) {
  if constexpr (ACT == GLQ_ACT_SILU) {
    const float s = sigmoid_f(x);
    *value = x * s;
    *slope = s * (1.0f + x * (1.0f - s));
  } else if constexpr (ACT == GLQ_ACT_GELU) {
    const float e = __expf(-0.5f * x * x);
    const float cdf = normal_cdf(x, e);
    *value = x * cdf;
    *slope = fmaf(x * kInvSqrt2Pi, e, cdf);
  } else if constexpr (ACT == GLQ_ACT_GELU_TANH) {
    // s (1 - s) is 0 long before x^2 overflows, and has to meet a finite factor.
    const float sq = fminf(x * x, 1e30f);
    const float s = sigmoid_f(kGeluC * x * (1.0f + kGeluCubic * sq));
    *value = x * s;
    *slope = s + x * s * (1.0f - s) * kGeluC * (1.0f + 3.0f * kGeluCubic * sq);
  } else if constexpr (ACT == GLQ_ACT_RELU) {
    *value = x > 0.0f || x != x ? x : 0.0f;
    *slope = x > 0.0f ? 1.0f : 0.0f;
  } else {
    *value = x;
    *slope = 1.0f;
  }
}

// Calls f(std::integral_constant<int, ACT>) for the run-time activation `act`.
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case GLQ_ACT_SILU: f(std::integral_constant<int, GLQ_ACT_SILU>()); break;
    case GLQ_ACT_GELU: f(std::integral_constant<int, GLQ_ACT_GELU>()); break;
    case GLQ_ACT_GELU_TANH: f(std::integral_constant<int, GLQ_ACT_GELU_TANH>()); break;
    case GLQ_ACT_RELU: f(std::integral_constant<int, GLQ_ACT_RELU>()); break;
    default: f(std::integral_constant<int, GLQ_ACT_NONE>()); break;
  }
}

}  // namespace glq
