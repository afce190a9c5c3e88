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

constexpr float kInvSqrt2Pi = 0.39894228040143268f;  // density of the standard normal at 0
constexpr float kGeluC = 1.59576912160573071f;       // 2 sqrt(2 / pi): tanh(t) = 2 sigmoid(2 t) - 1
constexpr float kGeluCubic = 0.044715f;

// exp(-x^2 / 2).
__device__ __forceinline__ float gauss(float x) {
  float e;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(x * x * -0.72134752044448170f));  // -1 / (2 ln 2)
  return e;
}

// Phi(-|x|) of the exact GELU from e = gauss(x), which its derivative needs
// anyway.  For negative x gelu(x) is x times this tail, so the error has to be
// small against the tail itself: Phi(-|x|) / e falls smoothly from 1/2 like
// 1 / |x|, and is t times a polynomial in t = 1 / (1 + 0.36 |x|), fitted here
// (least squares of the relative error, reweighted towards its least maximum,
// |x| up to 15): within 1.4e-6 of it with 32-bit evaluation.  e adds the
// roundings of its argument, 2^-23 x^2 at most; the half-step of a 16-bit
// result is 4.9e-4 or more.  erff costs twice the instructions and bounded the
// backward kernel (4096 x 11008: 80 us), and 1 + erff cancels in the tail.
__device__ __forceinline__ float normal_tail(float x, float e) {
  const float t = __fdividef(1.0f, fmaf(0.36f, fabsf(x), 1.0f));
  float p = fmaf(0.0465226406f, t, -0.17793574f);
  p = fmaf(p, t, 0.178466204f);
  p = fmaf(p, t, 0.0282575622f);
  p = fmaf(p, t, 0.13909894f);
  p = fmaf(p, t, 0.14188469f);
  p = fmaf(p, t, 0.143705188f);
  return p * t * e;
}

// act(x).  ACT is a glq_activation; the callers switch on it once per tile.
template <int ACT>
__device__ __forceinline__ float act_f(float x) {
  if constexpr (ACT == GLQ_ACT_SILU) {
    return x * sigmoid_f(x);
  } else if constexpr (ACT == GLQ_ACT_GELU) {
    // x Phi(x) = max(x, 0) - |x| Phi(-|x|); the cap keeps infinity from its tail of 0.
    return fmaf(-fabsf(fminf(x, 1e30f)), normal_tail(x, gauss(x)), fmaxf(x, 0.0f));
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
    const float e = gauss(x);
    const float tail = normal_tail(x, e);
    const float cdf = x > 0.0f ? 1.0f - tail : tail;
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
