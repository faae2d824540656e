// What the kernels of ncnn_b200_op_inner_product_tokens share.
#pragma once

#include <cmath>
#include <type_traits>

#include "op_common.cuh"

namespace nb {

struct TokensParams {
  long long tokens;
  int k, n;
  long long q_pitch, weight_pitch, y_pitch;
  const int8_t* q;      // [tokens] rows of k integers
  const float* steps;   // [tokens]
  const int8_t* weight;
  const float* weight_steps;
  const float* bias;    // or null
  void* y;
  int act;
  int ranks;    // CTAs that share out a tile's K blocks
  int aligned;  // steps and bias of four channels can be read at a time
};

// A sum of integers (exact) before its activation: the sum and the product of the steps are rounded to fp32, then one fma.
__device__ __forceinline__ float tokens_sum(int sum, float step, float weight_step, float bias) {
  return fmaf(static_cast<float>(sum), step * weight_step, bias);
}
// Called, not inlined: results leave in unrolled loops, which a copy of these for every value makes too long for the instruction
// cache (64 tokens through 4096 x 11008, no activation: 5400 of a tile's 28000 clocks went into the last 16 values of each thread).
// Swish by the exponential of -|t|: that of -t passes fp32's largest number where t e^t is still far from its smallest.
__device__ __noinline__ float tokens_activate(float t, int act) {
  if (act == NCNN_B200_ACT_SWISH) {
    const float e = expf(-fabsf(t));
    return t * ((t < 0.0f ? e : 1.0f) / (1.0f + e));
  }
  return 0.5f * t * erfcf(t * -0.7071067811865476f);
}
// Swish for 16-bit results: good to (5 + 1.2 |t|) 2^-23, most of it the fast exponential's, whose error grows with its argument; 2^-16
// where results pass fp32's smallest number.
__device__ __forceinline__ float tokens_swish16(float t) {
  const float e = __expf(-fabsf(t));
  return t * __fdividef(t < 0.0f ? e : 1.0f, 1.0f + e);
}
// GELU for 16-bit results: erfc(z) = exp(-z^2) u P(u) with u = 1 / (1 + 0.65 z), P of degree 5 fitted to erfcx in equal relative
// error over z from 0 to 9.6 (2^-16.8; with the exponential, whose error grows with z^2, and the reciprocal, 2^-16 down to t = -10 and 2^-15
// below), where erfc(z) passes fp32's smallest number.
__device__ __forceinline__ float tokens_gelu16(float t) {
  const float z = fabsf(t) * 0.7071067811865476f;
  const float u = __fdividef(1.0f, fmaf(0.65f, z, 1.0f));
  float p = fmaf(0.14425337314605713f, u, -0.4733123183250427f);
  p = fmaf(p, u, 0.3572801351547241f);
  p = fmaf(p, u, 0.23145082592964172f);
  p = fmaf(p, u, 0.3739560544490814f);
  p = fmaf(p, u, 0.36638039350509644f);
  const float half = 0.5f * u * p * __expf(-z * z);
  return t * (t < 0.0f ? half : 1.0f - half);
}
// f is given what kind of loop it is: one with ReLU or nothing, one with the Swish or GELU of 16-bit results in line, or one that calls.
// (4096 x 4096 x 4096 to bf16: 56 us plain, GELU 122 when it was called.)
enum class Loop { kPlain, kSwish, kGelu, kCalls };
template <class T, class F>
__device__ __forceinline__ void tokens_by_activation(int act, F&& f) {
  if (act == NCNN_B200_ACT_NONE || act == NCNN_B200_ACT_RELU) f(std::integral_constant<Loop, Loop::kPlain>{});
  else if (sizeof(T) == 2 && act == NCNN_B200_ACT_SWISH) f(std::integral_constant<Loop, Loop::kSwish>{});
  else if (sizeof(T) == 2 && act == NCNN_B200_ACT_GELU) f(std::integral_constant<Loop, Loop::kGelu>{});
  else f(std::integral_constant<Loop, Loop::kCalls>{});
}
template <class T, class LOOP>
__device__ __forceinline__ T tokens_result(LOOP, int sum, float step, float weight_step, float bias, int act) {
  const float t = tokens_sum(sum, step, weight_step, bias);
  if constexpr (LOOP::value == Loop::kPlain) {
    const float least = act == NCNN_B200_ACT_RELU ? 0.0f : -INFINITY;
    return op_put<T>(t < least ? least : t);  // (a NaN stays one)
  }
  if constexpr (LOOP::value == Loop::kSwish) return op_put<T>(tokens_swish16(t));
  if constexpr (LOOP::value == Loop::kGelu) return op_put<T>(tokens_gelu16(t));
  return op_put<T>(tokens_activate(t, act));
}

}  // namespace nb
