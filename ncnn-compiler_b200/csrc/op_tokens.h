// What the kernels of ncnn_b200_op_inner_product_tokens share.
#pragma once

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
};

template <class T>
__device__ __forceinline__ float tokens_activate(float t, int act) {
  if (act == NCNN_B200_ACT_RELU) return t > 0.0f ? t : t == t ? 0.0f : t;  // (a NaN stays one)
  if (act == NCNN_B200_ACT_SWISH) return sizeof(T) == 4 ? t / (1.0f + expf(-t)) : __fdividef(t, 1.0f + __expf(-t));  // (16 bits: good to 2^-20)
  if (act == NCNN_B200_ACT_GELU) return 0.5f * t * erfcf(t * -0.7071067811865476f);
  return t;
}
// A sum of integers (exact) as the result: the sum and the product of the steps are rounded to fp32, then one fma.
template <class T>
__device__ __forceinline__ float tokens_result(int sum, float step, float weight_step, float bias, int act) {
  return tokens_activate<T>(fmaf(static_cast<float>(sum), step * weight_step, bias), act);
}

}  // namespace nb
