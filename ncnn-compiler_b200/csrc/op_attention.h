// What the kernels of ncnn_b200_op_cross_attention share.
#pragma once

#include <array>
#include <tuple>
#include <type_traits>

#include "op_common.cuh"

namespace nb {

struct AttendParams {
  const void *q, *k, *v;
  void* o;
  int batch, lq, lk, heads, kv_heads, d;
  long long q_batch, q_row, q_head, k_batch, k_row, k_head, v_batch, v_row, v_head, o_batch, o_row, o_head;  // elements
  const int* lens;      // keys of each sequence, or null: lk
  const uint8_t* mask;  // [batch][lk], or null
  float scale;
};

// Probabilities of long keys and their sum are held this many powers of two higher.  fp16 has nothing below 2^-24 (2^-25 rounds to
// 0), and many keys of little weight behind one of much would be in the sum but not in the products (131071 keys of 2^-25.07 each:
// 0 instead of 0.0037).  With the slack of 2^8 that the running maximum has, probabilities stay at 2^15 or less, and weights from
// 2^-32 of a row's largest on are there.  bf16 has fp32's range.
template <class T> constexpr float kProbabilityLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;

}  // namespace nb
