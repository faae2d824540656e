// What the kernels of ncnn_b200_op_cross_attention share.
#pragma once

#include <array>
#include <tuple>

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

}  // namespace nb
