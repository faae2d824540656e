// A tensor of a graph in HBM and the loads and stores of its formats (kernels.cuh says what they are).
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "tc_gemm_common.cuh"

namespace nb {

enum : int { FMT_F32 = 0, FMT_SPLIT = 1, FMT_I8 = 2, FMT_TF32 = 3, FMT_BF16X2 = 4 };

struct ActRef {
  float* p0 = nullptr;
  float* p1 = nullptr;
  int8_t* q = nullptr;
  int fmt = FMT_F32;
};

__device__ __forceinline__ float act_load(const ActRef& a, long long i) {
  if (a.fmt == FMT_I8) return static_cast<float>(a.q[i]);
  if (a.fmt == FMT_BF16X2) {
    const uint32_t h = reinterpret_cast<const uint16_t*>(a.p0)[i], m = reinterpret_cast<const uint16_t*>(a.p1)[i];
    return __fadd_rn(__uint_as_float(h << 16), __uint_as_float(m << 16));
  }
  float v = a.p0[i];
  if (a.fmt == FMT_SPLIT) v = __fadd_rn(v, a.p1[i]);
  return v;
}

__device__ __forceinline__ void act_store(const ActRef& a, long long i, float v) {
  if (a.fmt == FMT_I8) {
    a.q[i] = static_cast<int8_t>(static_cast<int>(v));
  } else if (a.fmt == FMT_F32) {
    a.p0[i] = v;
  } else if (a.fmt == FMT_BF16X2) {
    uint32_t hi, mid;
    split_bf16x2(v, 0.0f, hi, mid);
    reinterpret_cast<uint16_t*>(a.p0)[i] = static_cast<uint16_t>(hi & 0xffffu);
    reinterpret_cast<uint16_t*>(a.p1)[i] = static_cast<uint16_t>(mid & 0xffffu);
  } else {
    const float hi = round_tf32(v);
    a.p0[i] = hi;
    if (a.fmt == FMT_SPLIT) a.p1[i] = __fadd_rn(v, -hi);
  }
}

__device__ __forceinline__ float4 act_load4(const ActRef& a, long long i) {
  if (a.fmt == FMT_I8) {
    const char4 c = *reinterpret_cast<const char4*>(a.q + i);
    return make_float4(c.x, c.y, c.z, c.w);
  }
  if (a.fmt == FMT_BF16X2) {
    const uint2 h = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(a.p0) + i);
    const uint2 m = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(a.p1) + i);
    return make_float4(__fadd_rn(bf16_low(h.x), bf16_low(m.x)), __fadd_rn(bf16_high(h.x), bf16_high(m.x)),
                       __fadd_rn(bf16_low(h.y), bf16_low(m.y)), __fadd_rn(bf16_high(h.y), bf16_high(m.y)));
  }
  float4 v = *reinterpret_cast<const float4*>(a.p0 + i);
  if (a.fmt == FMT_SPLIT) {
    const float4 l = *reinterpret_cast<const float4*>(a.p1 + i);
    v.x = __fadd_rn(v.x, l.x);
    v.y = __fadd_rn(v.y, l.y);
    v.z = __fadd_rn(v.z, l.z);
    v.w = __fadd_rn(v.w, l.w);
  }
  return v;
}

__device__ __forceinline__ void act_store4(const ActRef& a, long long i, float4 v) {
  if (a.fmt == FMT_I8) {
    *reinterpret_cast<char4*>(a.q + i) =
        make_char4(static_cast<signed char>(static_cast<int>(v.x)),
                   static_cast<signed char>(static_cast<int>(v.y)),
                   static_cast<signed char>(static_cast<int>(v.z)),
                   static_cast<signed char>(static_cast<int>(v.w)));
  } else if (a.fmt == FMT_F32) {
    *reinterpret_cast<float4*>(a.p0 + i) = v;
  } else if (a.fmt == FMT_BF16X2) {
    uint2 h, m;
    split_bf16x2(v.x, v.y, h.x, m.x);
    split_bf16x2(v.z, v.w, h.y, m.y);
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.p0) + i) = h;
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.p1) + i) = m;
  } else {
    const float4 hi = make_float4(round_tf32(v.x), round_tf32(v.y), round_tf32(v.z), round_tf32(v.w));
    *reinterpret_cast<float4*>(a.p0 + i) = hi;
    if (a.fmt == FMT_SPLIT)
      *reinterpret_cast<float4*>(a.p1 + i) =
          make_float4(__fadd_rn(v.x, -hi.x), __fadd_rn(v.y, -hi.y), __fadd_rn(v.z, -hi.z),
                      __fadd_rn(v.w, -hi.w));
  }
}

}  // namespace nb
