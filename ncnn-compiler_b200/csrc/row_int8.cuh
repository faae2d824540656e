// Rows of numbers as 8-bit integers and a step, found in the row itself: what products of tokens and the cache share.
//
//   top = max |x|, step = top / 127, q = 127 x / top to the nearest whole number, halves away from zero
//
// The integers are those of real arithmetic, so that no order of operations shows in them.  One fma with 1.5 2^23 rounds a product
// to a whole number, whose low byte is the integer: halves would go to the even one.
// * 16-bit elements: x = X 2^e with X below 2^11, top = A 2^f.  127 x / top differs from every half that it does not equal by
//   1 / (2 A 2^(f - e)) = |127 x / top| / (254 X) or more: 2^-19 of itself.  The factor 127 / top is taken 2^-21 too large (its two
//   roundings are 2^-23): halves go up, away from zero on either side, and nothing else passes one.
// * fp32 elements: the product is good to 127 2^-24 < 2^-17; where it is that near to a half, the quotient is taken in 64 bits.
//   (Halves are 2^-33 of a quotient away or more: 127 x is exact in 64 bits, and the quotient's rounding 2^-53.)
#pragma once

#include "op_common.cuh"

namespace nb {

constexpr float kRowLeast = 7.888609052210118e-31f;  // 2^-100: rows below are zeros
constexpr float kRowMagic = 12582912.0f;             // 1.5 2^23

// |x| as an integer that orders infinities and NaN above all numbers
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The largest magnitude of some elements so far: 16-bit types as the larger of two halves' bits, which row_top_bits joins and
// makes fp32's.
template <class T, int V>
__device__ __forceinline__ uint32_t row_top(const OpVec<T, V>& v, uint32_t top) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
  } else if constexpr (sizeof(T) == 2) {
    top = __vmaxu2(top, *reinterpret_cast<const uint16_t*>(&v) & 0x7fffu);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) top = max(top, magnitude_bits(op_get(v.e[i])));
  }
  return top;
}
template <class T>
__device__ __forceinline__ uint32_t row_top_bits(uint32_t top) {
  if constexpr (sizeof(T) == 4) return top;
  const unsigned short bits = static_cast<unsigned short>(max(top & 0xffffu, top >> 16));
  return __float_as_uint(op_get(*reinterpret_cast<const T*>(&bits)));
}

struct RowScale {
  float factor;  // 127 / top, or 0
  float top;
  float step;
};

template <class T>
__device__ __forceinline__ RowScale row_scale(uint32_t top_bits) {
  RowScale r;
  r.top = __uint_as_float(top_bits);
  const bool number = top_bits < 0x7f800000u, live = number && r.top >= kRowLeast;
  r.factor = live ? __fdiv_rn(127.0f, r.top) : 0.0f;
  if (sizeof(T) == 2) r.factor *= 1.0f + 0x1p-21f;
  r.step = live ? __fdiv_rn(r.top, 127.0f) : number ? 0.0f : __uint_as_float(0x7fc00000u);
  return r;
}

static __device__ __noinline__ float row_round_near_half(float x, float top) {
  const double q = floor(127.0 * fabs(static_cast<double>(x)) / top + 0.5);
  return kRowMagic + static_cast<float>(x < 0.0f ? -q : q);
}

// The integer in the low byte, for rows whose factor is not 0 (the others are zeros, whatever is in them).
template <class T>
__device__ __forceinline__ uint32_t row_integer(float x, const RowScale& r) {
  float v = fmaf(x, r.factor, kRowMagic);
  if (sizeof(T) == 4) {
    const float rest = fmaf(x, r.factor, -(v - kRowMagic));
    if (fabsf(rest) > 0.4999f) v = row_round_near_half(x, r.top);
  }
  return __float_as_uint(v);
}

__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

}  // namespace nb
