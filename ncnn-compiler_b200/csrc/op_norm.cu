// Group norm with an activation over channel-last feature maps on device arrays (ncnn_b200_op_group_norm):
//   y[i][p][c] = act((x[i][p][c] - m) / sqrt(v + eps) * gamma[c] + beta[c])
// with the mean m and the (biased) variance v over the pixels and the channels of c's group in image i.
#include <cmath>

#include "op_common.cuh"

namespace nb {
namespace {

struct NormParams {
  const void* x;
  void* y;
  long long n, pixels, x_pitch, y_pitch;
  int channels, groups, act;
  const float *gamma, *beta;
  float eps;
};

__device__ __forceinline__ float norm_act(float y, int act) {
  if (act == NCNN_B200_ACT_RELU) return y < 0.0f ? 0.0f : y;  // (a NaN stays one)
  if (act == NCNN_B200_ACT_SWISH) return __fdividef(y, 1.0f + __expf(-y));
  if (act == NCNN_B200_ACT_GELU) return 0.5f * y * erfcf(y * -0.70710678118654752f);
  return y;
}

__device__ float block_sum(float v) {
  __shared__ float parts[32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
  __syncthreads();
  v = threadIdx.x < (blockDim.x >> 5) ? parts[threadIdx.x] : 0.0f;
  if (threadIdx.x < 32) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (threadIdx.x == 0) parts[0] = v;
  }
  __syncthreads();
  return parts[0];
}

// One CTA to an image's group: mean, variance about it, result; x is read three times.
template <class T>
__global__ void __launch_bounds__(512) k_group_norm(const __grid_constant__ NormParams p) {
  const int size = p.channels / p.groups;
  const long long image = blockIdx.x / p.groups;
  const int c0 = static_cast<int>(blockIdx.x % p.groups) * size;
  const T* x = static_cast<const T*>(p.x) + image * p.pixels * p.x_pitch + c0;
  T* y = static_cast<T*>(p.y) + image * p.pixels * p.y_pitch + c0;
  const long long count = p.pixels * size;
  float sum = 0.0f;
  for (long long i = threadIdx.x; i < count; i += 512) sum += op_get(x[i / size * p.x_pitch + i % size]);
  const float mean = block_sum(sum) / static_cast<float>(count);
  sum = 0.0f;
  for (long long i = threadIdx.x; i < count; i += 512) {
    const float d = op_get(x[i / size * p.x_pitch + i % size]) - mean;
    sum = fmaf(d, d, sum);
  }
  const float scale = 1.0f / sqrtf(block_sum(sum) / static_cast<float>(count) + p.eps);
  for (long long i = threadIdx.x; i < count; i += 512) {
    const int c = static_cast<int>(i % size);
    float v = (op_get(x[i / size * p.x_pitch + c]) - mean) * scale;
    v = fmaf(v, p.gamma ? p.gamma[c0 + c] : 1.0f, p.beta ? p.beta[c0 + c] : 0.0f);
    y[i / size * p.y_pitch + c] = op_put<T>(norm_act(v, p.act));
  }
}

}  // namespace
}  // namespace nb

extern "C" int ncnn_b200_op_group_norm(const void* x, void* y, int32_t type, int64_t n, int64_t pixels, int32_t channels, int32_t groups,
                                       int64_t x_pitch, int64_t y_pitch, const float* gamma, const float* beta, float eps, int32_t activation,
                                       void* stream) {
  using namespace nb;
  static const char* kOp = "op_group_norm";
  return op_guarded(kOp, [&]() -> int {
    if (x == nullptr || y == nullptr) return op_fail(NCNN_B200_STATUS_NULL_POINTER, "op_group_norm: NULL argument");
    if (!op_type_ok(type)) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_group_norm: unknown element type");
    if (n < 0 || pixels < 0 || channels <= 0 || groups <= 0 || channels % groups != 0)
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_group_norm: n and pixels must not be negative, channels a positive multiple of groups");
    if (!(eps >= 0.0f) || std::isinf(eps)) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_group_norm: eps must be finite and not negative");
    if (activation != NCNN_B200_ACT_NONE && activation != NCNN_B200_ACT_RELU && activation != NCNN_B200_ACT_SWISH && activation != NCNN_B200_ACT_GELU)
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_group_norm: unknown activation");
    if (x_pitch == 0) x_pitch = channels;
    if (y_pitch == 0) y_pitch = channels;
    if (x_pitch < channels || y_pitch < channels)
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_group_norm: a pitch is smaller than a pixel's channels");
    if (x == y && x_pitch != y_pitch) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_group_norm: in place, both pitches have to be the same");
    if (n == 0 || pixels == 0) return NCNN_B200_STATUS_SUCCESS;
    if (pixels > (1ll << 40) / std::max(x_pitch, y_pitch) || n > (1ll << 40) / (pixels * std::max(x_pitch, y_pitch)) || n * groups > 0x7fffffffll)
      return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_group_norm: more than 2^40 elements, or 2^31 groups");
    std::string why;
    const int device = op_common_device(kOp, {x, y, gamma, beta}, &why);
    if (device < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, why);
    DeviceGuard guard(device);
    NormParams p{x, y, n, pixels, x_pitch, y_pitch, channels, groups, activation, gamma, beta, eps};
    op_by_type(type, [&](auto t) {
      k_group_norm<decltype(t)><<<static_cast<unsigned>(n * groups), 512, 0, static_cast<cudaStream_t>(stream)>>>(p);
      return 0;
    });
    return op_launched(kOp);
  });
}
