// Attention of one sequence's tokens to another's (an encoder's states) on device arrays (ncnn_b200_op_cross_attention):
//   o[b][i][h] = sum_j softmax_j(scale * q[b][i][h] . k[b][j][h']) v[b][j][h']
// over the keys j < kv_lens[b] with key_mask[b][j] != 0; h' = h / (heads / kv_heads).  A sequence without such a key has
// zeros for its result.  What lies at keys that take no part is never used, NaN or infinity as it may be.
#include <cmath>

#include "op_attention.h"

namespace nb {
namespace {

// One warp to a query's head, a key at a time: components over the lanes, running maximum and sum.
template <class T, int PER_LANE>
__global__ void __launch_bounds__(256) k_attend_row(const __grid_constant__ AttendParams p) {
  const long long at = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int h = static_cast<int>(at % p.heads);
  const long long rest = at / p.heads;
  const int i = static_cast<int>(rest % p.lq);
  const int b = static_cast<int>(rest / p.lq);
  if (b >= p.batch) return;
  const int kv = h / (p.heads / p.kv_heads);
  const T* q = static_cast<const T*>(p.q) + b * p.q_batch + i * p.q_row + h * p.q_head;
  const T* k = static_cast<const T*>(p.k) + b * p.k_batch + kv * p.k_head;
  const T* v = static_cast<const T*>(p.v) + b * p.v_batch + kv * p.v_head;
  T* o = static_cast<T*>(p.o) + b * p.o_batch + i * p.o_row + h * p.o_head;
  const int keys = p.lens == nullptr ? p.lk : min(max(p.lens[b], 0), p.lk);
  const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + static_cast<long long>(b) * p.lk;
  float qv[PER_LANE], sum[PER_LANE];
#pragma unroll
  for (int c = 0; c < PER_LANE; ++c) {
    qv[c] = lane + 32 * c < p.d ? op_get(q[lane + 32 * c]) * p.scale : 0.0f;
    sum[c] = 0.0f;
  }
  float top = -INFINITY, total = 0.0f;
  for (int j = 0; j < keys; ++j) {
    if (mask != nullptr && mask[j] == 0) continue;
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < PER_LANE; ++c)
      if (lane + 32 * c < p.d) s = fmaf(qv[c], op_get(k[j * p.k_row + lane + 32 * c]), s);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(~0u, s, w);
    const float next = fmaxf(top, s);
    const float base = next == -INFINITY ? 0.0f : next;
    const float keep = expf(top - base), e = expf(s - base);
    total = fmaf(total, keep, e);
#pragma unroll
    for (int c = 0; c < PER_LANE; ++c)
      if (lane + 32 * c < p.d) sum[c] = fmaf(e, op_get(v[j * p.v_row + lane + 32 * c]), sum[c] * keep);
    top = next;
  }
  const float scale = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int c = 0; c < PER_LANE; ++c)
    if (lane + 32 * c < p.d) o[lane + 32 * c] = op_put<T>(total == 0.0f ? 0.0f : sum[c] * scale);
}

}  // namespace
}  // namespace nb

extern "C" int ncnn_b200_op_cross_attention(const void* q, const void* k, const void* v, void* o, int32_t type, int64_t batch, int64_t lq,
                                            int64_t lk, int32_t heads, int32_t kv_heads, int32_t head_dim, const int64_t* strides,
                                            const int32_t* kv_lens, const uint8_t* key_mask, float scale, void* stream) {
  using namespace nb;
  static const char* kOp = "op_cross_attention";
  return op_guarded(kOp, [&]() -> int {
    if (!op_type_ok(type)) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_cross_attention: unknown element type");
    if (batch < 0 || lq < 0 || lk < 0 || batch > 65535 || lq > (1 << 30) || lk > (1 << 30) || heads <= 0 || heads > 65535 || kv_heads <= 0 ||
        heads % kv_heads != 0 || head_dim <= 0 || head_dim > 256)
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE,
                     "op_cross_attention: batch 0 to 65535, lengths 0 to 2^30, heads a multiple of kv_heads up to 65535, head_dim 1 to 256");
    if (!(scale >= 0.0f) || std::isinf(scale)) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_cross_attention: scale must be finite and not negative");
    if (batch == 0 || lq == 0) return NCNN_B200_STATUS_SUCCESS;
    if (q == nullptr || o == nullptr || (lk > 0 && (k == nullptr || v == nullptr)))
      return op_fail(NCNN_B200_STATUS_NULL_POINTER, "op_cross_attention: NULL argument");
    if (o == q || o == k || o == v) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_cross_attention: the result must not lie over an input");
    AttendParams p{};
    p.q = q;
    p.k = k;
    p.v = v;
    p.o = o;
    p.batch = static_cast<int>(batch);
    p.lq = static_cast<int>(lq);
    p.lk = static_cast<int>(lk);
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.d = head_dim;
    p.lens = kv_lens;
    p.mask = key_mask;
    p.scale = scale == 0.0f ? 1.0f / std::sqrt(static_cast<float>(head_dim)) : scale;
    if (strides != nullptr) {
      for (int i = 0; i < 12; ++i)
        if (strides[i] < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_cross_attention: a stride is negative");
      std::tie(p.q_batch, p.q_row, p.q_head) = std::make_tuple(strides[0], strides[1], strides[2]);
      std::tie(p.k_batch, p.k_row, p.k_head) = std::make_tuple(strides[3], strides[4], strides[5]);
      std::tie(p.v_batch, p.v_row, p.v_head) = std::make_tuple(strides[6], strides[7], strides[8]);
      std::tie(p.o_batch, p.o_row, p.o_head) = std::make_tuple(strides[9], strides[10], strides[11]);
      // the result's axes from the innermost out: each has to step over what lies inside it
      std::array<std::pair<int64_t, int64_t>, 3> axes = {{{p.o_batch, batch}, {p.o_row, lq}, {p.o_head, heads}}};
      std::sort(axes.begin(), axes.end());
      int64_t extent = head_dim;
      for (const auto& a : axes) {
        if (a.second == 1) continue;
        if (a.first < extent) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_cross_attention: the result's rows overlap");
        if (a.first > (1ll << 50) / a.second) return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_cross_attention: a stride is too large");
        extent = a.first * (a.second - 1) + extent;
      }
      for (int i = 0; i < 9; ++i)
        if (strides[i] > (1ll << 50) / std::max<int64_t>({batch, lq, lk, heads}))
          return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_cross_attention: a stride is too large");
    } else {
      p.q_head = p.o_head = p.k_head = p.v_head = head_dim;
      p.q_row = p.o_row = static_cast<long long>(heads) * head_dim;
      p.k_row = p.v_row = static_cast<long long>(kv_heads) * head_dim;
      p.q_batch = p.o_batch = p.q_row * lq;
      p.k_batch = p.v_batch = p.k_row * lk;
    }
    std::string why;
    const int device = op_common_device(kOp, {q, o, lk > 0 ? k : nullptr, lk > 0 ? v : nullptr, kv_lens, key_mask}, &why);
    if (device < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, why);
    DeviceGuard guard(device);
    const long long rows = batch * lq * heads;
    if (rows > (1ll << 33)) return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_cross_attention: more than 2^33 rows");
    op_by_type(type, [&](auto t) {
      using T = decltype(t);
      const unsigned grid = static_cast<unsigned>((rows + 7) / 8);
      cudaStream_t st = static_cast<cudaStream_t>(stream);
      if (p.d <= 64) k_attend_row<T, 2><<<grid, 256, 0, st>>>(p);
      else if (p.d <= 128) k_attend_row<T, 4><<<grid, 256, 0, st>>>(p);
      else k_attend_row<T, 8><<<grid, 256, 0, st>>>(p);
      return 0;
    });
    return op_launched(kOp);
  });
}
