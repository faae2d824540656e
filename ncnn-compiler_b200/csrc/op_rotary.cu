// Rotary positions with several axes on device arrays (ncnn_b200_op_rotary_axes).
//
// A pair (u, v) of a head's components becomes (u cos t - v sin t, u sin t + v cos t) with t = position * frequency,
// the position being the token's on the pair's axis.
//
// Angles.  fp32 products lose a far position's angle (position 100 000: 0.008 rad).  A frequency is held as turns
// per position in 64-bit fixed point, F = frequency / 2 pi * 2^64; position * F modulo 2^64 is the fraction of a turn:
// the wrap of the integer product is the range reduction, exact for every 32-bit position, negative ones too.  F itself is off by
// its rounding and by those of the powers before it (up to 127 products of 64-bit mantissas): 2^-30 of a turn at a position of 2^31.
// The signed product over 2^63 is in half turns, which sincospif takes as fp32: off by 2^-26 of a turn.
//
// Bound: HBM, each element read and written once.  A thread turns the same pairs of several heads of a token, so
// that angles are computed once per `heads_per_thread` heads.
#include <cmath>

#include "op_common.cuh"

namespace nb {
namespace {

constexpr int kMaxPairs = 128;
constexpr int kMaxAxes = 4;

struct RotaryParams {
  const void* x;
  void* y;
  long long tokens, first_token, position_rows;  // up to 2^31
  int repeats;  // position_rows < the call's tokens
  int heads, head_dim, pairs, axes;
  long long x_token, x_head, y_token, y_head;  // strides in elements
  const int* positions;
  int tail_units;  // units of components behind the pairs that are copied (0 in place)
  int head_groups;
  uint8_t axis[kMaxPairs];
  unsigned long long turns[kMaxPairs];
};

// V elements to an access; a unit is V pairs (halves apart: two accesses), V / 2 pairs (neighbours: one access; V = 1: one
// pair, two accesses) or V elements of the tail.
template <class T, int V, bool NEIGHBOURS, int HEADS>
__global__ void __launch_bounds__(256) k_rotary_axes(const __grid_constant__ RotaryParams p) {
  constexpr int PAIRS = NEIGHBOURS ? (V > 1 ? V / 2 : 1) : V;
  using Vec = OpVec<T, V>;
  // (lanes that read different parameters are served one after the other: 125 us for a 32 760-token video that takes 73 this way)
  __shared__ unsigned long long turns[kMaxPairs];
  __shared__ uint8_t axis[kMaxPairs];
  for (int i = threadIdx.x; i < p.pairs; i += 256) {
    turns[i] = p.turns[i];
    axis[i] = p.axis[i];
  }
  __syncthreads();
  const uint32_t pair_units = p.pairs / PAIRS;
  const uint32_t units = pair_units + p.tail_units;
  const uint32_t threads = static_cast<uint32_t>(p.tokens) * p.head_groups * units;  // (the host keeps this below 2^31)
  for (uint32_t thread = blockIdx.x * 256u + threadIdx.x; thread < threads; thread += gridDim.x * 256u) {
    const uint32_t rest = thread / units, unit = thread - rest * units;
    const uint32_t token_at = rest / p.head_groups;
    const int group = static_cast<int>(rest - token_at * p.head_groups);
    const long long token = token_at;
    const T* x = static_cast<const T*>(p.x) + token * p.x_token;
    T* y = static_cast<T*>(p.y) + token * p.y_token;
    if (unit >= pair_units) {
      const int c = 2 * p.pairs + static_cast<int>(unit - pair_units) * V;
#pragma unroll
      for (int i = 0; i < HEADS; ++i) {
        const int h = group + i * p.head_groups;
        if (h < p.heads) *reinterpret_cast<Vec*>(y + h * p.y_head + c) = *reinterpret_cast<const Vec*>(x + h * p.x_head + c);
      }
      continue;
    }
    const int first = static_cast<int>(unit) * PAIRS;
    // the accesses of a unit: u's, and v's where they are not in the same one
    const int cu = NEIGHBOURS ? 2 * first : first;
    const int cv = NEIGHBOURS ? cu + 1 : first + p.pairs;
    constexpr bool TWO = !NEIGHBOURS || V == 1;
    Vec a[HEADS], b[TWO ? HEADS : 1];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int h = group + i * p.head_groups;
      if (h < p.heads) {
        a[i] = *reinterpret_cast<const Vec*>(x + h * p.x_head + cu);
        if constexpr (TWO) b[i] = *reinterpret_cast<const Vec*>(x + h * p.x_head + cv);
      }
    }
    float sine[PAIRS], cosine[PAIRS];
    const int* position = p.positions + (p.repeats ? static_cast<uint32_t>(p.first_token + token) % static_cast<uint32_t>(p.position_rows) : p.first_token + token) * p.axes;
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      const unsigned long long turn = static_cast<unsigned long long>(static_cast<long long>(__ldg(position + axis[first + j]))) * turns[first + j];
      sincospif(static_cast<float>(static_cast<long long>(turn)) * 0x1p-63f, &sine[j], &cosine[j]);
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      const int h = group + i * p.head_groups;
      if (h >= p.heads) break;
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        T& eu = TWO ? a[i].e[j] : a[i].e[(2 * j) % V];
        T& ev = TWO ? b[TWO ? i : 0].e[j % V] : a[i].e[(2 * j + 1) % V];
        const float u = op_get(eu), v = op_get(ev);
        eu = op_put<T>(u * cosine[j] - v * sine[j]);
        ev = op_put<T>(u * sine[j] + v * cosine[j]);
      }
      *reinterpret_cast<Vec*>(y + h * p.y_head + cu) = a[i];
      if constexpr (TWO) *reinterpret_cast<Vec*>(y + h * p.y_head + cv) = b[i];
    }
  }
}

template <class T, int V, bool NEIGHBOURS, int HEADS>
cudaError_t launch_heads(RotaryParams p, long long units, int sms, cudaStream_t st) {
  p.head_groups = (p.heads + HEADS - 1) / HEADS;
  const long long tokens = p.tokens, a_token = p.head_groups * units;
  const long long most = std::max<long long>(1, (1ll << 30) / a_token);  // tokens of a launch: thread numbers have 32 bits
  for (p.first_token = 0; p.first_token < tokens; p.first_token += most) {
    p.tokens = std::min(most, tokens - p.first_token);
    const long long blocks = (p.tokens * a_token + 255) / 256;
    const dim3 grid(static_cast<unsigned>(std::min<long long>(blocks, sms * 16ll)));
    if (const cudaError_t e = op_launch(k_rotary_axes<T, V, NEIGHBOURS, HEADS>, grid, 256, 0, st, 0, p); e != cudaSuccess) return e;
    p.x = static_cast<const T*>(p.x) + most * p.x_token;
    p.y = static_cast<T*>(p.y) + most * p.y_token;
  }
  return cudaSuccess;
}

template <class T, int V, bool NEIGHBOURS>
cudaError_t launch(RotaryParams& p, bool in_place, int sms, cudaStream_t st) {
  constexpr int PAIRS = NEIGHBOURS ? (V > 1 ? V / 2 : 1) : V;
  p.tail_units = in_place ? 0 : (p.head_dim - 2 * p.pairs) / V;
  const long long units = p.pairs / PAIRS + p.tail_units;
  // Several heads to a thread where that leaves enough threads to fill the device: four accesses under way.  32760 tokens of 24
  // heads of 128, one, two, four, eight heads: neighbours 153, 95, 74, 82 us, halves apart (two accesses a head) 129, 91, 108, 165.
  constexpr int HEADS = NEIGHBOURS ? 4 : 2;
  if (p.heads >= HEADS && p.tokens * ((p.heads + HEADS - 1) / HEADS) * units >= sms * 2048ll / 4 * HEADS) return launch_heads<T, V, NEIGHBOURS, HEADS>(p, units, sms, st);
  return launch_heads<T, V, NEIGHBOURS, 1>(p, units, sms, st);
}

}  // namespace
}  // namespace nb

extern "C" int ncnn_b200_op_rotary_axes(const void* x, void* y, int32_t type, int64_t tokens, int32_t heads, int32_t head_dim,
                                        const int64_t* strides, const int32_t* positions, int64_t position_rows, int32_t axes,
                                        const int32_t* sections, double base, int32_t interleaved, int32_t shared_spectrum, void* stream) {
  using namespace nb;
  static const char* kOp = "op_rotary_axes";
  return op_guarded(kOp, [&]() -> int {
    if (x == nullptr || y == nullptr || positions == nullptr || sections == nullptr)
      return op_fail(NCNN_B200_STATUS_NULL_POINTER, "op_rotary_axes: NULL argument");
    if (!op_type_ok(type)) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_rotary_axes: unknown element type");
    if (!op_starts(x, op_elem_bytes(type)) || !op_starts(y, op_elem_bytes(type)) || !op_starts(positions, 4))
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_rotary_axes: an array does not start at a multiple of its elements' size");
    if (tokens < 0 || tokens > (1ll << 31) || heads <= 0 || heads > 65536 || head_dim <= 0 || head_dim > 65536 || axes <= 0 || axes > kMaxAxes)
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_rotary_axes: tokens must be 0 to 2^31, heads and head_dim 1 to 65536, axes 1 to 4");
    if (position_rows < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_rotary_axes: position_rows must not be negative");
    if (!(base >= 1.0) || !(base <= 1e30)) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_rotary_axes: base must be 1 to 1e30");
    RotaryParams p{};
    int64_t pairs = 0;
    for (int a = 0; a < axes; ++a) {
      if (sections[a] < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_rotary_axes: a section is negative");
      pairs += sections[a];
    }
    if (pairs <= 0 || pairs > kMaxPairs || 2 * pairs > head_dim)
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_rotary_axes: the sections must hold 1 to 128 pairs, and head_dim twice as many components");
    if (position_rows == 0 || position_rows > tokens) position_rows = tokens;
    if (tokens == 0) return NCNN_B200_STATUS_SUCCESS;
    p.x = x;
    p.y = y;
    p.tokens = tokens;
    p.position_rows = position_rows;
    p.repeats = position_rows < tokens;
    p.heads = heads;
    p.head_dim = head_dim;
    p.pairs = static_cast<int>(pairs);
    p.axes = axes;
    p.x_token = p.y_token = static_cast<long long>(heads) * head_dim;
    p.x_head = p.y_head = head_dim;
    if (strides != nullptr) {
      for (int i = 0; i < 4; ++i)
        if (strides[i] > (1ll << 50) / std::max<int64_t>(tokens, heads)) return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_rotary_axes: a stride is too large");
      p.x_token = strides[0];
      p.x_head = strides[1];
      p.y_token = strides[2];
      p.y_head = strides[3];
      // heads (and tokens) of the result that overlap would be written twice; an axis of one entry is never stepped over
      bool apart = p.x_token >= 0 && p.x_head >= 0 && p.y_token >= 0 && p.y_head >= 0;
      if (apart) {
        const bool heads_inside = (heads == 1 || p.y_head >= head_dim) && (tokens == 1 || p.y_token >= (heads - 1) * p.y_head + head_dim);
        const bool tokens_inside = (tokens == 1 || p.y_token >= head_dim) && (heads == 1 || p.y_head >= (tokens - 1) * p.y_token + head_dim);
        apart = heads_inside || tokens_inside;
      }
      if (!apart) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_rotary_axes: negative strides, or results that overlap");
    }
    const bool in_place = x == y;
    if (in_place && ((tokens > 1 && p.x_token != p.y_token) || (heads > 1 && p.x_head != p.y_head)))
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_rotary_axes: in place, both sides need the same strides");
    p.positions = positions;
    // the frequencies of an axis are powers of one ratio; 64-bit mantissas keep the 53 bits that double would round to
    long double ratio = 1.0L, rate = 1.0L;
    for (int a = 0, at = 0, period = 0; a < axes; ++a) {
      const int count = sections[a], to = shared_spectrum ? static_cast<int>(pairs) : count;
      if (count == 0) continue;
      if (to != period) ratio = std::pow(static_cast<long double>(base), -1.0L / static_cast<long double>(to));
      period = to;
      if (!shared_spectrum) rate = 1.0L;
      for (int j = 0; j < count; ++j, ++at, rate *= ratio) {
        p.axis[at] = static_cast<uint8_t>(a);
        p.turns[at] = static_cast<unsigned long long>(rate * (0x1p64L / 6.283185307179586476925286766559L) + 0.5L);
      }
    }
    if (tokens > (1ll << 38) / (static_cast<int64_t>(heads) * head_dim))
      return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_rotary_axes: more than 2^38 components");
    std::string why;
    const int device = op_common_device(kOp, {x, y, positions}, &why);
    if (device < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, why);
    DeviceGuard guard(device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int sms = op_sm_count(device);
    const int wide = 16 / op_elem_bytes(type);  // elements of a 16-byte access
    auto all_multiples = [&](int v) {
      const uintptr_t bytes = static_cast<uintptr_t>(v) * op_elem_bytes(type);
      const int pairs_a_unit = interleaved ? v / 2 : v;
      return reinterpret_cast<uintptr_t>(x) % bytes == 0 && reinterpret_cast<uintptr_t>(y) % bytes == 0 && p.x_token % v == 0 && p.x_head % v == 0 &&
             p.y_token % v == 0 && p.y_head % v == 0 && p.pairs % pairs_a_unit == 0 && (interleaved ? 2 * p.pairs : p.pairs) % v == 0 && head_dim % v == 0;
    };
    const int v = all_multiples(wide) ? wide : all_multiples(2) ? 2 : 1;  // elements of an access
    return op_by_type(type, [&](auto t) {
      using T = decltype(t);
      constexpr int V = 16 / sizeof(T);
      cudaError_t e;
      if (interleaved) e = v == V ? launch<T, V, true>(p, in_place, sms, st) : v == 2 ? launch<T, 2, true>(p, in_place, sms, st) : launch<T, 1, true>(p, in_place, sms, st);
      else e = v == V ? launch<T, V, false>(p, in_place, sms, st) : v == 2 ? launch<T, 2, false>(p, in_place, sms, st) : launch<T, 1, false>(p, in_place, sms, st);
      return op_launched(kOp, e);
    });
  });
}
