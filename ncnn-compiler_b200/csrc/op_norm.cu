// Group norm with an activation over channel-last feature maps on device arrays (ncnn_b200_op_group_norm):
//   y[i][p][c] = act((x[i][p][c] - m) / sqrt(v + eps) * gamma[c] + beta[c])
// with the mean m and the (biased) variance v over the pixels and the channels of c's group in image i.
#include <cmath>

#include <cooperative_groups.h>

#include "op_common.cuh"
#include "op_norm.h"

namespace nb {
namespace {

struct NormParams {
  const void* x;
  void* y;
  long long n, pixels, x_pitch, y_pitch;
  int channels, groups;
  const float *gamma, *beta;
  float eps, floor;
  ActRef in, out;  // fp32: x and y, or a graph's tensors
  long long first_image;
  int by_image;  // cut images alike whatever their number
};

// No activation and ReLU are one kernel: the line above a floor of minus infinity or 0.
// Swish of fp32 is good to 9 F of the result, F = 2^-24 (measured: 5; a graph's other Swish, expf and a rounded division: 4).  The
// plain approximations lose 2 F more for every unit of y, 57 F at -45; they serve results of 16 bits, where that is below a
// hundredth of fp16's half step.  8 maps of 64 x 64 x 320: 25 us, 24 with the approximations, 33 with expf and the division.
template <class T, int ACT>
__device__ __forceinline__ float norm_act(float y, float floor) {
  if (ACT == NCNN_B200_ACT_NONE) return y < floor ? floor : y;  // (a NaN stays one)
  if (ACT == NCNN_B200_ACT_SWISH && sizeof(T) == 4) {
    // e^-y = 2^t 2^rest with t + rest = -y log2(e) to twice fp32's bits; the reciprocal and a Newton step.  (No more than 100, where
    // e is 0 to 1 + e: infinity has no rest.  Beyond fp32's range 1 / (1 + e) is 0.)
    const float x = fminf(y, 100.0f), t = x * -1.44269504f, rest = fmaf(x, -1.92596299e-8f, fmaf(x, -1.44269504f, -t));
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    const float d = 1.0f + fminf(fmaf(e * 0.693147181f, rest, e), 3.4e38f);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return y * fmaf(r, fmaf(-d, r, 1.0f), r);
  }
  if (ACT == NCNN_B200_ACT_SWISH) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y * -1.44269504088896340736f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));  // (0 where e is infinite)
    return y * r;
  }
  if (ACT == NCNN_B200_ACT_GELU) return 0.5f * y * erfcf(y * -0.70710678118654752f);
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

// Moves the shift of n values' sums (s1 of their differences from it, s2 of the squares) to their mean.
__device__ __forceinline__ void recentre(float n, float inverse, float& shift, float& s1, float& s2) {
  const float to = fmaf(s1, inverse, shift), off = to - shift;
  s2 = fmaxf(fmaf(-off, fmaf(-n, off, 2.0f * s1), s2), 0.0f);
  s1 = fmaf(-n, off, s1);
  shift = to;
}

// Several groups of an image, `channels` neighbouring channels, belong to a cluster of CTAs, and each CTA has a range of the
// pixels.  A thread owns V channels (a 16-byte access where addresses allow it) and every ROWS-th pixel of the range, so that
// scale and offset of the second pass are registers.
//
// Statistics.  A thread sums its values and their squares about its own first value of the channel, in fp32, and turns the
// sums into a mean and a sum of squared deviations from it; from there on those are combined (n, mean, deviations), over the
// CTA's threads and then over the cluster's CTAs, with the deviations taken about the combined mean.  Sums about zero lose the
// variance of maps that lie far from it (a mean of 1000 deviations: all of it), and a common shift loses it to one outlier; one
// that is a thread's first value would stand in all of its differences (4096 of them, the first of 100 000 deviations: the
// variance off by a seventh), so the shift moves to the mean after 64, 256, 1024, ... values.
//
// Bound: HBM, x once and y once, where x stays on the SM or in L2 between the passes.  Every thread has a ring of 16 (or 12) of its own
// pixels in shared memory, filled by cp.async four at a time (no registers for what is under way: 48 KB a CTA, three CTAs to an
// SM).  The second pass goes backwards: it begins with what the first one left in the ring and goes on with what L2 saw last.
// Device times of captured calls: 8 maps of 64 x 64 x 320, bf16 19.5 us; 2 of 512 x 512 x 128, fp32 162 us, where two thirds of x have
// to come from HBM again (5 TB/s in each pass; CTAs of 768 threads, stores that leave L2 first, and whole pixels to a CTA were no
// faster).
constexpr int kNormThreads = 256;
constexpr int kNormMostGroups = 128;
constexpr int kNormGroup = 4;   // pixels that are asked for together
constexpr int kNormFirstMove = 64;  // pixels of a thread before its shift moves

template <int V>
constexpr int kNormSlots = V == 8 ? 12 : 16;  // pixels of a thread's ring (three CTAs' rings and statistics fit an SM)

struct NormShape {
  int channels;       // of a cluster
  int size, groups;   // channels of a group, groups of a cluster
  int each;           // pixels of a CTA (the last ones may have fewer)
  int columns, rows;  // threads: columns of V channels, rows of pixels
  int slots;          // of a ring: kNormSlots, or fewer where no thread has as many pixels
};

struct Moments {
  float mean, m2;
};

__device__ __forceinline__ void graph_load(const ActRef& a, long long i, OpVec<float, 4>& v) { *reinterpret_cast<float4*>(&v) = act_load4(a, i); }
__device__ __forceinline__ void graph_load(const ActRef& a, long long i, OpVec<float, 1>& v) { v.e[0] = act_load(a, i); }
__device__ __forceinline__ void graph_store(const ActRef& a, long long i, const OpVec<float, 4>& v) { act_store4(a, i, *reinterpret_cast<const float4*>(&v)); }
__device__ __forceinline__ void graph_store(const ActRef& a, long long i, const OpVec<float, 1>& v) { act_store(a, i, v.e[0]); }

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else if constexpr (BYTES >= 4) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}

// LONG: ranges of more than 64 pixels to a thread.
// fp32 tensors are those of a loaded graph, too, in whatever format their other readers and writers want.
template <class T, int V, int ACT, bool LONG>
__global__ void __launch_bounds__(kNormThreads, 3) k_group_norm(const __grid_constant__ NormParams p, const __grid_constant__ NormShape s) {
  namespace cg = cooperative_groups;
  using Vec = OpVec<T, V>;
  constexpr bool GRAPH = sizeof(T) == 4;
  extern __shared__ __align__(16) uint8_t norm_smem[];
  // the CTA's, and the cluster's mean and 1 / sqrt(variance + eps), of each group
  __shared__ Moments group_parts[kNormMostGroups];
  __shared__ float2 result[kNormMostGroups];
  Vec* ring = reinterpret_cast<Vec*>(norm_smem) + threadIdx.x;  // [slot][thread]
  const int size = s.size, groups = s.groups;
  const int ranks = gridDim.x, rank = blockIdx.x;
  const long long image = blockIdx.z;
  const int c0 = blockIdx.y * s.channels;
  // this CTA's pixels, and this thread's: `longer` rows of threads have a pixel more
  const int pixels = static_cast<int>(p.pixels), each = s.each;
  const int begin = static_cast<int>(min(static_cast<long long>(each) * rank, p.pixels)), here = min(each, pixels - begin);
  const int row = static_cast<int>(threadIdx.x / static_cast<unsigned>(s.columns)), column = static_cast<int>(threadIdx.x) - row * s.columns;
  const int whole_rows = here / s.rows, longer = here - whole_rows * s.rows;
  const int count = row < s.rows ? whole_rows + (row < longer ? 1 : 0) : 0;
  const T* x = static_cast<const T*>(p.x) + (image * p.pixels + begin + row) * p.x_pitch + c0 + column * V;
  T* y = static_cast<T*>(p.y) + (image * p.pixels + begin + row) * p.y_pitch + c0 + column * V;
  const long long x_step = s.rows * p.x_pitch, y_step = s.rows * p.y_pitch;
  // (fp32) elements from the tensors' starts
  const long long pixel0 = GRAPH ? (p.first_image + image) * p.pixels + begin + row : 0;
  const long long x_element = GRAPH ? pixel0 * p.x_pitch + c0 + column * V : 0, y_element = GRAPH ? pixel0 * p.y_pitch + c0 + column * V : 0;
  const int steps = (count + kNormGroup - 1) / kNormGroup;
  // four pixels of this thread on their way to their slots (2-byte pieces, which cp.async does not take: through registers)
  auto request = [&](int step) {
    if (step >= 0 && step < steps) {
      const T* from = x + step * kNormGroup * x_step;
      Vec* to = ring + step * kNormGroup % kNormSlots<V> * kNormThreads;
      if (GRAPH && p.in.fmt != FMT_F32) {
        if constexpr (GRAPH) {
#pragma unroll
          for (int u = 0; u < kNormGroup; ++u)
            if (step * kNormGroup + u < count) graph_load(p.in, x_element + (step * kNormGroup + u) * x_step, to[u * kNormThreads]);
        }
      } else if constexpr (sizeof(Vec) >= 4) {
#pragma unroll
        for (int u = 0; u < kNormGroup; ++u)
          if (step * kNormGroup + u < count) copy_async<sizeof(Vec)>(static_cast<uint32_t>(__cvta_generic_to_shared(to + u * kNormThreads)), from + u * x_step);
      } else {
        Vec at[kNormGroup];
#pragma unroll
        for (int u = 0; u < kNormGroup; ++u)
          if (step * kNormGroup + u < count) at[u] = *reinterpret_cast<const Vec*>(from + u * x_step);
#pragma unroll
        for (int u = 0; u < kNormGroup; ++u)
          if (step * kNormGroup + u < count) to[u * kNormThreads] = at[u];
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  constexpr int kAhead = kNormSlots<V> / kNormGroup - 1;

  Moments part[V];
  {
    float shift[V], s1[V], s2[V];
#pragma unroll
    for (int v = 0; v < V; ++v) shift[v] = s1[v] = s2[v] = 0.0f;
#pragma unroll
    for (int g = 0; g < kAhead; ++g) request(g);
    auto add = [&](int g) {
      request(g + kAhead);
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
      const Vec* at = ring + g * kNormGroup % kNormSlots<V> * kNormThreads;
      if (g == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) shift[v] = op_get(at->e[v]);
      }
#pragma unroll
      for (int u = 0; u < kNormGroup; ++u)
        if (g * kNormGroup + u < count) {
          const Vec in = at[u * kNormThreads];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float d = op_get(in.e[v]) - shift[v];
            s1[v] += d;
            s2[v] = fmaf(d, d, s2[v]);
          }
        }
    };
    // (ranges that need no move of the shift have a kernel without one: code that they only pass cost 8 maps of 64 x 64 x 320 0.6 of 20 us)
    int g = 0;
    for (int until = LONG ? min(kNormFirstMove / kNormGroup, steps) : steps; g < steps;) {
      for (; g < until; ++g) add(g);
      if (LONG && g < steps) {
        const float n = static_cast<float>(g * kNormGroup), inverse = 1.0f / n;
#pragma unroll
        for (int v = 0; v < V; ++v) recentre(n, inverse, shift[v], s1[v], s2[v]);
        until = min(4 * until, steps);
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    const float inverse = count > 0 ? 1.0f / static_cast<float>(count) : 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float off = s1[v] * inverse;
      part[v] = {shift[v] + off, fmaxf(s2[v] - s1[v] * off, 0.0f)};
    }
  }
  // [row][v][column] in shared memory behind the rings
  Moments* parts = reinterpret_cast<Moments*>(norm_smem + static_cast<size_t>(s.slots) * kNormThreads * sizeof(Vec));
  if (row < s.rows) {
#pragma unroll
    for (int v = 0; v < V; ++v) parts[row * s.channels + v * s.columns + column] = part[v];
  }
  float scale[V], offset[V];  // asked for here, needed behind the statistics
  int to_group = column * V / size, in_group = column * V - to_group * size;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = c0 + column * V + v;
    const bool mine = row < s.rows;
    scale[v] = p.gamma != nullptr && mine ? __ldg(p.gamma + c) : 1.0f;
    offset[v] = p.beta != nullptr && mine ? __ldg(p.beta + c) : 0.0f;
  }
  __syncthreads();
  // A warp to a group: lanes over its channels and as many rows as fit; the mean first, the deviations about it second.
  const int lane = threadIdx.x & 31;
  const int lane_rows = size < 32 ? 32 / size : 1, lane_row = size < 32 ? lane / size : 0, lane_channel = size < 32 ? lane - lane_row * size : lane;
  const int rows_in_use = min(s.rows, here);
  for (int g = threadIdx.x >> 5; g < groups; g += kNormThreads / 32) {
    auto over = [&](auto&& f) {
      if (lane_row < lane_rows)
        for (int i = lane_channel; i < size; i += 32) {
          const int c = g * size + i;
          const Moments* of = parts + c % V * s.columns + c / V;
#pragma unroll 4
          for (int r = lane_row; r < rows_in_use; r += lane_rows) f(of[r * s.channels], static_cast<float>(whole_rows + (r < longer ? 1 : 0)));
        }
    };
    const float about = parts[g * size % V * s.columns + g * size / V].mean;  // (a group of one value has that for its mean, exactly)
    float sum = 0.0f, m2 = 0.0f;
    over([&](const Moments& m, float n) { sum = fmaf(n, m.mean - about, sum); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    const float mean = here > 0 ? about + sum / (static_cast<float>(here) * size) : 0.0f;
    over([&](const Moments& m, float n) { m2 += fmaf(n * (m.mean - mean), m.mean - mean, m.m2); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m2 += __shfl_xor_sync(~0u, m2, o);
    if (lane == 0) group_parts[g] = {mean, m2};
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (ranks > 1) cluster.sync();
  else __syncthreads();
  // the cluster's, the same way: lanes over its CTAs, 16 to a group
  const float inverse_total = 1.0f / (static_cast<float>(pixels) * size);
  for (int g0 = threadIdx.x >> 5; g0 * 2 < groups; g0 += kNormThreads / 32) {
    const int g = g0 * 2 + (lane >> 4), r = lane & 15;
    Moments m = {0.0f, 0.0f};
    float n = 0.0f;
    if (g < groups && r < ranks) {
      m = ranks > 1 ? *cluster.map_shared_rank(&group_parts[g], r) : group_parts[g];
      n = static_cast<float>(min(static_cast<long long>(each), max(p.pixels - static_cast<long long>(each) * r, 0ll))) * size;
    }
    const float about = __shfl_sync(~0u, m.mean, lane & 16);
    float sum = n > 0.0f ? n * (m.mean - about) : 0.0f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    const float mean = fmaf(sum, inverse_total, about);
    float m2 = n > 0.0f ? fmaf(n * (m.mean - mean), m.mean - mean, m.m2) : 0.0f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m2 += __shfl_xor_sync(~0u, m2, o);
    if (g < groups && r == 0) result[g] = make_float2(mean, 1.0f / sqrtf(m2 * inverse_total + p.eps));
  }
  __syncthreads();
  // no CTA's shared memory goes while another reads it: said here, waited for at the end
  if (ranks > 1) cluster.barrier_arrive();
  float mean[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float2 r = row < s.rows ? result[to_group] : make_float2(0.0f, 0.0f);
    mean[v] = r.x;
    scale[v] *= r.y;
    if (++in_group == size) {
      in_group = 0;
      ++to_group;
    }
  }
  for (int g = steps - 1; g >= 0; --g) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
    Vec at[kNormGroup];
    const Vec* from = ring + g * kNormGroup % kNormSlots<V> * kNormThreads;
#pragma unroll
    for (int u = 0; u < kNormGroup; ++u)
      if (g * kNormGroup + u < count) at[u] = from[u * kNormThreads];
    request(g - kAhead - 1);
    T* to = y + g * kNormGroup * y_step;
#pragma unroll
    for (int u = 0; u < kNormGroup; ++u)
      if (g * kNormGroup + u < count) {
        // (x - mean is exact where x is close to the mean)
#pragma unroll
        for (int v = 0; v < V; ++v) at[u].e[v] = op_put<T>(norm_act<T, ACT>(fmaf(op_get(at[u].e[v]) - mean[v], scale[v], offset[v]), p.floor));
        if constexpr (GRAPH) graph_store(p.out, y_element + (g * kNormGroup + u) * y_step, at[u]);
        else *reinterpret_cast<Vec*>(to + u * y_step) = at[u];
      }
  }
  if (ranks > 1) cluster.barrier_wait();
}

// Groups of more channels than a CTA has threads for: one CTA to a group, which reads x twice, four elements of a thread at a time.
//
// Statistics.  A thread may have tens of thousands of values: a sum about zero drifts by deviations there (a map of 128 x 128 x 1028
// with a mean of 1003 deviations: by 0.18).  So they are summed as in k_group_norm, about the thread's first value, and the shift
// follows the mean after 4, 8, 16, ... values: a first value far from the others would otherwise stand in every difference.
template <class T, int ACT>
__global__ void __launch_bounds__(kNormThreads) k_group_norm_wide(const __grid_constant__ NormParams p) {
  constexpr int kTogether = 4;
  const int size = p.channels / p.groups;
  const long long image = blockIdx.x / p.groups;
  const int c0 = static_cast<int>(blockIdx.x % p.groups) * size;
  const T* x = static_cast<const T*>(p.x) + image * p.pixels * p.x_pitch + c0;
  T* y = static_cast<T*>(p.y) + image * p.pixels * p.y_pitch + c0;
  // this thread's elements, every 256th of the group's: f gets pixels (from p.pixels on: none) and channels
  auto over = [&](auto&& f) {
    long long pixel = static_cast<int>(threadIdx.x) / size;
    int c = static_cast<int>(threadIdx.x) % size;
    while (pixel < p.pixels) {
      long long at_pixel[kTogether];
      int at_c[kTogether];
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        at_pixel[u] = pixel;
        at_c[u] = c;
        for (c += kNormThreads; c >= size; c -= size) ++pixel;
      }
      f(at_pixel, at_c);
    }
  };
  float shift = 0.0f, s1 = 0.0f, s2 = 0.0f;
  int n = 0;
  over([&](const long long (&pixel)[kTogether], const int (&c)[kTogether]) {
    T in[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; ++u)
      if (pixel[u] < p.pixels) in[u] = x[pixel[u] * p.x_pitch + c[u]];
    if (n == 0) shift = op_get(in[0]);
#pragma unroll
    for (int u = 0; u < kTogether; ++u)
      if (pixel[u] < p.pixels) {
        const float d = op_get(in[u]) - shift;
        s1 += d;
        s2 = fmaf(d, d, s2);
        ++n;
      }
    if ((n & (n - 1)) == 0) recentre(static_cast<float>(n), 1.0f / static_cast<float>(n), shift, s1, s2);
  });
  if (n > 0) recentre(static_cast<float>(n), 1.0f / static_cast<float>(n), shift, s1, s2);
  // the CTA's, about its first thread's mean (a group of one value has that for its mean, exactly)
  __shared__ float first;
  if (threadIdx.x == 0) first = shift;
  __syncthreads();
  const float about = first, count = static_cast<float>(p.pixels * size);
  const float mean = about + block_sum(n > 0 ? n * (shift - about) + s1 : 0.0f) / count;
  const float m2 = block_sum(n > 0 ? fmaf(n * (shift - mean), shift - mean, s2) : 0.0f);
  const float scale = 1.0f / sqrtf(m2 / count + p.eps);
  over([&](const long long (&pixel)[kTogether], const int (&c)[kTogether]) {
    T in[kTogether];
#pragma unroll
    for (int u = 0; u < kTogether; ++u)
      if (pixel[u] < p.pixels) in[u] = x[pixel[u] * p.x_pitch + c[u]];
#pragma unroll
    for (int u = 0; u < kTogether; ++u)
      if (pixel[u] < p.pixels) {
        const float v = fmaf((op_get(in[u]) - mean) * scale, p.gamma ? p.gamma[c0 + c[u]] : 1.0f, p.beta ? p.beta[c0 + c[u]] : 0.0f);
        y[pixel[u] * p.y_pitch + c[u]] = op_put<T>(norm_act<T, ACT>(v, p.floor));
      }
  });
}

template <class T, int V, int ACT>
int launch_shape(const NormParams& p, int take, int device, cudaStream_t st) {
  const int size = p.channels / p.groups, sms = op_sm_count(device);
  NormShape s{};
  s.channels = take * size;
  s.size = size;
  s.groups = take;
  s.columns = s.channels / V;
  s.rows = kNormThreads / s.columns;
  // (a graph's images are cut alike whatever the batch: a batch equals its images run alone, bit for bit)
  const long long items = (p.by_image ? 1 : p.n) * (p.groups / take);
  // CTAs to an item: two to an SM at most, while each thread has four pixels; a power of two (clusters of 9 or 13 leave SMs of a
  // GPC idle: 8 maps of 64 x 64 x 320 18 us with 8, 22 with 9)
  int ranks = 1;
  while (ranks < 16 && items * ranks * 2 <= 2 * sms && p.pixels > kNormGroup * ranks * static_cast<long long>(s.rows)) ranks *= 2;
  const long long each = (p.pixels + ranks - 1) / ranks;
  constexpr int kSlot = static_cast<int>(kNormThreads * sizeof(T) * V);
  constexpr int kSmem = kNormSlots<V> * kSlot + kNormThreads * V * static_cast<int>(sizeof(Moments));
  static_assert(kSmem * (3) <= (220 << 10), "shared memory of the CTAs of an SM");
  s.each = static_cast<int>(each);
  s.slots = static_cast<int>(std::min<long long>((each + s.rows - 1) / s.rows, kNormSlots<V>));
  const int smem = s.slots * kSlot + s.rows * s.channels * static_cast<int>(sizeof(Moments));
  const bool far = (each + s.rows - 1) / s.rows > kNormFirstMove;
  auto kernel = far ? k_group_norm<T, V, ACT, true> : k_group_norm<T, V, ACT, false>;
  static std::atomic<uint64_t> grants[2];
  std::atomic<uint64_t>& granted = grants[far ? 1 : 0];
  const uint64_t bit = 1ull << (device & 63);
  if (device >= 64 || !(granted.load(std::memory_order_acquire) & bit)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return op_launched("op_group_norm", e);
    if (device < 64) granted.fetch_or(bit, std::memory_order_acq_rel);
  }
  const long long images = 65535;  // blockIdx.z holds that many: more go in several launches
  for (long long at = 0; at < p.n; at += images) {
    NormParams q = p;
    q.n = std::min(images, p.n - at);
    q.x = static_cast<const T*>(p.x) + at * p.pixels * p.x_pitch;
    q.y = static_cast<T*>(p.y) + at * p.pixels * p.y_pitch;
    q.first_image = at;
    const dim3 grid(ranks, p.groups / take, static_cast<unsigned>(q.n));
    if (const cudaError_t e = op_launch(kernel, grid, kNormThreads, smem, st, ranks, q, s); e != cudaSuccess) return op_launched("op_group_norm", e);
  }
  return NCNN_B200_STATUS_SUCCESS;
}

template <class T, int V, int ACT>
int launch_act(const NormParams& p, int device, cudaStream_t st) {
  const int size = p.channels / p.groups, sms = op_sm_count(device);
  // The fewest groups whose channels are whole accesses and 128 bytes of a pixel; 64 to 16 where clusters of 16 CTAs to 128
  // bytes would be fewer than three quarters of the SMs (2 maps of 512 x 512 x 128: fp32 168, 186 and 397 us with 128, 64 and 32
  // bytes, bf16 176, 144 and 205).
  auto pick = [&](int bytes) {
    int take = 0;
    for (int g = 1; g <= p.groups; ++g) {
      if (p.groups % g != 0 || g * size % V != 0) continue;
      if (g * size / V > kNormThreads || g > kNormMostGroups) break;
      take = g;
      if (g * size * static_cast<int>(sizeof(T)) >= bytes) break;
    }
    return take;
  };
  int take = pick(128);
  for (int bytes = 64; bytes >= 16 && take > 0 && (p.by_image ? 1 : p.n) * (p.groups / take) * 16 * 4 < 3 * sms; bytes /= 2) take = pick(bytes);
  if (take == 0) {
    if (p.by_image) return NCNN_B200_STATUS_CONSTRAINT_VIOLATION;  // (the import refuses such groups)
    return op_launched("op_group_norm", op_launch(k_group_norm_wide<T, ACT>, dim3(static_cast<unsigned>(p.n * p.groups)), kNormThreads, 0, st, 0, p));
  }
  return launch_shape<T, V, ACT>(p, take, device, st);
}

template <class T, int V>
int launch(NormParams p, int activation, int device, cudaStream_t st) {
  p.floor = activation == NCNN_B200_ACT_RELU ? 0.0f : -INFINITY;
  switch (activation) {
    case NCNN_B200_ACT_SWISH: return launch_act<T, V, NCNN_B200_ACT_SWISH>(p, device, st);
    case NCNN_B200_ACT_GELU: return launch_act<T, V, NCNN_B200_ACT_GELU>(p, device, st);
    default: return launch_act<T, V, NCNN_B200_ACT_NONE>(p, device, st);
  }
}

}  // namespace

bool group_norm_fits(int channels, int groups) {
  const int size = channels / groups, v = channels % 4 == 0 ? 4 : 1;
  int take = 1;  // groups that are whole accesses together
  while (take <= groups && (groups % take != 0 || take * size % v != 0)) ++take;
  return take <= kNormMostGroups && take * size / v <= kNormThreads;
}

cudaError_t launch_group_norm(const ActRef& in, const ActRef& out, long long images, long long pixels, int channels, int groups, const float* gamma,
                              const float* beta, float eps, int act, int device, cudaStream_t st) {
  NormParams p{in.p0, out.p0, images, pixels, channels, channels, channels, groups, gamma, beta, eps, 0.0f, in, out, 0, 1};
  const int status = channels % 4 == 0 ? launch<float, 4>(p, act, device, st) : launch<float, 1>(p, act, device, st);
  return status == NCNN_B200_STATUS_SUCCESS ? cudaSuccess : cudaErrorLaunchFailure;
}

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
    if (!op_starts(x, op_elem_bytes(type)) || !op_starts(y, op_elem_bytes(type)) || !op_starts(gamma, 4) || !op_starts(beta, 4))
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_group_norm: an array does not start at a multiple of its elements' size");
    if (n == 0 || pixels == 0) return NCNN_B200_STATUS_SUCCESS;
    if (groups > 65535 || pixels > (1ll << 30) || pixels > (1ll << 40) / std::max(x_pitch, y_pitch) || n > (1ll << 40) / (pixels * std::max(x_pitch, y_pitch)) || n * groups > 0x7fffffffll)
      return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_group_norm: more than 2^30 pixels, 2^40 elements, 65535 groups of an image or 2^31 in all");
    std::string why;
    const int device = op_common_device(kOp, {x, y, gamma, beta}, &why);
    if (device < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, why);
    DeviceGuard guard(device);
    NormParams p{x, y, n, pixels, x_pitch, y_pitch, channels, groups, gamma, beta, eps, 0.0f, {}, {}, 0, 0};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // the widest access that every pixel's and every cluster's channels start and end with
    auto whole = [&](int v) {
      const uintptr_t bytes = static_cast<uintptr_t>(v) * op_elem_bytes(type);
      return reinterpret_cast<uintptr_t>(x) % bytes == 0 && reinterpret_cast<uintptr_t>(y) % bytes == 0 && channels % v == 0 && x_pitch % v == 0 &&
             y_pitch % v == 0;
    };
    const int status = op_by_type(type, [&](auto t) {
      using T = decltype(t);
      constexpr int V = 16 / sizeof(T);
      if constexpr (sizeof(T) == 4) {
        p.in.p0 = const_cast<float*>(static_cast<const float*>(x));
        p.out.p0 = static_cast<float*>(y);
      }
      if (whole(V)) return launch<T, V>(p, activation, device, st);
      if constexpr (sizeof(T) == 2)
        if (whole(2)) return launch<T, 2>(p, activation, device, st);
      return launch<T, 1>(p, activation, device, st);
    });
    return status;
  });
}
