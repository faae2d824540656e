// Rows of numbers to 8-bit integers (ncnn_b200_op_quantize_rows) and products of tokens with them
// (ncnn_b200_op_inner_product_tokens).
#include <cmath>

#include "op_tokens.h"
#include "row_int8.cuh"
#include "tc_tokens.cuh"

namespace nb {
namespace {

// ------------------------------------------------------------------ rows to integers
// A row to WARPS warps, V elements to an access.  What a thread reads first it keeps (KEEP accesses: rows of up to 32 WARPS V KEEP
// elements are read once); the rest is read again out of the caches.  Bound: HBM.
template <class T, int V, int WARPS>
__global__ void __launch_bounds__(256) k_quantize_rows(const T* x, long long rows, int columns, long long x_pitch, int8_t* q, long long q_pitch,
                                                       float* steps) {
  constexpr int KEEP = WARPS == 1 ? 16 : 8, THREADS = WARPS * 32, ROWS = 256 / THREADS;
  using Vec = OpVec<T, V>;
  // Launched early, too, where a product follows: the trigger lets that one ask for its weights, which the kernel before this one may
  // have written, so it comes after the wait.
  ptx::grid_dependency_wait();
  ptx::grid_dependency_trigger();
  __shared__ uint32_t tops[8];
  const int lane = threadIdx.x % THREADS, warp = threadIdx.x >> 5;
  const long long row = static_cast<long long>(blockIdx.x) * ROWS + threadIdx.x / THREADS;
  const bool there = row < rows;
  const int count = there ? columns / V : 0;
  const Vec* from = reinterpret_cast<const Vec*>(x + (there ? row : 0) * x_pitch);
  Vec kept[KEEP];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (lane + i * THREADS < count) kept[i] = from[lane + i * THREADS];
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (lane + i * THREADS < count) top = row_top(kept[i], top);
  for (int i = lane + KEEP * THREADS; i < count; i += THREADS) top = row_top(from[i], top);
  top = __reduce_max_sync(~0u, row_top_bits<T>(top));
  if (WARPS > 1) {
    if ((threadIdx.x & 31) == 0) tops[warp] = top;
    __syncthreads();
    top = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = max(top, tops[warp / WARPS * WARPS + w]);
  }
  if (!there) return;
  const RowScale scale = row_scale<T>(top);
  if (lane == 0) steps[row] = scale.step;
  int8_t* to = q + row * q_pitch;
  auto put = [&](int i, const Vec& v) {
    if constexpr (V == 1) {
      to[i] = static_cast<int8_t>(row_integer<T>(op_get(v.e[0]), scale));
    } else {
      uint32_t w[V / 4];
#pragma unroll
      for (int g = 0; g < V / 4; ++g)
        w[g] = low_bytes(row_integer<T>(op_get(v.e[4 * g]), scale), row_integer<T>(op_get(v.e[4 * g + 1]), scale),
                         row_integer<T>(op_get(v.e[4 * g + 2]), scale), row_integer<T>(op_get(v.e[4 * g + 3]), scale));
      if constexpr (V == 8) *reinterpret_cast<uint2*>(to + i * 8) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(to + i * 4) = w[0];
    }
  };
  if (scale.factor == 0.0f) {
    for (int i = lane; i < count; i += THREADS) put(i, Vec{});
    return;
  }
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (lane + i * THREADS < count) put(lane + i * THREADS, kept[i]);
  for (int i = lane + KEEP * THREADS; i < count; i += THREADS) put(i, from[i]);
}

template <class T>
cudaError_t quantize_rows(bool early, const T* x, long long rows, int columns, long long x_pitch, int8_t* q, long long q_pitch, float* steps, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = columns % V == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && (rows == 1 || x_pitch % V == 0) &&
                    reinterpret_cast<uintptr_t>(q) % V == 0 && (rows == 1 || q_pitch % V == 0);
  // a warp to rows that it can keep, unless there are too few of them to fill the device
  const bool warps = wide && columns <= 32 * V * 16 && rows >= 2048;
  const long long ctas = warps ? (rows + 7) / 8 : rows;
  if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(ctas));
  if (!wide) return op_launch_early(early, k_quantize_rows<T, 1, 8>, grid, 256, 0, st, 0, x, rows, columns, x_pitch, q, q_pitch, steps);
  if (warps) return op_launch_early(early, k_quantize_rows<T, V, 1>, grid, 256, 0, st, 0, x, rows, columns, x_pitch, q, q_pitch, steps);
  return op_launch_early(early, k_quantize_rows<T, V, 8>, grid, 256, 0, st, 0, x, rows, columns, x_pitch, q, q_pitch, steps);
}

// ------------------------------------------------------------------ products at any alignment
// 64 x 64 results to a CTA, 32 bytes of every row a step, brought byte by byte where rows are not aligned; dp4a.
template <class T>
__global__ void __launch_bounds__(256) k_product_tokens(const TokensParams p) {
  __shared__ uint32_t a[64][9], b[64][9];  // (nine words a row: columns of threads read all banks)
  const long long t0 = static_cast<long long>(blockIdx.y) * 64;
  const long long c0 = static_cast<long long>(blockIdx.x) * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int sum[4][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += 32) {
    for (int i = threadIdx.x; i < 64 * 32; i += 256) {
      const int r = i >> 5, c = i & 31;
      reinterpret_cast<int8_t*>(&a[r][0])[c] = t0 + r < p.tokens && k0 + c < p.k ? p.q[(t0 + r) * p.q_pitch + k0 + c] : 0;
      reinterpret_cast<int8_t*>(&b[r][0])[c] = c0 + r < p.n && k0 + c < p.k ? p.weight[(c0 + r) * p.weight_pitch + k0 + c] : 0;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      int x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = static_cast<int>(a[ty + 16 * i][w]);
        y[i] = static_cast<int>(b[tx + 16 * i][w]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = __dp4a(x[i], y[j], sum[i][j]);
    }
    __syncthreads();
  }
  tokens_by_activation<T>(p.act, [&](auto loop) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long t = t0 + ty + 16 * i, c = c0 + tx + 16 * j;
        if (t < p.tokens && c < p.n)
          static_cast<T*>(p.y)[t * p.y_pitch + c] = tokens_result<T>(loop, sum[i][j], p.steps[t], p.weight_steps[c], p.bias == nullptr ? 0.0f : p.bias[c], p.act);
      }
  });
}

// ------------------------------------------------------------------ single tokens
// One or two tokens in one launch: a pass over the weights, a warp to a channel, 16 bytes to a lane and access, dp4a.  What bounds it is
// the weights' way from HBM and the time until the first of them are there; meanwhile every CTA quantises the tokens for itself (their
// bytes are few, and out of L2).  Nothing goes through the workspace.
constexpr int kOneThreads = 512, kOneAhead = 8;
constexpr int kOneSmem = 46 * 1024;

// fewer than 16 bytes, zeros behind them
__device__ __noinline__ uint4 last_bytes(const int8_t* from, int count) {
  uint32_t w[4] = {};
  for (int i = 0; i < count; ++i) w[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(from[i])) << (8 * (i % 4));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <class T, int M>
__global__ void __launch_bounds__(kOneThreads, 2) k_product_one(const T* x, long long x_pitch, const __grid_constant__ TokensParams p, int wide) {
  constexpr int WARPS = kOneThreads / 32, V = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t one_smem[];  // [M] rows of integers, zeros up to a multiple of 512
  __shared__ uint32_t tops[M][WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pieces = (p.k + 15) / 16, row = (p.k + 511) / 512 * 512;
  const int step = gridDim.x * WARPS;
  ptx::grid_dependency_wait();
  ptx::grid_dependency_trigger();
  // the first channel's weights.  A row's last piece may reach behind the row, as far as the pitch, where zeros stand in the tokens; the
  // last row need not have a pitch's bytes: its last piece is taken byte by byte.
  uint4 w[kOneAhead];
  auto ask = [&](int c, int i0) {
    const uint4* from = reinterpret_cast<const uint4*>(p.weight + c * p.weight_pitch) + lane;
#pragma unroll
    for (int i = 0; i < kOneAhead; ++i) {
      const int at = i0 + i * 32;
      w[i] = make_uint4(0u, 0u, 0u, 0u);
      if (c >= p.n || at + lane >= pieces) continue;
      if (c + 1 < p.n || (at + lane + 1) * 16 <= p.k) w[i] = __ldcs(from + at);
      else w[i] = last_bytes(p.weight + c * p.weight_pitch + (at + lane) * 16, p.k - (at + lane) * 16);
    }
  };
  int c = blockIdx.x * WARPS + warp;
  ask(c, 0);
  RowScale scale[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const T* from = x + (m < p.tokens ? m : 0) * x_pitch;
    uint32_t top = 0;
    if (wide) {
      for (int i = threadIdx.x; i < p.k / V; i += kOneThreads) top = row_top(reinterpret_cast<const OpVec<T, V>*>(from)[i], top);
    } else {
      for (int i = threadIdx.x; i < p.k; i += kOneThreads) top = row_top(reinterpret_cast<const OpVec<T, 1>*>(from)[i], top);
    }
    top = __reduce_max_sync(~0u, row_top_bits<T>(top));
    if (lane == 0) tops[m][warp] = top;
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < M; ++m) {
    scale[m] = row_scale<T>(__reduce_max_sync(~0u, lane < WARPS ? tops[m][lane] : 0u));
    const T* from = x + (m < p.tokens ? m : 0) * x_pitch;
    uint8_t* to = one_smem + m * row;
    const bool zeros = scale[m].factor == 0.0f;
    for (int i = threadIdx.x; i < row / V; i += kOneThreads) {
      uint32_t q[V];
      if (wide) {
        OpVec<T, V> v{};
        if (i * V < p.k) v = reinterpret_cast<const OpVec<T, V>*>(from)[i];
#pragma unroll
        for (int e = 0; e < V; ++e) q[e] = zeros ? 0u : row_integer<T>(op_get(v.e[e]), scale[m]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) q[e] = zeros || i * V + e >= p.k ? 0u : row_integer<T>(op_get(from[i * V + e]), scale[m]);
      }
#pragma unroll
      for (int g = 0; g < V / 4; ++g) reinterpret_cast<uint32_t*>(to + i * V)[g] = low_bytes(q[4 * g], q[4 * g + 1], q[4 * g + 2], q[4 * g + 3]);
    }
  }
  __syncthreads();
  const uint4* ints = reinterpret_cast<const uint4*>(one_smem);
  for (; c < p.n; c += step) {
    int sum[M] = {};
    for (int i0 = 0; i0 < pieces; i0 += 32 * kOneAhead) {
#pragma unroll
      for (int i = 0; i < kOneAhead; ++i) {
        const int at = i0 + i * 32 + lane;
        if (i0 + i * 32 >= pieces) break;
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const uint4 a = ints[m * (row / 16) + at];
          sum[m] = __dp4a(static_cast<int>(a.x), static_cast<int>(w[i].x), sum[m]);
          sum[m] = __dp4a(static_cast<int>(a.y), static_cast<int>(w[i].y), sum[m]);
          sum[m] = __dp4a(static_cast<int>(a.z), static_cast<int>(w[i].z), sum[m]);
          sum[m] = __dp4a(static_cast<int>(a.w), static_cast<int>(w[i].w), sum[m]);
        }
      }
      if (i0 + 32 * kOneAhead < pieces) ask(c, i0 + 32 * kOneAhead);
      else ask(c + step, 0);
    }
#pragma unroll
    for (int m = 0; m < M; ++m) sum[m] = __reduce_add_sync(~0u, sum[m]);
    // lane m finishes token m
    int mine = sum[0];
    float token_step = scale[0].step;
#pragma unroll
    for (int m = 1; m < M; ++m) {
      mine = lane == m ? sum[m] : mine;
      token_step = lane == m ? scale[m].step : token_step;
    }
    if (lane < M && lane < p.tokens) {
      T* y = static_cast<T*>(p.y) + lane * p.y_pitch + c;
      const float ws = __ldg(p.weight_steps + c), bias = p.bias == nullptr ? 0.0f : __ldg(p.bias + c);
      tokens_by_activation<T>(p.act, [&](auto loop) { *y = tokens_result<T>(loop, mine, token_step, ws, bias, p.act); });
    }
  }
}

// ------------------------------------------------------------------ tensor cores
// Rows of bytes as TMA sees them, boxes of 128 bytes of `box_rows` rows.
bool encode_bytes(CUtensorMap* map, const void* base, long long columns, long long rows, long long pitch, int box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {rows == 1 ? static_cast<cuuint64_t>((columns + 15) / 16 * 16) : static_cast<cuuint64_t>(pitch)};  // (a stride that is never stepped)
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)}, ones[2] = {1, 1};
  return encode_tiled()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Results as TMA stores them: 32 rows of 128 bytes.
template <class T>
bool encode_results(CUtensorMap* map, void* base, long long columns, long long rows, long long pitch) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch) * sizeof(T)};
  const cuuint32_t box[2] = {128 / sizeof(T), 32}, ones[2] = {1, 1};
  const CUtensorMapDataType kind = sizeof(T) == 4                          ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode_tiled()(map, kind, 2, base, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int no_token_maps() { return op_fail(NCNN_B200_STATUS_RUNTIME, "op_inner_product_tokens: the tensor maps could not be made"); }

template <class T>
int product_few(TcTokensParams p, int device, int sms, cudaStream_t st) {
  const TokensParams& t = p.t;
  p.columns = t.tokens >= 128 ? 128 : static_cast<int>((t.tokens + 15) / 16 * 16);
  p.tiles_c = (t.n + 127) / 128;
  auto tiles_of = [&](int columns) { return (t.tokens + columns - 1) / columns * p.tiles_c; };
  // Narrower tiles, down to 32 tokens, and then shares of the K blocks, until the SMs have a CTA each with a deep ring.  Tiles and ranks
  // of calls that leave SMs idle: 256 tokens through 4096 x 4096 64 x 1 13.5 us, 128 x 2 15.7; 333 through 1000 x 1234 32 x 1 10.0, 64 x 4
  // 11.1, 128 x 4 12.7; 128 through 4096 x 4096 32 x 1 12.4, 128 x 4 12.9.  64 tokens go the other way: 4096 x 4096 64 x 4 10.4, 32 x 2 10.8;
  // 4096 x 11008 64 x 1 14.5, 32 x 1 15.0, 64 x 2 (172 CTAs on 148 SMs) 16.8.
  while (t.tokens > 64 && p.columns > 32 && 2 * tiles_of(p.columns) <= sms) p.columns = (p.columns / 2 + 15) / 16 * 16;
  p.tiles_t = static_cast<int>((t.tokens + p.columns - 1) / p.columns);
  const long long tiles = tiles_of(p.columns);
  int ranks = 1;
  while (ranks < 8 && tiles * ranks * 2 <= sms && ranks * 2 <= p.k_blocks) ranks *= 2;
  if (tiles * ranks > (1 << 30)) return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_inner_product_tokens: too many tokens");
  p.t.ranks = ranks;
  p.stage_bytes = 16384 + p.columns * 128;
  const int room = tiles * ranks <= sms ? 200 * 1024 : 110 * 1024;  // one CTA to an SM, or two
  const int sums = ranks > 1 ? ranks * ((p.columns + ranks - 1) / ranks) * 512 : 0;
  p.stages = std::max(2, std::min({kTokStagesMost, (room - sums) / p.stage_bytes, (p.k_blocks + ranks - 1) / ranks}));
  const int smem = p.stages * p.stage_bytes + sums + 1024;
  CUtensorMap map_w, map_q;
  if (!encode_bytes(&map_w, t.weight, t.k, t.n, t.weight_pitch, 128) || !encode_bytes(&map_q, t.q, t.k, t.tokens, t.q_pitch, p.columns)) return no_token_maps();
  static std::atomic<uint64_t> granted{0};
  if (const cudaError_t e = op_grant_smem(tc_tokens_few_kernel<T>, 201 * 1024, device, &granted); e != cudaSuccess) return op_launched("op_inner_product_tokens", e);
  op_will_wait_on(device);
  return op_launched("op_inner_product_tokens", op_launch_early(true, tc_tokens_few_kernel<T>, dim3(static_cast<unsigned>(tiles * ranks)), kTokFewThreads, smem, st,
                                                                ranks > 1 ? ranks : 0, p, map_w, map_q));
}

template <class T>
int product_pair(TcTokensParams p, int columns, int device, int sms, cudaStream_t st) {
  const TokensParams& t = p.t;
  p.columns = columns;
  p.tiles_t = static_cast<int>((t.tokens + 255) / 256);
  p.tiles_c = (t.n + columns - 1) / columns;
  const long long tiles = static_cast<long long>(p.tiles_t) * p.tiles_c;
  if (tiles > (1 << 30)) return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_inner_product_tokens: too many tokens");
  p.stage_bytes = 16384 + columns / 2 * 128;
  p.stages = std::min(kTokStagesMost, (192 * 1024) / p.stage_bytes);
  // (rows whose ends are no multiple of 16 bytes: TMA stores fill the last 16 with what lies in the box behind the row)
  p.stored = reinterpret_cast<uintptr_t>(t.y) % 16 == 0 && t.n * static_cast<long long>(sizeof(T)) % 16 == 0 &&
                     t.y_pitch * static_cast<long long>(sizeof(T)) % 16 == 0 && t.y_pitch < (1ll << 37)
                 ? 1
                 : 0;
  const int smem = p.stages * p.stage_bytes + 8 * 4096 + 1024;
  CUtensorMap map_w, map_q, map_y{};
  if (!encode_bytes(&map_w, t.weight, t.k, t.n, t.weight_pitch, columns / 2) || !encode_bytes(&map_q, t.q, t.k, t.tokens, t.q_pitch, 128)) return no_token_maps();
  if (p.stored && !encode_results<T>(&map_y, t.y, t.n, t.tokens, t.y_pitch)) return no_token_maps();
  static std::atomic<uint64_t> granted{0};
  if (const cudaError_t e = op_grant_smem(tc_tokens_pair_kernel<T>, 226 * 1024, device, &granted); e != cudaSuccess) return op_launched("op_inner_product_tokens", e);
  op_will_wait_on(device);
  const int pairs = static_cast<int>(std::min<long long>(sms / 2, tiles));
  return op_launched("op_inner_product_tokens",
                     op_launch_early(true, tc_tokens_pair_kernel<T>, dim3(pairs * 2), kTokPairThreads, smem, st, 2, p, map_w, map_q, map_y));
}

template <class T>
cudaError_t product_one(const T* x, long long x_pitch, const TokensParams& t, int sms, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int wide = t.k % V == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && (t.tokens == 1 || x_pitch % V == 0) ? 1 : 0;
  const dim3 grid(std::min(2 * sms, (t.n + kOneThreads / 32 - 1) / (kOneThreads / 32)));
  const int row = (t.k + 511) / 512 * 512;
  if (t.tokens == 1) return op_launch_early(true, k_product_one<T, 1>, grid, kOneThreads, row, st, 0, x, x_pitch, t, wide);
  return op_launch_early(true, k_product_one<T, 2>, grid, kOneThreads, 2 * row, st, 0, x, x_pitch, t, wide);
}
// Whether a call takes k_product_one: its integers fit in shared memory without asking for more.  (Four tokens through 4096 x 4096: 10.2 us,
// 9.3 on the tensor cores; one: 5.8 and 9.1.)
bool one_fits(long long tokens, int k) { return tokens <= 2 && tokens * ((k + 511ll) / 512 * 512) <= kOneSmem; }

template <class T>
int product_tc(const TokensParams& t, int device, cudaStream_t st) {
  TcTokensParams p{};
  p.t = t;
  p.k_blocks = (t.k + 127) / 128;
  p.wait_ns = op_wait_ns(kTcWaitLimitNs);
  p.stall = op_stalled() ? 1 : 0;
  const int sms = op_sm_count(device);
  p.t.aligned = reinterpret_cast<uintptr_t>(t.weight_steps) % 16 == 0 && reinterpret_cast<uintptr_t>(t.bias) % 16 == 0 ? 1 : 0;
  // Tiles of 128 x 128 while two of them to an SM hold the call (1024 tokens through 4096 x 4096 24.1 us, 24.0 in pairs; 160 through
  // 4096 x 12288 22.2 and 22.6), otherwise pairs; their tiles' width by the columns that the busiest pair has (512 through
  // 4096 x 11008: 3 tiles of 128 29.7 us, 2 of 256 31.6, 128 x 128 37.3; 300 through 4096 x 14336: 4 of 128 50, 2 of 256 35).
  const long long rows = (t.tokens + 255) / 256, pairs = sms / 2;
  if ((t.tokens + 127) / 128 * ((t.n + 127) / 128) <= 2ll * sms) return product_few<T>(p, device, sms, st);
  auto busiest = [&](int columns) { return (rows * ((t.n + columns - 1) / columns) + pairs - 1) / pairs * columns; };
  return product_pair<T>(p, busiest(128) < busiest(256) ? 128 : 256, device, sms, st);
}

constexpr long long kTokensMost = 1ll << 31, kColumnsMost = 1 << 24, kSumMost = 131072;

long long padded_row(int k) { return (static_cast<long long>(k) + 15) / 16 * 16; }
// steps first, then the integers
long long steps_bytes(long long tokens) { return (tokens * 4 + 15) / 16 * 16; }

}  // namespace

cudaError_t tokens_gave_up(unsigned* count) { return cudaMemcpyFromSymbol(count, g_tokens_gave_up, sizeof *count); }

}  // namespace nb

extern "C" int ncnn_b200_op_quantize_rows(const void* x, int32_t type, int64_t rows, int32_t columns, int64_t x_pitch, int8_t* q, int64_t q_pitch,
                                          float* steps, void* stream) {
  using namespace nb;
  static const char* kOp = "op_quantize_rows";
  return op_guarded(kOp, [&]() -> int {
    if (!op_type_ok(type)) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_quantize_rows: unknown element type");
    if (rows < 0 || columns <= 0 || columns > kColumnsMost) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_quantize_rows: rows not below 0, columns 1 to 2^24");
    if (x_pitch == 0) x_pitch = columns;
    if (q_pitch == 0) q_pitch = columns;
    if (x_pitch < columns || q_pitch < columns) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_quantize_rows: a pitch is smaller than a row");
    if (rows > kTokensMost || x_pitch > (1ll << 50) / std::max<int64_t>(rows, 1) || q_pitch > (1ll << 50) / std::max<int64_t>(rows, 1))
      return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_quantize_rows: too many rows");
    if (rows == 0) return NCNN_B200_STATUS_SUCCESS;
    if (x == nullptr || q == nullptr || steps == nullptr) return op_fail(NCNN_B200_STATUS_NULL_POINTER, "op_quantize_rows: NULL argument");
    if (!op_starts(x, op_elem_bytes(type)) || !op_starts(steps, 4))
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_quantize_rows: an array does not start at a multiple of its elements' size");
    if (static_cast<const void*>(q) == x || static_cast<const void*>(steps) == x || static_cast<const void*>(steps) == q)
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_quantize_rows: the results must not lie over the input or each other");
    std::string why;
    const int device = op_common_device(kOp, {x, q, steps}, &why);
    if (device < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, why);
    DeviceGuard guard(device);
    return op_by_type(type, [&](auto t) {
      using T = decltype(t);
      return op_launched(kOp, quantize_rows<T>(false, static_cast<const T*>(x), rows, columns, x_pitch, q, q_pitch, steps, static_cast<cudaStream_t>(stream)));
    });
  });
}

extern "C" int64_t ncnn_b200_op_inner_product_tokens_workspace(int64_t tokens, int32_t k) {
  using namespace nb;
  if (tokens < 0 || tokens > kTokensMost || k <= 0 || k > kSumMost) return -1;
  return steps_bytes(tokens) + tokens * padded_row(k);
}

extern "C" int ncnn_b200_op_inner_product_tokens(const void* x, void* y, int32_t type, int64_t tokens, int32_t k, int32_t n, int64_t x_pitch,
                                                 int64_t y_pitch, const int8_t* weight, int64_t weight_pitch, const float* weight_steps,
                                                 const float* bias, int32_t activation, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace nb;
  static const char* kOp = "op_inner_product_tokens";
  return op_guarded(kOp, [&]() -> int {
    if (!op_type_ok(type)) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_inner_product_tokens: unknown element type");
    if (activation != NCNN_B200_ACT_NONE && activation != NCNN_B200_ACT_RELU && activation != NCNN_B200_ACT_SWISH && activation != NCNN_B200_ACT_GELU)
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_inner_product_tokens: unknown activation");
    if (tokens < 0 || k <= 0 || k > kSumMost || n <= 0 || n > kColumnsMost)
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_inner_product_tokens: tokens not below 0, k 1 to 131072, n 1 to 2^24");
    if (x_pitch == 0) x_pitch = k;
    if (y_pitch == 0) y_pitch = n;
    if (weight_pitch == 0) weight_pitch = k;
    if (x_pitch < k || y_pitch < n || weight_pitch < k) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_inner_product_tokens: a pitch is smaller than a row");
    const int64_t most = std::max<int64_t>(tokens, 1);
    if (tokens > kTokensMost || x_pitch > (1ll << 50) / most || y_pitch > (1ll << 50) / most || weight_pitch > (1ll << 50) / n)
      return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, "op_inner_product_tokens: too many tokens, or a pitch is too large");
    if (tokens == 0) return NCNN_B200_STATUS_SUCCESS;
    if (x == nullptr || y == nullptr || weight == nullptr || weight_steps == nullptr || workspace == nullptr)
      return op_fail(NCNN_B200_STATUS_NULL_POINTER, "op_inner_product_tokens: NULL argument");
    const int size = op_elem_bytes(type);
    if (!op_starts(x, size) || !op_starts(y, size) || !op_starts(weight_steps, 4) || !op_starts(bias, 4) || !op_starts(workspace, 16))
      return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_inner_product_tokens: an array does not start at a multiple of its elements' size (workspace: of 16 bytes)");
    if (workspace_bytes < ncnn_b200_op_inner_product_tokens_workspace(tokens, k))
      return op_fail(NCNN_B200_STATUS_OUTPUT_CAPACITY, "op_inner_product_tokens: the workspace is too small");
    for (const void* a : {x, static_cast<const void*>(weight), static_cast<const void*>(weight_steps), static_cast<const void*>(bias)})
      if (a == y || a == workspace || y == workspace)
        return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, "op_inner_product_tokens: the result and the workspace must not lie over an input or each other");
    std::string why;
    const int device = op_common_device(kOp, {x, y, weight, weight_steps, bias, workspace}, &why);
    if (device < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, why);
    DeviceGuard guard(device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    TokensParams p{};
    p.tokens = tokens;
    p.k = k;
    p.n = n;
    p.q_pitch = padded_row(k);
    p.weight_pitch = weight_pitch;
    p.y_pitch = y_pitch;
    float* steps = static_cast<float*>(workspace);
    int8_t* q = static_cast<int8_t*>(workspace) + steps_bytes(tokens);
    p.steps = steps;
    p.q = q;
    p.weight = weight;
    p.weight_steps = weight_steps;
    p.bias = bias;
    p.y = y;
    p.act = activation;
    return op_by_type(type, [&](auto t) {
      using T = decltype(t);
      const bool aligned = reinterpret_cast<uintptr_t>(weight) % 16 == 0 && (n == 1 || (weight_pitch % 16 == 0 && weight_pitch < (1ll << 39)));
      if (aligned && one_fits(tokens, k)) return op_launched(kOp, product_one<T>(static_cast<const T*>(x), x_pitch, p, op_sm_count(device), st));
      if (const cudaError_t e = quantize_rows<T>(true, static_cast<const T*>(x), tokens, k, x_pitch, q, p.q_pitch, steps, st); e != cudaSuccess) return op_launched(kOp, e);
      // (weights whose rows TMA cannot start at go through the CUDA cores)
      if (aligned) {
        if (encode_tiled() == nullptr) return op_fail(NCNN_B200_STATUS_RUNTIME, "op_inner_product_tokens: cuTensorMapEncodeTiled is not available from this driver");
        return product_tc<T>(p, device, st);
      }
      const long long rows = (tokens + 63) / 64, columns = (n + 63ll) / 64;
      // (a launch has at most 65535 rows of CTAs)
      for (long long r = 0; r < rows; r += 65535) {
        TokensParams part = p;
        part.tokens = std::min<long long>(tokens - r * 64, 65535ll * 64);
        part.q += r * 64 * p.q_pitch;
        part.steps += r * 64;
        part.y = static_cast<T*>(p.y) + r * 64 * p.y_pitch;
        const dim3 grid(static_cast<unsigned>(columns), static_cast<unsigned>(std::min<long long>(rows - r, 65535)));
        if (const cudaError_t e = op_launch(k_product_tokens<T>, grid, 256, 0, st, 0, part); e != cudaSuccess) return op_launched(kOp, e);
      }
      return static_cast<int>(NCNN_B200_STATUS_SUCCESS);
    });
  });
}
