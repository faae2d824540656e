// Attention on the CUDA cores, every product and sum in fp32: fp32 arrays, and 16-bit ones that the tensor-core kernels do not
// take (rows that do not start at multiples of 16 bytes).
#pragma once

#include <cooperative_groups.h>

#include "op_attention.h"

namespace nb {

// four components of a row from `c` on, fp32; zeros behind its end
template <class T, bool WIDE>
__device__ __forceinline__ float4 four_of(const T* row, int c, int d) {
  if constexpr (WIDE) {  // (d is a multiple of four, and so are all addresses)
    if (c >= d) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const OpVec<T, 4> v = *reinterpret_cast<const OpVec<T, 4>*>(row + c);
    return make_float4(op_get(v.e[0]), op_get(v.e[1]), op_get(v.e[2]), op_get(v.e[3]));
  } else {
    return make_float4(c < d ? op_get(row[c]) : 0.0f, c + 1 < d ? op_get(row[c + 1]) : 0.0f, c + 2 < d ? op_get(row[c + 2]) : 0.0f,
                       c + 3 < d ? op_get(row[c + 3]) : 0.0f);
  }
}

__device__ __forceinline__ float dot4(float4 a, float4 b, float c) { return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, c)))); }

constexpr int kF32Ranks = 8;  // CTAs of a cluster at most

struct F32Params {
  AttendParams a;
  float scale_log2;
  int row_tiles;
  int ranks;  // CTAs to a tile of many queries
};

// ------------------------------------------------------------------ few queries
// A pass over the keys.  The rows are (query, head of the key head) pairs, ROWS to a tile; a warp takes four keys at a time, eight
// lanes to a key, so that a lane holds the same components of queries, keys, values and results: scores are joined over eight
// lanes, results over everybody once, at the end.  The keys of a tile are cut over the warps of a cluster of CTAs.
// Bound: HBM (fp32 keys and values once a tile; ROWS of 4 take 1 product a byte).
constexpr int kSplitWarps = 8;

template <class T, int D, int ROWS, bool WIDE>
__global__ void __launch_bounds__(kSplitWarps * 32) k_attend_split(const __grid_constant__ F32Params p) {
  namespace cg = cooperative_groups;
  constexpr int PER = D / 32;  // pieces of four components of a lane: 4 (lane % 8) + 32 i
  __shared__ float top_of[kSplitWarps][ROWS], total_of[kSplitWarps][ROWS];
  __shared__ __align__(16) float part[kSplitWarps][ROWS][D];
  __shared__ float cta_top[ROWS], cta_total[ROWS];
  const AttendParams& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, at_key = lane >> 3, at_c = (lane & 7) * 4;
  const int rank = blockIdx.x, ranks = gridDim.x;
  const int kv_head = blockIdx.y / p.row_tiles, row0 = blockIdx.y % p.row_tiles * ROWS;
  const int batch = blockIdx.z, shared = a.heads / a.kv_heads;
  const int rows = min(ROWS, a.lq * shared - row0);
  const int keys = a.lens == nullptr ? a.lk : min(max(__ldg(a.lens + batch), 0), a.lk);
  const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + static_cast<long long>(batch) * a.lk;
  const T* k = static_cast<const T*>(a.k) + batch * a.k_batch + kv_head * a.k_head;
  const T* v = static_cast<const T*>(a.v) + batch * a.v_batch + kv_head * a.v_head;
  float4 q[ROWS][PER], o[ROWS][PER];
  float top[ROWS], total[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int row = row0 + r;
    const T* from = static_cast<const T*>(a.q) + batch * a.q_batch + row / shared * a.q_row + (kv_head * shared + row % shared) * a.q_head;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      o[r][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      q[r][i] = r < rows ? four_of<T, WIDE>(from, at_c + 32 * i, a.d) : o[r][i];
      q[r][i] = make_float4(q[r][i].x * p.scale_log2, q[r][i].y * p.scale_log2, q[r][i].z * p.scale_log2, q[r][i].w * p.scale_log2);
    }
    top[r] = -INFINITY;
    total[r] = 0.0f;
  }
  const int step = ranks * kSplitWarps * 4;
  for (int j0 = (rank * kSplitWarps + warp) * 4; j0 < keys; j0 += step) {
    const int j = j0 + at_key;
    const bool takes = j < keys && (mask == nullptr || __ldg(mask + j) != 0);
    float4 kk[PER], vv[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      kk[i] = vv[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (takes) {
        kk[i] = four_of<T, WIDE>(k + j * a.k_row, at_c + 32 * i, a.d);
        vv[i] = four_of<T, WIDE>(v + j * a.v_row, at_c + 32 * i, a.d);
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < PER; ++i) s = dot4(q[r][i], kk[i], s);
#pragma unroll
      for (int w = 4; w > 0; w >>= 1) s += __shfl_xor_sync(~0u, s, w);
      // each quarter of the warp has a running maximum of its own
      if (takes) {
        if (!(s <= top[r])) {  // (a NaN, too)
          const float next = fmaxf(top[r], s);
          const float keep = next == -INFINITY ? 1.0f : exp2f(top[r] - next);
          top[r] = next;
          total[r] *= keep;
#pragma unroll
          for (int i = 0; i < PER; ++i) o[r][i] = make_float4(o[r][i].x * keep, o[r][i].y * keep, o[r][i].z * keep, o[r][i].w * keep);
        }
        const float e = exp2f(s - (top[r] == -INFINITY ? 0.0f : top[r]));
        total[r] += e;
#pragma unroll
        for (int i = 0; i < PER; ++i)
          o[r][i] = make_float4(fmaf(e, vv[i].x, o[r][i].x), fmaf(e, vv[i].y, o[r][i].y), fmaf(e, vv[i].z, o[r][i].z), fmaf(e, vv[i].w, o[r][i].w));
      }
    }
  }
  // the warp's quarters, the CTA's warps, the cluster's CTAs, in this order
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    float m = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], 8));
    m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
    const float f = exp2f(top[r] - (m == -INFINITY ? 0.0f : m));
    auto over = [&](float x) {
      x *= f;
      x += __shfl_xor_sync(~0u, x, 8);
      return x + __shfl_xor_sync(~0u, x, 16);
    };
    const float all = over(total[r]);
    if (lane == 0) {
      top_of[warp][r] = m;
      total_of[warp][r] = all;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float4 x = make_float4(over(o[r][i].x), over(o[r][i].y), over(o[r][i].z), over(o[r][i].w));
      if (lane < 8) *reinterpret_cast<float4*>(&part[warp][r][at_c + 32 * i]) = x;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * D; i += kSplitWarps * 32) {
    const int r = i / D, c = i % D;
    float m = top_of[0][r];
    for (int w = 1; w < kSplitWarps; ++w) m = fmaxf(m, top_of[w][r]);
    const float base = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f, all = 0.0f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
      const float f = exp2f(top_of[w][r] - base);
      sum = fmaf(f, part[w][r][c], sum);
      all = fmaf(f, total_of[w][r], all);
    }
    part[0][r][c] = sum;  // (read above by this thread alone)
    if (c == 0) {
      cta_top[r] = m;
      cta_total[r] = all;
    }
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (ranks > 1) cluster.sync();
  else __syncthreads();
  for (int i = rank * kSplitWarps * 32 + threadIdx.x; i < rows * a.d; i += ranks * kSplitWarps * 32) {
    const int r = i / a.d, c = i % a.d;
    // (loads of other CTAs' memory are asked for together)
    float tops[kF32Ranks], totals[kF32Ranks], x[kF32Ranks], m = -INFINITY;
#pragma unroll
    for (int n = 0; n < kF32Ranks; ++n) {
      const int from = min(n, ranks - 1);
      tops[n] = *cluster.map_shared_rank(&cta_top[r], from);
      totals[n] = *cluster.map_shared_rank(&cta_total[r], from);
      x[n] = *cluster.map_shared_rank(&part[0][r][c], from);
    }
#pragma unroll
    for (int n = 0; n < kF32Ranks; ++n) m = fmaxf(m, tops[n]);
    const float base = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f, all = 0.0f;
#pragma unroll
    for (int n = 0; n < kF32Ranks; ++n)
      if (n < ranks) {
        const float f = exp2f(tops[n] - base);
        sum = fmaf(f, x[n], sum);
        all = fmaf(f, totals[n], all);
      }
    const int row = row0 + r;
    static_cast<T*>(a.o)[batch * a.o_batch + row / shared * a.o_row + (kv_head * shared + row % shared) * a.o_head + c] =
        op_put<T>(all == 0.0f ? 0.0f : sum / all);
  }
  if (ranks > 1) cluster.sync();  // no CTA's shared memory goes while another reads it
}

// ------------------------------------------------------------------ many queries
// A tile of rows (query, head of the key head) against blocks of KEYS keys, all in shared memory as fp32; 16 threads to TM rows.  A thread computes TM rows by KEYS / 16 keys of scores, then TM rows by D / 16 components of results out of the
// probabilities, which its own half warp wrote.  Every 4 x 4 products take two 16-byte loads of which one is a broadcast.
// Bound: the FMA pipe (32 of 74 TFLOP/s over 1024 x 1024, 64 heads of 64: half the issue slots are loads, addresses and the softmax).
// Where the tiles are fewer than the device holds, a tile's blocks of keys are dealt to the CTAs of a cluster, which join their
// results over distributed shared memory (2394 queries over 1768 keys, two heads of 128 on one key head: 498 us without, 176 so).
template <int D, int TM, int KEYS, int THREADS>
struct TileShape {
  static constexpr int kRows = THREADS / 16 * TM;
  static constexpr int kBlocksPerSm = D > 64 ? 1 : 2;  // (three, of 80 registers a thread, are slower)
  static constexpr int kPitch = D + 4;  // floats: rows start in different banks
  static constexpr int kSmem = (kRows * kPitch + KEYS * kPitch + KEYS * D + kRows * (KEYS + 4)) * 4;
};

template <class T, int D, int TM, int KEYS, int THREADS, bool WIDE>
__global__ void __launch_bounds__(THREADS, TileShape<D, TM, KEYS, THREADS>::kBlocksPerSm) k_attend_tile(const __grid_constant__ F32Params p) {
  namespace cg = cooperative_groups;
  using Shape = TileShape<D, TM, KEYS, THREADS>;
  constexpr int ROWS = Shape::kRows, PITCH = Shape::kPitch, TN = KEYS / 16, PER = D / 64;
  extern __shared__ __align__(16) float tile_smem[];
  float* qs = tile_smem;                // [row][component]
  float* ks = qs + ROWS * PITCH;        // [key][component]
  float* vs = ks + KEYS * PITCH;        // [key][component]
  float* ps = vs + KEYS * D;            // [row][key]
  __shared__ uint8_t takes[2][KEYS];
  const AttendParams& a = p.a;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int kv_head = blockIdx.y, batch = blockIdx.z, shared = a.heads / a.kv_heads;
  const int ranks = p.ranks, rank = blockIdx.x % ranks;
  const int all_rows = a.lq * shared, row0 = blockIdx.x / ranks * ROWS;
  const int keys = a.lens == nullptr ? a.lk : min(max(__ldg(a.lens + batch), 0), a.lk);
  const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + static_cast<long long>(batch) * a.lk;
  const T* k = static_cast<const T*>(a.k) + batch * a.k_batch + kv_head * a.k_head;
  const T* v = static_cast<const T*>(a.v) + batch * a.v_batch + kv_head * a.v_head;
  const int pieces = (a.d + 3) / 4;  // of four components; the others stay zero
  for (int i = threadIdx.x; i < ROWS * (D / 4); i += THREADS) {
    const int r = i / (D / 4), c = i % (D / 4) * 4, row = row0 + r;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (row < all_rows)
      x = four_of<T, WIDE>(static_cast<const T*>(a.q) + batch * a.q_batch + row / shared * a.q_row + (kv_head * shared + row % shared) * a.q_head, c, a.d);
    *reinterpret_cast<float4*>(qs + r * PITCH + c) = make_float4(x.x * p.scale_log2, x.y * p.scale_log2, x.z * p.scale_log2, x.w * p.scale_log2);
  }
  float top[TM], total[TM];
  float4 o[TM][PER];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    top[i] = -INFINITY;
    total[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < PER; ++c) o[i][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  // A block's keys are asked for when the last block's scores are done, its values when the last block's products are: fp32 rows
  // come by cp.async meanwhile.
  auto flag = [&](int at, int j0) {
    if (threadIdx.x < KEYS) {
      const int j = j0 + threadIdx.x;
      takes[at][threadIdx.x] = j < keys && (mask == nullptr || __ldg(mask + j) != 0);
    }
  };
  auto fetch = [&](float* to, int pitch, const T* from, long long stride, int j0, const uint8_t* part) {
    if (j0 < keys)
      for (int i = threadIdx.x; i < KEYS * (D / 4); i += THREADS) {
        const int r = i / (D / 4), c = i % (D / 4) * 4;
        const bool used = part[r] != 0 && c < a.d;
        if constexpr (WIDE && sizeof(T) == 4)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to + r * pitch + c))),
                       "l"(used ? from + (j0 + r) * stride + c : from), "r"(used ? 16 : 0)
                       : "memory");
        else
          *reinterpret_cast<float4*>(to + r * pitch + c) = used ? four_of<T, WIDE>(from + (j0 + r) * stride, c, a.d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int step = ranks * KEYS;
  int now = 0;
  flag(0, rank * KEYS);
  __syncthreads();
  fetch(ks, PITCH, k, a.k_row, rank * KEYS, takes[0]);
  fetch(vs, D, v, a.v_row, rank * KEYS, takes[0]);
  for (int j0 = rank * KEYS; j0 < keys; j0 += step, now ^= 1) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();  // the keys are there
    float s[TM][TN] = {};
#pragma unroll 2
    for (int c = 0; c < pieces; ++c) {
      float4 x[TM], y[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) x[i] = *reinterpret_cast<const float4*>(qs + (ty * TM + i) * PITCH + 4 * c);
#pragma unroll
      for (int n = 0; n < TN; ++n) y[n] = *reinterpret_cast<const float4*>(ks + (tx + 16 * n) * PITCH + 4 * c);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int n = 0; n < TN; ++n) s[i][n] = dot4(x[i], y[n], s[i][n]);
    }
    flag(now ^ 1, j0 + step);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the values are there, nobody needs the keys
    fetch(ks, PITCH, k, a.k_row, j0 + step, takes[now ^ 1]);
    uint32_t out = 0;  // this thread's keys without a part
#pragma unroll
    for (int n = 0; n < TN; ++n) out |= (takes[now][tx + 16 * n] ? 0u : 1u) << n;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      float m = top[i];
#pragma unroll
      for (int n = 0; n < TN; ++n) {
        if (out >> n & 1u) s[i][n] = -INFINITY;
        m = fmaxf(m, s[i][n]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, w));
      const float base = m == -INFINITY ? 0.0f : m;
      const float keep = exp2f(top[i] - base);
      top[i] = m;
      total[i] *= keep;
#pragma unroll
      for (int n = 0; n < TN; ++n) {
        const float e = exp2f(s[i][n] - base);
        total[i] += e;
        ps[(ty * TM + i) * (KEYS + 4) + tx + 16 * n] = e;
      }
#pragma unroll
      for (int c = 0; c < PER; ++c) o[i][c] = make_float4(o[i][c].x * keep, o[i][c].y * keep, o[i][c].z * keep, o[i][c].w * keep);
    }
    __syncwarp();
    const int left = min(KEYS, keys - j0);
    for (int j = 0; j < left; j += 4) {
      float4 e[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) e[i] = *reinterpret_cast<const float4*>(ps + (ty * TM + i) * (KEYS + 4) + j);
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int c = 0; c < PER; ++c) {
          const float4 y = *reinterpret_cast<const float4*>(vs + (j + n) * D + 64 * c + 4 * tx);
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            const float f = n == 0 ? e[i].x : n == 1 ? e[i].y : n == 2 ? e[i].z : e[i].w;
            o[i][c] = make_float4(fmaf(f, y.x, o[i][c].x), fmaf(f, y.y, o[i][c].y), fmaf(f, y.z, o[i][c].z), fmaf(f, y.w, o[i][c].w));
          }
        }
    }
    __syncthreads();  // nobody needs the values
    fetch(vs, D, v, a.v_row, j0 + step, takes[now ^ 1]);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (ranks > 1) {
    // a CTA's results take the place of its queries, and each CTA joins its share of the rows
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ float tops[ROWS], totals[ROWS];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      float all = total[i];
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) all += __shfl_xor_sync(~0u, all, w);
      const int r = ty * TM + i;
      if (tx == 0) {
        tops[r] = top[i];
        totals[r] = all;
      }
#pragma unroll
      for (int c = 0; c < PER; ++c) *reinterpret_cast<float4*>(qs + r * PITCH + 64 * c + 4 * tx) = o[i][c];
    }
    cluster.sync();
    const int share = (ROWS + ranks - 1) / ranks, from = rank * share;
    for (int i = threadIdx.x; i < share * (D / 4); i += THREADS) {
      const int r = from + i / (D / 4), c = i % (D / 4) * 4, row = row0 + r;
      if (r >= ROWS || row >= all_rows || c >= a.d) continue;
      float4 y[kF32Ranks];
      float their_top[kF32Ranks], their_total[kF32Ranks], m = -INFINITY;
#pragma unroll
      for (int n = 0; n < kF32Ranks; ++n) {
        const int of = min(n, ranks - 1);
        their_top[n] = *cluster.map_shared_rank(&tops[r], of);
        their_total[n] = *cluster.map_shared_rank(&totals[r], of);
        y[n] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(qs + r * PITCH + c, of));
      }
#pragma unroll
      for (int n = 0; n < kF32Ranks; ++n) m = fmaxf(m, their_top[n]);
      const float base = m == -INFINITY ? 0.0f : m;
      float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, all = 0.0f;
#pragma unroll
      for (int n = 0; n < kF32Ranks; ++n)
        if (n < ranks) {
          const float f = exp2f(their_top[n] - base);
          all = fmaf(f, their_total[n], all);
          x[0] = fmaf(f, y[n].x, x[0]);
          x[1] = fmaf(f, y[n].y, x[1]);
          x[2] = fmaf(f, y[n].z, x[2]);
          x[3] = fmaf(f, y[n].w, x[3]);
        }
      const float scale = all == 0.0f ? 0.0f : 1.0f / all;
      T* to = static_cast<T*>(a.o) + batch * a.o_batch + row / shared * a.o_row + (kv_head * shared + row % shared) * a.o_head + c;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < a.d) to[e] = op_put<T>(all == 0.0f ? 0.0f : x[e] * scale);
    }
    cluster.sync();  // no CTA's shared memory goes while another reads it
    return;
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    float all = total[i];
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) all += __shfl_xor_sync(~0u, all, w);
    const int row = row0 + ty * TM + i;
    if (row >= all_rows) continue;
    const float scale = all == 0.0f ? 0.0f : 1.0f / all;
    T* to = static_cast<T*>(a.o) + batch * a.o_batch + row / shared * a.o_row + (kv_head * shared + row % shared) * a.o_head;
#pragma unroll
    for (int c = 0; c < PER; ++c) {
      const int at = 64 * c + 4 * tx;
      const float x[4] = {o[i][c].x, o[i][c].y, o[i][c].z, o[i][c].w};
      if constexpr (WIDE) {
        OpVec<T, 4> out;
#pragma unroll
        for (int e = 0; e < 4; ++e) out.e[e] = op_put<T>(all == 0.0f ? 0.0f : x[e] * scale);
        if (at < a.d) *reinterpret_cast<OpVec<T, 4>*>(to + at) = out;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (at + e < a.d) to[at + e] = op_put<T>(all == 0.0f ? 0.0f : x[e] * scale);
      }
    }
  }
}

}  // namespace nb
