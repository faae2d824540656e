// Attention of few queries (a decoding step) for 16-bit types: a pass over keys and values at HBM speed.
//
// The queries that read one key head (its heads' queries, 16 of them to a tile) are the rows of mma.sync m16n8k16 products;
// keys go 16 at a time, tile after tile, to the warps of a cluster of CTAs, and each warp keeps a running maximum, sum and
// result of its own.  tcgen05 has no use here: it would take 128 rows for the one to 16 that there are, and HBM is the bound
// (the products of a tile take a fifth of the time that its 8 KB take to arrive).
//
// Each warp has a ring of three to six tiles in shared memory that its own lanes fill with cp.async, whole rows at a time (HBM
// needs some 60 KB under way on each SM), 16-byte pieces exchanged by the row's number so that ldmatrix, which brings both
// operands into fragments, reads all banks; values are transposed by it on the way.
// Probabilities are split into two terms of the type, for which the products have room: 16 of their bits are kept in bf16, 22 in
// fp16 (fewer below 2^-14, none below 2^-25, of 2^-7 of the running maximum: kProbabilityLift).
// The warps' results are joined in shared memory, the CTAs' over distributed shared memory, in a fixed order.
#pragma once

#include <cooperative_groups.h>

#include "op_attention.h"

namespace nb {

constexpr int kFewRows = 16;
constexpr int kFewRanks = 16;  // CTAs of a cluster at most

struct FewParams {
  AttendParams a;
  float scale_log2;
  int row_tiles;  // of kFewRows (query, head of the key head) pairs
};

template <class T> __device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16x8x16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 bytes of global memory on their way to shared memory, or zeros
__device__ __forceinline__ void copy_16(uint32_t to, const void* from, bool take) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(take ? 16 : 0) : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// two probabilities as packed pairs of the type: the rounded ones, and what the rounding left
template <class T>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
  const T hx = op_put<T>(x), hy = op_put<T>(y);
  const OpVec<T, 2> h{{hx, hy}}, l{{op_put<T>(x - op_get(hx)), op_put<T>(y - op_get(hy))}};
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

template <class T, int D, int WARPS, int STAGES>
struct FewShared {
  static constexpr int kPieces = D / 8;  // 16-byte pieces of a row
  union {
    uint4 ring[WARPS][STAGES][2][16][kPieces];  // keys, then values
    struct {
      float part[WARPS][kFewRows][D + 4];  // the warps' results, then (in [0]) the CTA's
      float top[WARPS][kFewRows], total[WARPS][kFewRows];
      float cta_top[kFewRows], cta_total[kFewRows];
    };
  };
};

template <class T, int D, int WARPS, int STAGES, int BLOCKS>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS) k_attend_few(const __grid_constant__ FewParams p) {
  namespace cg = cooperative_groups;
  using Shared = FewShared<T, D, WARPS, STAGES>;
  constexpr int STEPS = D / 16, PIECES = Shared::kPieces, ROWS_A_COPY = 32 / PIECES;
  constexpr uint32_t STAGE_BYTES = 2 * 16 * PIECES * 16, VALUES = 16 * PIECES * 16;
  extern __shared__ __align__(128) uint8_t few_smem[];
  Shared& sh = *reinterpret_cast<Shared*>(few_smem);
  const AttendParams& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane >> 2, quad = lane & 3;
  const int rank = blockIdx.x, ranks = gridDim.x;
  const int kv_head = blockIdx.y / p.row_tiles, row0 = blockIdx.y % p.row_tiles * kFewRows;
  const int batch = blockIdx.z;
  const int shared = a.heads / a.kv_heads;
  const int rows = min(kFewRows, a.lq * shared - row0);
  const int keys = a.lens == nullptr ? a.lk : min(max(__ldg(a.lens + batch), 0), a.lk);
  const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + static_cast<long long>(batch) * a.lk;

  // copies: this lane's piece of rows lane / PIECES, + ROWS_A_COPY, ...
  const int copy_row = lane / PIECES, copy_piece = lane % PIECES;
  const bool copies = copy_piece * 8 < a.d;
  const T* k = static_cast<const T*>(a.k) + batch * a.k_batch + kv_head * a.k_head + (copies ? copy_piece * 8 : 0);
  const T* v = static_cast<const T*>(a.v) + batch * a.v_batch + kv_head * a.v_head + (copies ? copy_piece * 8 : 0);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(&sh.ring[warp][0]));
  const int step = ranks * WARPS * 16;
  const int first = (rank * WARPS + warp) * 16;
  // a byte of the mask for the tile's key `lane`, asked for a tile ahead of its use
  auto mask_of = [&](int j0) -> uint32_t {
    const int j = j0 + lane;
    return mask == nullptr || lane >= 16 || j >= keys ? 1u : __ldg(mask + j);
  };
  auto request = [&](int stage, int j0, uint32_t part) {
    if (j0 < keys) {
      const uint32_t to = ring + stage * STAGE_BYTES;
#pragma unroll
      for (int i = 0; i < 16 / ROWS_A_COPY; ++i) {
        const int r = copy_row + i * ROWS_A_COPY;
        const uint32_t at = to + static_cast<uint32_t>(r * PIECES + (copy_piece ^ (r & 7))) * 16u;
        const bool inside = copies && j0 + r < keys, used = copies && (part >> r & 1u);
        copy_16(at, k + (inside ? (j0 + r) * a.k_row : 0), inside);
        copy_16(at + VALUES, v + (used ? (j0 + r) * a.v_row : 0), used);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto parts_of = [&](int j0, uint32_t byte) { return __ballot_sync(~0u, lane < 16 && j0 + lane < keys && byte != 0); };

  uint32_t history[STAGES];  // the tiles under way: which keys take part
#pragma unroll
  for (int n = 0; n < STAGES - 1; ++n) {
    history[n] = parts_of(first + n * step, mask_of(first + n * step));
    request(n, first + n * step, history[n]);
  }
  uint32_t byte = mask_of(first + (STAGES - 1) * step);

  // the queries as A fragments: rows `group` and `group + 8`
  uint32_t q[STEPS][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = row0 + group + 8 * r;
    const T* at = static_cast<const T*>(a.q) + batch * a.q_batch + row / shared * a.q_row + (kv_head * shared + row % shared) * a.q_head;
#pragma unroll
    for (int c = 0; c < STEPS; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at_c = 16 * c + 8 * e + 2 * quad;
        q[c][r + 2 * e] = group + 8 * r < rows && at_c < a.d ? __ldg(reinterpret_cast<const uint32_t*>(at + at_c)) : 0u;
      }
  }
  float o[2 * STEPS][4] = {};
  float base[2] = {-INFINITY, -INFINITY}, total[2] = {0.0f, 0.0f};
  // where this lane's rows of the matrices lie: keys 8 (lane / 16) + lane % 8, piece (lane / 8) % 2 for Q K^T;
  // keys lane % 16, piece lane / 16 for P V
  const uint32_t k_row = static_cast<uint32_t>(8 * (lane >> 4) + (lane & 7)), k_piece = lane >> 3 & 1;
  const uint32_t v_row = static_cast<uint32_t>(lane & 15), v_piece = lane >> 4;

  int stage = 0;
  for (int j0 = first; j0 < keys; j0 += step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();  // every lane's copies are there, and the stage before this one has been read
    const int next = j0 + (STAGES - 1) * step;
    history[STAGES - 1] = parts_of(next, byte);
    request(stage == 0 ? STAGES - 1 : stage - 1, next, history[STAGES - 1]);
    byte = mask_of(next + step);
    const uint32_t part = history[0];
#pragma unroll
    for (int n = 0; n < STAGES - 1; ++n) history[n] = history[n + 1];
    const uint32_t k_at = ring + stage * STAGE_BYTES + k_row * PIECES * 16, v_at = ring + stage * STAGE_BYTES + VALUES + v_row * PIECES * 16;
    float s[2][2][4] = {};  // (two sums each: shorter chains)
#pragma unroll
    for (int c = 0; c < STEPS; ++c) {
      if (D == 256 && 16 * c >= a.d) break;  // (heads between 128 and 256 share an instantiation)
      uint32_t b[4];
      ldmatrix_x4(b, k_at + (((2 * c + k_piece) ^ (k_row & 7)) << 4));
      mma_16x8x16<T>(s[0][c & 1], q[c], b[0], b[1]);
      mma_16x8x16<T>(s[1][c & 1], q[c], b[2], b[3]);
    }
    // s[n][.][e]: row group + 8 (e / 2), key 8 n + 2 quad + e % 2
    const bool whole = part == 0xffffu;
    float x[2][4], m[2];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[n][e] = (s[n][0][e] + s[n][1][e]) * p.scale_log2;
        if (!whole && !(part >> (8 * n + 2 * quad + (e & 1)) & 1u)) x[n][e] = -INFINITY;
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      m[r] = fmaxf(fmaxf(x[0][2 * r], x[0][2 * r + 1]), fmaxf(x[1][2 * r], x[1][2 * r + 1]));
      m[r] = fmaxf(m[r], __shfl_xor_sync(~0u, m[r], 1));
      m[r] = fmaxf(m[r], __shfl_xor_sync(~0u, m[r], 2));
    }
    // the base of the exponentials follows the maximum when that is 2^8 or more above it
    if (__any_sync(~0u, m[0] > base[0] + 8.0f || m[1] > base[1] + 8.0f)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float to = fmaxf(base[r], m[r]);
        const float keep = to == -INFINITY ? 1.0f : exp2_approx(base[r] - to);
        base[r] = to;
        total[r] *= keep;
#pragma unroll
        for (int t = 0; t < 2 * STEPS; ++t) {
          o[t][2 * r] *= keep;
          o[t][2 * r + 1] *= keep;
        }
      }
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float from = base[r] == -INFINITY ? 0.0f : base[r] - kProbabilityLift<T>;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float e0 = exp2_approx(x[n][2 * r] - from), e1 = exp2_approx(x[n][2 * r + 1] - from);
        total[r] += e0 + e1;
        split_pair<T>(e0, e1, hi[2 * n + r], lo[2 * n + r]);
      }
    }
#pragma unroll
    for (int c = 0; c < STEPS; ++c) {
      if (D == 256 && 16 * c >= a.d) break;
      uint32_t b[4];
      ldmatrix_x4_trans(b, v_at + (((2 * c + v_piece) ^ (v_row & 7)) << 4));
      mma_16x8x16<T>(o[2 * c], lo, b[0], b[1]);
      mma_16x8x16<T>(o[2 * c + 1], lo, b[2], b[3]);
      mma_16x8x16<T>(o[2 * c], hi, b[0], b[1]);
      mma_16x8x16<T>(o[2 * c + 1], hi, b[2], b[3]);
    }
    stage = stage == STAGES - 1 ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // the results take the ring's place
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    total[r] += __shfl_xor_sync(~0u, total[r], 1);
    total[r] += __shfl_xor_sync(~0u, total[r], 2);
    if (quad == 0) {
      sh.top[warp][group + 8 * r] = base[r];
      sh.total[warp][group + 8 * r] = total[r];
    }
  }
  // o[t][e]: row group + 8 (e / 2), component 8 t + 2 quad + e % 2
#pragma unroll
  for (int r = 0; r < 2; ++r)
    if (group + 8 * r < rows)
#pragma unroll
      for (int t = 0; t < 2 * STEPS; ++t)
        *reinterpret_cast<float2*>(&sh.part[warp][group + 8 * r][8 * t + 2 * quad]) = make_float2(o[t][2 * r], o[t][2 * r + 1]);
  __syncthreads();
  // the CTA's
  for (int i = threadIdx.x; i < rows * (D / 4); i += WARPS * 32) {
    const int row = i / (D / 4), at = i % (D / 4) * 4;
    float m = sh.top[0][row];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) m = fmaxf(m, sh.top[w][row]);
    const float base = m == -INFINITY ? 0.0f : m;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float all = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = exp2f(sh.top[w][row] - base);
      const float4 x = *reinterpret_cast<const float4*>(&sh.part[w][row][at]);
      sum = make_float4(fmaf(f, x.x, sum.x), fmaf(f, x.y, sum.y), fmaf(f, x.z, sum.z), fmaf(f, x.w, sum.w));
      all = fmaf(f, sh.total[w][row], all);
    }
    *reinterpret_cast<float4*>(&sh.part[0][row][at]) = sum;  // (read above by this thread alone)
    if (at == 0) {
      sh.cta_top[row] = m;
      sh.cta_total[row] = all;
    }
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (ranks > 1) cluster.sync();
  else __syncthreads();
  // the cluster's: its CTAs share out the tile's pieces of eight components
  const int pieces = a.d / 8;
  for (int i = rank * WARPS * 32 + threadIdx.x; i < rows * pieces; i += ranks * WARPS * 32) {
    const int row = i / pieces, at = i % pieces * 8;
    // (every load of another CTA's memory takes some 700 clocks: they are asked for together)
    float tops[kFewRanks], factor[kFewRanks], m = -INFINITY;
#pragma unroll
    for (int c = 0; c < kFewRanks; ++c) tops[c] = c < ranks ? *cluster.map_shared_rank(&sh.cta_top[row], c) : -INFINITY;
#pragma unroll
    for (int c = 0; c < kFewRanks; ++c) {
      factor[c] = c < ranks ? *cluster.map_shared_rank(&sh.cta_total[row], c) : 0.0f;
      m = fmaxf(m, tops[c]);
    }
    const float base = m == -INFINITY ? 0.0f : m;
    float sum[8] = {}, all = 0.0f;
#pragma unroll
    for (int c = 0; c < kFewRanks; ++c) {
      const float f = exp2f(tops[c] - base);
      all = fmaf(f, factor[c], all);
      factor[c] = f;
    }
#pragma unroll
    for (int c0 = 0; c0 < kFewRanks; c0 += 4) {
      if (c0 >= ranks) break;
      float4 x[4][2];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4* from = reinterpret_cast<const float4*>(cluster.map_shared_rank(&sh.part[0][row][at], min(c0 + c, ranks - 1)));
        x[c][0] = from[0];
        x[c][1] = from[1];
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (c0 + c >= ranks) break;
        const float f = factor[c0 + c];
        sum[0] = fmaf(f, x[c][0].x, sum[0]);
        sum[1] = fmaf(f, x[c][0].y, sum[1]);
        sum[2] = fmaf(f, x[c][0].z, sum[2]);
        sum[3] = fmaf(f, x[c][0].w, sum[3]);
        sum[4] = fmaf(f, x[c][1].x, sum[4]);
        sum[5] = fmaf(f, x[c][1].y, sum[5]);
        sum[6] = fmaf(f, x[c][1].z, sum[6]);
        sum[7] = fmaf(f, x[c][1].w, sum[7]);
      }
    }
    const float scale = all == 0.0f ? 0.0f : 1.0f / all;
    OpVec<T, 8> out;
#pragma unroll
    for (int e = 0; e < 8; ++e) out.e[e] = op_put<T>(all == 0.0f ? 0.0f : sum[e] * scale);
    const int r = row0 + row;
    T* to = static_cast<T*>(a.o) + batch * a.o_batch + r / shared * a.o_row + (kv_head * shared + r % shared) * a.o_head + at;
    *reinterpret_cast<OpVec<T, 8>*>(to) = out;
  }
  if (ranks > 1) cluster.sync();  // no CTA's shared memory goes while another reads it
}

}  // namespace nb
