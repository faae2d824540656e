// Products of tokens in 8-bit integers on tensor cores: tcgen05.mma kind::i8, operands by TMA, exact int32 sums in tensor memory.
//
// tc_tokens_few_kernel: tiles of 128 channels x 16 to 128 tokens.  The weights are the 128-row operand, so that a call of one token
// multiplies 16 columns and not 128 rows; what bounds it is the weights' way from HBM.  The K blocks of a tile are dealt to the CTAs
// of a cluster (up to 8) while there are SMs without a CTA.  Each CTA finishes a share of the tokens: the others store their
// sums (integers: any order gives the same) into its shared memory, so that nobody waits for a load from another SM.
//
// tc_tokens_pair_kernel: tiles of 256 tokens x 256 or 128 channels on pairs of CTAs (cta_group::2), persistent, two accumulators in
// tensor memory so that a tile's results leave while the next one is summed.
//
// 64 tokens through 4096 x 11008 with Swish 15.1 us, of which the weights' bytes are 6.9; 8192 through 4096 x 8192 183 us with the 17 of the
// rows, 3.3 PFLOP/s in between.
//
// Either is launched while the kernel that quantises the tokens still runs (programmatic dependent launch): the weights of the first
// ring of K blocks are asked for before that kernel is waited for.
#pragma once

#include "op_tokens.h"
#include "ptx_sm100.cuh"
#include "tc_gemm_common.cuh"

namespace nb {

__device__ unsigned g_tokens_gave_up;  // CTAs in which a wait ran out, ever: ncnn_b200_op_check_status

constexpr int kTokStagesMost = 8;

struct TcTokensParams {
  TokensParams t;
  int k_blocks;     // of 128 integers
  int stages;
  int columns;      // few: tokens of a tile; pair: channels of a tile
  int tiles_t, tiles_c;
  int stage_bytes;
  int stored;       // pair: results leave through TMA
  int stall;        // tests of the time-out path: nothing is ever loaded (pair: by one of the CTAs, and one ring by the other)
  unsigned long long wait_ns;
};

constexpr int kTokFewThreads = 320;  // warps: 0 loads, 1 MMAs, 2 to 5 and 6 to 9 results of every second 16 tokens

__device__ __forceinline__ void store_cluster(uint32_t at, uint32_t v) { asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <class T>
__global__ void __launch_bounds__(kTokFewThreads, 2)
tc_tokens_few_kernel(const __grid_constant__ TcTokensParams p, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q) {
  using namespace ptx;
  extern __shared__ uint8_t tokens_smem[];
  __shared__ __align__(8) uint64_t full[kTokStagesMost], empty[kTokStagesMost], done;
  __shared__ float steps[128];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const int warp = __shfl_sync(~0u, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int ranks = p.t.ranks, rank = static_cast<int>(blockIdx.x) % ranks, tile = static_cast<int>(blockIdx.x) / ranks;
  const int c0 = tile / p.tiles_t * 128, t0 = tile % p.tiles_t * p.columns;
  const int kb0 = static_cast<int>(static_cast<long long>(p.k_blocks) * rank / ranks);
  const int count = static_cast<int>(static_cast<long long>(p.k_blocks) * (rank + 1) / ranks) - kb0;
  const uint32_t ring = (smem_u32(tokens_smem) + 1023u) & ~1023u;
  const int S = p.stages;
  const uint32_t stage_bytes = static_cast<uint32_t>(p.stage_bytes);
  const uint32_t tmem_cols = p.columns <= 32 ? 32u : p.columns <= 64 ? 64u : 128u;
  volatile int* abort_ptr = &abort_flag;

  // (the weights are asked for before the CTA is set up, which takes some 1500 clocks; one thread of warp 0 does all that TMA needs)
  const bool loads = warp == 0 && elect_one();
  const int ahead = p.stall == 0 ? min(count, S) : 0;
  if (loads) {
    abort_flag = 0;
    for (int i = 0; i < S; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), 1);
    }
    mbar_init(smem_u32(&done), 1);
    fence_mbar_init();
    for (int i = 0; i < ahead; ++i) {
      mbar_arrive_expect_tx(smem_u32(&full[i]), stage_bytes);
      tma_load_2d(ring + i * stage_bytes, &map_w, smem_u32(&full[i]), (kb0 + i) * 128, c0);
    }
    prefetch_tensormap(&map_q);
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (ranks > 1) cluster_arrive();  // (waited for below, where another CTA's memory is first written: it has begun by then)
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(~0u, tmem_slot, 0);
  auto gave_up = [&] {
    if (atomicCAS(&abort_flag, 0, 1) == 0) atomicAdd(&g_tokens_gave_up, 1u);
  };

  if (warp == 0) {
    if (loads) {
      int issued = ahead;
      if (p.stall == 0) {
        grid_dependency_wait();
        for (int i = 0; i < ahead; ++i) tma_load_2d(ring + i * stage_bytes + 16384u, &map_q, smem_u32(&full[i]), (kb0 + i) * 128, t0);
        int s = 0;
        uint32_t ph = 0;
        for (int i = ahead; i < count; ++i) {
          if (!mbar_wait_bounded(smem_u32(&empty[s]), ph, abort_ptr, p.wait_ns)) {
            gave_up();
            break;
          }
          mbar_arrive_expect_tx(smem_u32(&full[s]), stage_bytes);
          tma_load_2d(ring + s * stage_bytes, &map_w, smem_u32(&full[s]), (kb0 + i) * 128, c0);
          tma_load_2d(ring + s * stage_bytes + 16384u, &map_q, smem_u32(&full[s]), (kb0 + i) * 128, t0);
          issued = i + 1;
          if (++s == S) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      ring_landed(full, S, issued);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = instr_desc(2u, 1u, 128u, static_cast<uint32_t>(p.columns));
      bool ok = true, full_seen = false;  // (tested before a commit: see tc_gemm_common.cuh)
      int s = 0;
      uint32_t ph = 0;
      for (int i = 0; i < count; ++i) {
        ok = full_seen || mbar_wait_bounded(smem_u32(&full[s]), ph, abort_ptr, p.wait_ns);
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t a = smem_desc_kmajor(ring + s * stage_bytes, 128), b = smem_desc_kmajor(ring + s * stage_bytes + 16384u, 128);
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_i8(tmem, a + 2u * k, b + 2u * k, idesc, i > 0 || k > 0);
        const int next = s + 1 == S ? 0 : s + 1;
        if (next == 0) ph ^= 1u;
        full_seen = i + 1 < count && mbar_test_wait(smem_u32(&full[next]), ph);
        tc_commit(smem_u32(&empty[s]));
        s = next;
      }
      if (!ok) gave_up();
      tc_commit(smem_u32(&done));
      ring_landed(&done, 1, 1);  // (whoever gave up: nor may MMAs be under way when the CTA gives its memory back)
    }
  }
  __syncwarp();
  const int row = (warp & 3) * 32 + lane, c = c0 + row;  // (warps 2 to 5)
  const bool there = warp >= 2 && c < p.t.n;
  const uint32_t t_row = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
  const float ws = there ? __ldg(p.t.weight_steps + c) : 0.0f;
  const float bias = there && p.t.bias != nullptr ? __ldg(p.t.bias + c) : 0.0f;
  const int left = static_cast<int>(min(p.t.tokens - t0, static_cast<long long>(p.columns)));  // tokens of the tile
  T* const y = static_cast<T*>(p.t.y) + t0 * p.t.y_pitch + c;
  const int share = p.columns / ranks;  // (columns is a multiple of 16, ranks 1, 2, 4 or 8)
  const uint32_t sums = ring + static_cast<uint32_t>(S) * stage_bytes;  // [rank][token of the share][channel]
  const int group = (warp - 2) >> 2;
  bool ok = true;
  if (warp >= 2) {
    grid_dependency_wait();
    if (group == 0 && row < p.columns) steps[row] = row < left ? __ldcg(p.t.steps + t0 + row) : 0.0f;
    named_barrier_sync(1, 256);
    // (all of a tile's K blocks: a millisecond at most)
    ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&done), 0, abort_ptr, p.wait_ns) && *abort_ptr == 0);
    if (!ok && lane == 0) gave_up();
    tc_fence_after_sync();
  }
  // (few warps do this, each a long way: what counts is instructions, so that addresses are stepped and not computed)
  if (ranks == 1) {
    if (warp >= 2 && ok)
      tokens_by_activation<T>(p.t.act, [&](auto loop) {
#pragma unroll 1
        for (int at = group * 16; at < left; at += 32) {
          uint32_t v[16];
          tmem_ld16(t_row + static_cast<uint32_t>(at), v);
          tmem_ld_wait();
          T* to = y + at * p.t.y_pitch;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (there && at + j < left) *to = tokens_result<T>(loop, static_cast<int>(v[j]), steps[at + j], ws, bias, p.t.act);
            to += p.t.y_pitch;
          }
        }
      });
  } else {
    cluster_wait();
    if (warp >= 2 && ok) {
#pragma unroll 1
      for (int at = group * 16; at < p.columns; at += 32) {
        uint32_t v[16];
        tmem_ld16(t_row + static_cast<uint32_t>(at), v);
        tmem_ld_wait();
        int to = at / share, i = at - to * share;
        const uint32_t mine = sums + static_cast<uint32_t>(rank * share * 128 + row) * 4u;
        uint32_t slot = map_to_cta(mine, to) + static_cast<uint32_t>(i) * 512u;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          store_cluster(slot, v[j]);
          slot += 512u;
          if (++i == share) {
            i = 0;
            slot = map_to_cta(mine, min(++to, ranks - 1));
          }
        }
      }
    }
    __syncwarp();
    cluster_sync_all();
    if (warp >= 2 && ok) {
      const int first = rank * share, mine = min(share, left - first);
      tokens_by_activation<T>(p.t.act, [&](auto loop) {
#pragma unroll 1
        for (int i0 = group; i0 < mine; i0 += 8) {
          // four tokens at a time: their loads are under way together
          int sum[4] = {};
          const uint32_t from = sums + static_cast<uint32_t>(i0 * 128 + row) * 4u;
          for (int r = 0; r < ranks; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              int v = 0;
              if (i0 + 2 * j < mine) asm volatile("ld.shared.s32 %0, [%1];" : "=r"(v) : "r"(from + static_cast<uint32_t>(r * share) * 512u + j * 1024u));
              sum[j] += v;
            }
          T* to = y + (first + i0) * p.t.y_pitch;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (there && i0 + 2 * j < mine) *to = tokens_result<T>(loop, sum[j], steps[first + i0 + 2 * j], ws, bias, p.t.act);
            to += 2 * p.t.y_pitch;
          }
        }
      });
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, tmem_cols);
  }
}

constexpr int kTokPairThreads = 320;  // warps: 0 loads, 1 MMAs, 2 to 9 results

// A pair's copies in flight after one of its CTAs gave up.  They are counted on CTA 0's barriers, for both CTAs: of K blocks that only one
// of the two asked for, the other's part is made good, or the barrier's phase would never end.  (In a slot of the ring that can only be
// the last use: the one before has ended when either CTA goes on.)
__device__ __forceinline__ void pair_landed(const uint64_t* full, int stages, uint32_t stage_bytes, int uses0, int uses1) {
  for (int u = uses0; u < uses1; ++u) ptx::mbar_arrive_expect_tx(ptx::smem_u32(full + u % stages), stage_bytes);
  for (int u = uses1; u < uses0; ++u) ptx::mbar_complete_tx(ptx::smem_u32(full + u % stages), stage_bytes);
  ptx::ring_landed(full, stages, max(uses0, uses1));
}

template <class T>
__global__ void __launch_bounds__(kTokPairThreads, 1)
tc_tokens_pair_kernel(const __grid_constant__ TcTokensParams p, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q,
                      const __grid_constant__ CUtensorMap map_y) {
  using namespace ptx;
  extern __shared__ uint8_t tokens_smem[];
  __shared__ __align__(8) uint64_t full[kTokStagesMost];   // CTA 0's: the bytes of both CTAs
  __shared__ __align__(8) uint64_t empty[kTokStagesMost];  // in each CTA
  __shared__ __align__(8) uint64_t summed[2];              // in each CTA: an accumulator is complete
  __shared__ __align__(8) uint64_t drained[2];             // CTA 0's: both CTAs have read it
  __shared__ __align__(8) uint64_t last;                   // CTA 0's: no MMA is under way any more
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int asked, ends[2];  // K blocks that this CTA has asked for; both CTAs', less than 0 (~blocks) where one gave up
  const int warp = __shfl_sync(~0u, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = static_cast<int>(blockIdx.x) / 2, pairs = static_cast<int>(gridDim.x) / 2;
  const int tiles = p.tiles_t * p.tiles_c, KB = p.k_blocks, S = p.stages;
  const uint32_t ring = (smem_u32(tokens_smem) + 1023u) & ~1023u;
  const uint32_t stage_bytes = static_cast<uint32_t>(p.stage_bytes);  // 128 tokens' and half of the channels' rows
  volatile int* abort_ptr = &abort_flag;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < S; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&summed[i]), 1);
      mbar_init(smem_u32(&drained[i]), 16);
    }
    mbar_init(smem_u32(&last), 1);
    fence_mbar_init();
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_q);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&tmem_slot), 512u);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(~0u, tmem_slot, 0);
  auto gave_up = [&] {
    if (atomicCAS(&abort_flag, 0, 1) == 0) atomicAdd(&g_tokens_gave_up, 1u);
  };

  if (warp == 0) {
    if (elect_one()) {
      const int half = p.columns / 2;
      int issued = 0;  // K blocks of all tiles
      bool ok = p.stall == 0;
      const bool begins = ok || static_cast<uint32_t>(pair & 1) == rank;
      // (counters are stepped: a block's divisions took 900 clocks, its MMAs take 512)
      int s = 0;
      uint32_t ph = 0;
      const uint32_t full0 = map_to_cta(smem_u32(&full[0]), 0u);
      auto rows_of = [&](int tile, int* c0, int* t0) {
        *c0 = tile / p.tiles_t * p.columns + static_cast<int>(rank) * half;
        *t0 = tile % p.tiles_t * 256 + static_cast<int>(rank) * 128;
      };
      // the first ring of weights, and when the kernel before has ended, its tokens
      int tile = pair, kb = 0, c0 = 0, t0 = 0;
      rows_of(tile, &c0, &t0);
      for (int pass = 0; begins && pass < 2; ++pass) {
        if (pass == 1) grid_dependency_wait();
        tile = pair;
        kb = 0;
        rows_of(tile, &c0, &t0);
        for (issued = 0; issued < S && tile < tiles; ++issued) {
          if (pass == 0) {
            if (rank == 0) mbar_arrive_expect_tx(smem_u32(&full[issued]), 2u * stage_bytes);
            tma_load_2d_pair(ring + issued * stage_bytes + 16384u, &map_w, full0 + issued * 8u, kb * 128, c0);
          } else {
            tma_load_2d_pair(ring + issued * stage_bytes, &map_q, full0 + issued * 8u, kb * 128, t0);
          }
          if (++kb == KB) {
            kb = 0;
            tile += pairs;
            rows_of(tile, &c0, &t0);
          }
        }
      }
      for (; ok && tile < tiles; tile += pairs, kb = 0) {
        rows_of(tile, &c0, &t0);
        for (; kb < KB; ++kb) {
          if (!mbar_wait_bounded(smem_u32(&empty[s]), ph, abort_ptr, p.wait_ns)) {
            ok = false;
            gave_up();
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(smem_u32(&full[s]), 2u * stage_bytes);
          tma_load_2d_pair(ring + s * stage_bytes + 16384u, &map_w, full0 + s * 8u, kb * 128, c0);
          tma_load_2d_pair(ring + s * stage_bytes, &map_q, full0 + s * 8u, kb * 128, t0);
          ++issued;
          if (++s == S) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      asked = issued;
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = instr_desc(2u, 1u, 256u, static_cast<uint32_t>(p.columns));
      const uint64_t a_first = smem_desc_kmajor(ring, 128), b_first = smem_desc_kmajor(ring + 16384u, 128), step = stage_bytes >> 4;
      int s = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      bool full_seen = false, drained_seen = false;  // (tested before a commit: see tc_gemm_common.cuh)
      for (int tile = pair; ok && tile < tiles; tile += pairs) {
        if (!drained_seen && !mbar_wait_bounded(smem_u32(&drained[acc]), acc_ph ^ 1u, abort_ptr, p.wait_ns)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t d = tmem + static_cast<uint32_t>(acc) * 256u;
        for (int kb = 0; kb < KB; ++kb) {
          if (!full_seen && !mbar_wait_bounded(smem_u32(&full[s]), ph, abort_ptr, p.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint64_t a = a_first + static_cast<uint64_t>(s) * step, b = b_first + static_cast<uint64_t>(s) * step;
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_i8_pair(d, a + 2u * k, b + 2u * k, idesc, kb > 0 || k > 0);
          const int next = s + 1 == S ? 0 : s + 1;
          const uint32_t next_ph = next == 0 ? ph ^ 1u : ph;
          full_seen = mbar_test_wait(smem_u32(&full[next]), next_ph);
          if (kb + 1 == KB) drained_seen = mbar_test_wait(smem_u32(&drained[acc ^ 1]), acc == 1 ? acc_ph : acc_ph ^ 1u);
          tc_commit_pair(smem_u32(&empty[s]), 3);
          s = next;
          ph = next_ph;
        }
        if (!ok) break;
        tc_commit_pair(smem_u32(&summed[acc]), 3);
        acc ^= 1;
        if (acc == 0) acc_ph ^= 1u;
      }
      if (!ok) gave_up();
      // MMAs under way are done before the CTAs leave, whoever gave up
      tc_commit_pair(smem_u32(&last), 1);
      ring_landed(&last, 1, 1);
    }
  } else {
    grid_dependency_wait();
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) * 32u;
    const int group = (warp - 2) >> 2;  // the first or second half of the columns
    const int half = p.columns / 2;
    const uint32_t drained0 = map_to_cta(smem_u32(&drained[0]), 0u), drained1 = map_to_cta(smem_u32(&drained[1]), 0u);
    const uint32_t staged = ring + static_cast<uint32_t>(S) * stage_bytes + static_cast<uint32_t>(warp - 2) * 4096u;
    constexpr int WIDE = 128 / static_cast<int>(sizeof(T));  // columns of a staged row
    int acc = 0;
    uint32_t acc_ph = 0;
    bool ok = true;
    for (int tile = pair; ok && tile < tiles; tile += pairs) {
      const long long first = tile % p.tiles_t * 256ll + rank * 128ll + lanes, t = first + lane;
      const int c0 = tile / p.tiles_t * p.columns + group * half;
      const float step = t < p.t.tokens ? __ldcg(p.t.steps + t) : 0.0f;
      ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&summed[acc]), acc_ph, abort_ptr, p.wait_ns));
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t at_tmem = tmem + (lanes << 16) + static_cast<uint32_t>(acc) * 256u + static_cast<uint32_t>(group * half);
      tokens_by_activation<T>(p.t.act, [&](auto loop) {
#pragma unroll 1
      for (int at = 0; at < half; at += WIDE) {
        if (p.stored) {
          if (lane == 0) bulk_wait_read();
          __syncwarp();
        }
#pragma unroll
        for (int w = 0; w < WIDE / 16; ++w) {
          uint32_t v[16];
          tmem_ld16(at_tmem + static_cast<uint32_t>(at + 16 * w), v);
          tmem_ld_wait();
          const int c = c0 + at + 16 * w;
          T y[16];
          if (c + 16 <= p.t.n && (p.t.aligned & 1)) {
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              const float4 ws = __ldg(reinterpret_cast<const float4*>(p.t.weight_steps + c + j));
              const float4 b = p.t.bias == nullptr ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : __ldg(reinterpret_cast<const float4*>(p.t.bias + c + j));
              y[j] = tokens_result<T>(loop, static_cast<int>(v[j]), step, ws.x, b.x, p.t.act);
              y[j + 1] = tokens_result<T>(loop, static_cast<int>(v[j + 1]), step, ws.y, b.y, p.t.act);
              y[j + 2] = tokens_result<T>(loop, static_cast<int>(v[j + 2]), step, ws.z, b.z, p.t.act);
              y[j + 3] = tokens_result<T>(loop, static_cast<int>(v[j + 3]), step, ws.w, b.w, p.t.act);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const bool there = c + j < p.t.n;
              y[j] = tokens_result<T>(loop, static_cast<int>(v[j]), step, there ? __ldg(p.t.weight_steps + c + j) : 0.0f,
                                      there && p.t.bias != nullptr ? __ldg(p.t.bias + c + j) : 0.0f, p.t.act);
            }
          }
          if (p.stored) {
            constexpr int PIECES = 16 * static_cast<int>(sizeof(T)) / 16;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                OpVec<T, 16 / sizeof(T)> u;
#pragma unroll
              for (int e = 0; e < static_cast<int>(16 / sizeof(T)); ++e) u.e[e] = y[i * static_cast<int>(16 / sizeof(T)) + e];
              const uint4 b = *reinterpret_cast<const uint4*>(&u);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staged + lane * 128 + (((w * PIECES + i) ^ (lane & 7)) << 4)), "r"(b.x), "r"(b.y),
                           "r"(b.z), "r"(b.w)
                           : "memory");
            }
          } else if (t < p.t.tokens) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (c + j < p.t.n) static_cast<T*>(p.t.y)[t * p.t.y_pitch + c + j] = y[j];
          }
        }
        if (p.stored) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && first < p.t.tokens && c0 + at < p.t.n) {
            tma_store_2d(&map_y, staged, c0 + at, static_cast<int>(first));
            bulk_commit();
          }
        }
      }
      });
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc ? drained1 : drained0);
      acc ^= 1;
      if (acc == 0) acc_ph ^= 1u;
    }
    if (!ok && lane == 0) gave_up();
    if (p.stored && lane == 0) bulk_wait_read();
  }
  // Neither CTA leaves while the other may signal its barriers or read its shared memory, or while copies are in flight: where nobody gave up
  // the MMAs have waited for all of them.
  tc_fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int mine = abort_flag != 0 ? ~asked : asked;
    ends[rank] = mine;
    store_cluster(map_to_cta(smem_u32(&ends[rank]), rank ^ 1u), static_cast<uint32_t>(mine));
  }
  __syncwarp();
  cluster_sync_all();
  tc_fence_after_sync();
  if (ends[0] < 0 || ends[1] < 0) {
    if (rank == 0 && threadIdx.x == 0) pair_landed(full, S, stage_bytes, ends[0] < 0 ? ~ends[0] : ends[0], ends[1] < 0 ? ~ends[1] : ends[1]);
    __syncwarp();
    cluster_sync_all();
  }
  if (warp == 1) tmem_dealloc_pair(tmem, 512u);
}

}  // namespace nb
