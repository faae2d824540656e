// Attention over a paged cache of 8-bit integers for many rows, 16-bit types: tcgen05 MMAs over tiles that warps convert on their way.
//
// A CTA has two tiles of 128 rows that read one key head (a row is a token and one of the head's query heads; of one sequence, or, for
// a shared prefix, of all) and walks a range of keys in blocks of 128 with a running maximum and sum, as tc_attend.cuh does:
//   S = Q K^T, P = 2^(S ks c - m) vs over S in tensor memory, O += P V
// Scores of a block lie in two halves of 64 keys, each with barriers of its own: while the softmax has one half, the other half's
// products and its scores of the next block are made, so that a softmax never waits for the MMAs (one buffer for whole blocks: 4420
// clocks a block, 3290 of them in the softmax).
// Integers are exact in 16 bits, so that keys and values are converted as they are and the steps ks, vs of a key meet its column in the
// softmax.  P goes in as two bf16 terms (16 bits, and a range that holds any step) and two products, as in the kernel for few rows: which of
// the two a call takes, by the largest number of rows in its batch or by a shared prefix, does not show in its results.
//
// Roles: warp 6 brings blocks, 16 keys of a page to a bulk copy, into a ring of three; warps 0 to 5 convert them (16 bytes to 32) and
// store them as TMA would with a 128-byte swizzle, keys and values in turn, in a second ring of three; warp 7 issues the MMAs; warps
// 8 to 11 are tile 0's softmax, 12 to 15 tile 1's.  256 rows to a CTA share a conversion.
//
// Bound: the chain of a block, scores - softmax - products, which two tiles and two halves hide in part.  A block's MMAs (two tiles: 1024
// clocks for the scores, as many for each term of P) read 320 KB of operands, converting moves 128 KB and every softmax warp reads the
// steps, some 4100 clocks at 128 bytes a clock; a block takes 5200, with the tensor pipe active for 51 % of them, shared memory's banks
// for 63 % and the issue slots for 58 %.
// Pieces of up to 2048 tokens of 4 sequences behind up to 4096, 32 heads on 8 of 128: bf16 460 us, 588 TFLOP/s, f16 471 (with P rounded
// once to bf16 404 us, but results 2.3e-3 off where their own rounding makes 1.7e-3; with every eighth pair of exponentials on the FMA pipe,
// as tc_attend.cuh has them, 463 and 471, every fourth 473 and 485).
#pragma once

#include "attend_cache.cuh"
#include "tc_attend.cuh"

namespace nb {

__device__ unsigned g_cache_gave_up;  // CTAs in which a wait ran out, ever: ncnn_b200_op_check_status

struct TcCacheParams {
  AttendCacheParams a;
  int q_wide;  // 16 bytes of q can be read at a time
  int stall;   // tests of the time-out path: no block is ever brought
  unsigned long long wait_ns;
};

template <int D>
struct TcCacheShape {
  static constexpr int kThreads = 512, kConverters = 6;
  static constexpr int kPanel = 128 * 128;  // 128 rows of 64 components
  static constexpr int kTile = kPanel * (D / 64);
  static constexpr int kSlots = 3, kSteps = 8, kQueue = 3;
  static constexpr int kUnits = 128 * D / 512;            // of 32 pieces of 16 bytes, in a block of keys or values
  static constexpr int kUnitsAWarp = (kUnits + kConverters - 1) / kConverters;
  static constexpr int kQueueTile = 128 * D;
  static constexpr int kRegsLaunch = 128, kRegsControl = 56, kRegsSoftmax = 200;
  static_assert(256 * kRegsControl + 256 * kRegsSoftmax <= kThreads * kRegsLaunch, "registers of the roles");
  static constexpr uint32_t kTmemCols = 512;
  static constexpr int kSmem = 1024 + 2 * kTile + kSlots * kTile + kQueue * kQueueTile + kSteps * 1024;
};

// one pair of columns: scores times the keys' steps
__device__ __forceinline__ uint64_t f32x2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <class T, int D>
__global__ void __launch_bounds__(TcCacheShape<D>::kThreads, 1) tc_attend_cache_kernel(const __grid_constant__ TcCacheParams p) {
  using namespace ptx;
  using Shape = TcCacheShape<D>;
  constexpr int kTile = Shape::kTile, kPanel = Shape::kPanel, kSlots = Shape::kSlots, kSteps = Shape::kSteps;
  constexpr bool HALF = std::is_same<T, __half>::value;
  extern __shared__ uint8_t cache_smem[];
  __shared__ __align__(8) uint64_t brought[Shape::kQueue], taken[Shape::kQueue];
  __shared__ __align__(8) uint64_t q_full, full[kSlots], empty[kSlots], steps_full[kSteps], s_full[2][2], p_full[2][2], o_done[2][2], o_full[2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, pages_there[kSteps];
  const AttendCacheParams& a = p.a;
  const CacheParams& c = a.c;
  const int warp = __shfl_sync(~0u, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int range = blockIdx.y, kv_head = static_cast<int>(blockIdx.x % c.kv_heads), G = a.rows_a_head;
  grid_dependency_trigger();

  // rows: 256 from row0 on (the last ones of all heads first: their walks are the longest)
  const int at = static_cast<int>((gridDim.x - 1 - blockIdx.x) / c.kv_heads);
  int sequence = 0;
  long long row0 = static_cast<long long>(at) * 256, first = 0, rows;
  int before = 0;
  if (a.prefix) {
    rows = c.tokens * G;
  } else {
    sequence = at % c.sequences;
    row0 = static_cast<long long>(at / c.sequences) * 256;
    first = cache_start(c, sequence);
    const long long count = max(cache_start(c, sequence + 1) - first, 0ll);
    rows = min(count, static_cast<long long>(c.max_tokens)) * G;
    before = static_cast<int>(max(cache_len(c, sequence) - count, -(1ll << 30)));
  }
  // the CTA's last position: of a sequence's rows it is the last one's; of all tokens' any may be the last
  int last = -2;
  if (row0 < rows) {
    const long long end_row = min(rows, row0 + 256) - 1;
    if (a.prefix) {
      for (long long t = row0 / G + lane; t <= end_row / G; t += 32) {
        const CachePlace place = cache_place(c, t);
        if (place.sequence >= 0) last = max(last, place.position);
      }
      last = __reduce_max_sync(~0u, last);
    } else {
      last = max(before + static_cast<int>(end_row / G), -1);
    }
  }
  const int from = a.prefix ? range * a.chunk : a.shared + range * a.chunk;
  const int end = a.prefix ? min(a.shared, last + 1) : last + 1;
  const int to = min(from + a.chunk, end);
  if (last == -2 || (from >= to && a.part != nullptr)) {
    grid_dependency_wait();
    return;
  }
  const int blocks = from < to ? (to - from + 127) / 128 : 0;
  const int tiles = row0 + 128 < rows ? 2 : 1;
  const uint32_t smem = (smem_u32(cache_smem) + 1023u) & ~1023u;
  const uint32_t q_at = smem, ring = smem + 2 * kTile, queue = ring + kSlots * kTile, steps_at = queue + Shape::kQueue * Shape::kQueueTile;
  volatile int* abort_ptr = &abort_flag;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    mbar_init(smem_u32(&q_full), 4u * tiles);
    mbar_init(smem_u32(&drained), 1);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(smem_u32(&full[i]), Shape::kConverters);
      mbar_init(smem_u32(&empty[i]), 1);
    }
    for (int i = 0; i < Shape::kQueue; ++i) {
      mbar_init(smem_u32(&brought[i]), 1);
      mbar_init(smem_u32(&taken[i]), Shape::kConverters);
    }
    for (int i = 0; i < kSteps; ++i) mbar_init(smem_u32(&steps_full[i]), Shape::kConverters);
    for (int t = 0; t < 2; ++t) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(smem_u32(&s_full[t][h]), 1);
        mbar_init(smem_u32(&p_full[t][h]), 4);
        mbar_init(smem_u32(&o_done[t][h]), 1);
      }
      mbar_init(smem_u32(&o_full[t]), 1);
    }
    fence_mbar_init();
  }
  if (warp == 7) {
    tmem_alloc(smem_u32(&tmem_slot), Shape::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(~0u, tmem_slot, 0);
  auto gave_up = [&] {
    if (atomicCAS(&abort_flag, 0, 1) == 0) atomicAdd(&g_cache_gave_up, 1u);
  };
  auto s_of = [&](int t) { return tmem + 128u * t; };
  auto o_of = [&](int t) { return tmem + 256u + static_cast<uint32_t>(D * t); };

  if (warp < 8) {
    reg_dealloc<Shape::kRegsControl>();
    if (warp < Shape::kConverters) {
      // ---- blocks of keys and values converted: a unit is a lane's 16 bytes of each of some rows
      constexpr int PIECES = D / 16, UNIT_ROWS = 32 / PIECES, UNITS = Shape::kUnitsAWarp;
      const int piece = lane % PIECES, row_in = lane / PIECES;
      const bool used_piece = piece * 16 < c.row;
      // where this lane's pieces go: 16 bytes become 32, that is, pieces 2 piece and 2 piece + 1 of a row of components.
      // The lanes of the second panel store them the other way round, so that eight neighbours reach all banks.
      const uint32_t panel = static_cast<uint32_t>(piece / 4) * kPanel;
      const int out = piece % 4 * 2, swap = D == 128 ? piece / 4 : 0;
      const uint32_t my_piece = queue + static_cast<uint32_t>((warp * UNIT_ROWS + row_in) * c.row + (used_piece ? piece * 16 : 0));
      const uint32_t unit_step = static_cast<uint32_t>(Shape::kConverters * UNIT_ROWS * c.row);
      bool ok = true;
      int slot = 0, in = 0;
      uint32_t ph = 1, in_ph = 0;
      for (int u = 0; u < 2 * blocks; ++u) {
        const bool value = u & 1;
        ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&brought[in]), in_ph, abort_ptr, p.wait_ns));
        if (!ok) break;
        uint4 held[UNITS];
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
          held[i] = make_uint4(0u, 0u, 0u, 0u);
          if (warp + Shape::kConverters * i < Shape::kUnits && used_piece) held[i] = lds_16(my_piece + static_cast<uint32_t>(in) * Shape::kQueueTile + i * unit_step);
        }
        ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&empty[slot]), ph, abort_ptr, p.wait_ns));
        if (!ok) break;
        const uint32_t to_at = ring + static_cast<uint32_t>(slot) * kTile + panel;
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
          const int unit = warp + Shape::kConverters * i, r = unit * UNIT_ROWS + row_in;
          if (unit >= Shape::kUnits) break;
          const uint4 w = held[i];
          uint32_t h[8];
          if (HALF && !value) {
            int8_quad<__half>(w.x, h[0], h[1]);
            int8_quad<__half>(w.y, h[2], h[3]);
            int8_quad<__half>(w.z, h[4], h[5]);
            int8_quad<__half>(w.w, h[6], h[7]);
          } else {
            int8_quad<__nv_bfloat16>(w.x, h[0], h[1]);
            int8_quad<__nv_bfloat16>(w.y, h[2], h[3]);
            int8_quad<__nv_bfloat16>(w.z, h[4], h[5]);
            int8_quad<__nv_bfloat16>(w.w, h[6], h[7]);
          }
          const uint32_t at = to_at + static_cast<uint32_t>(r) * 128u;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int which = n ^ swap;
            const uint32_t x0 = which ? h[4] : h[0], x1 = which ? h[5] : h[1], x2 = which ? h[6] : h[2], x3 = which ? h[7] : h[3];
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + (((out + which) ^ (r & 7)) << 4)), "r"(x0), "r"(x1), "r"(x2), "r"(x3) : "memory");
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&full[slot]));
          mbar_arrive(smem_u32(&taken[in]));
          if (value) mbar_arrive(smem_u32(&steps_full[(u >> 1) % kSteps]));  // (keys' and values' steps, and which pages are there)
        }
        if (++slot == kSlots) {
          slot = 0;
          ph ^= 1u;
        }
        if (++in == Shape::kQueue) {
          in = 0;
          in_ph ^= 1u;
        }
      }
      if (!ok && lane == 0) gave_up();
    } else if (warp == 6) {
      // ---- blocks brought: lanes 0 to 7 sixteen keys' rows each, lanes 8 to 15 their steps
      const int table_row = a.prefix ? 0 : sequence;
      const long long page_rows = static_cast<long long>(c.kv_heads) << c.page_shift, head_rows = static_cast<long long>(kv_head) << c.page_shift;
      const int in_page = (1 << c.page_shift) - 1;
      const uint32_t rows_bytes = 16u * c.row;
      // eight pages to a block, four blocks to the lanes, looked up while the four blocks before are asked for
      auto look_up = [&](int j0) {
        const int key = from + j0 * 128 + lane * 16;
        return key < to ? cache_page(c, table_row, key) : -1;
      };
      int pages = -1, next_pages = look_up(0);
      int issued = 0, in = 0;
      uint32_t ph = 1;
      bool ok = p.stall == 0;
      for (int u = 0; ok && u < 2 * blocks; ++u) {
        const int j = u >> 1;
        const bool value = u & 1;
        if (!value && (j & 3) == 0) {
          pages = next_pages;
          next_pages = look_up(j + 4);
        }
        const int page = __shfl_sync(~0u, pages, (j & 3) * 8 + (lane & 7));
        const uint32_t there = __ballot_sync(~0u, page >= 0) & 0xffu;
        const long long line = page_rows * page + head_rows + ((from + j * 128 + (lane & 7) * 16) & in_page);
        ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&taken[in]), ph, abort_ptr, p.wait_ns));
        if (!ok) break;
        const uint32_t bar = smem_u32(&brought[in]);
        if (lane == 0) {
          if (!value) pages_there[j % kSteps] = static_cast<int>(there);
          mbar_arrive_expect_tx(bar, __popc(there) * (rows_bytes + 64u));
        }
        __syncwarp();
        if (page >= 0 && lane < 8) bulk_load(queue + static_cast<uint32_t>(in) * Shape::kQueueTile + lane * rows_bytes, (value ? c.v : c.k) + line * c.row, rows_bytes, bar);
        if (page >= 0 && lane >= 8 && lane < 16)
          bulk_load(steps_at + static_cast<uint32_t>(j % kSteps) * 1024u + (value ? 512u : 0u) + (lane & 7) * 64u, (value ? c.v_steps : c.k_steps) + line, 64u, bar);
        issued = u + 1;
        if (++in == Shape::kQueue) {
          in = 0;
          ph ^= 1u;
        }
      }
      if (!ok && p.stall == 0 && lane == 0) gave_up();
      // no copy may be under way when the CTA's shared memory is given back
      if (lane == 0) ring_landed(brought, Shape::kQueue, issued);
    } else if (blocks > 0) {
      // ---- MMAs
      if (elect_one()) {
        constexpr uint32_t kBMnMajor = 1u << 16;
        const uint32_t s_idesc = instr_desc(1, HALF ? 0u : 1u, 128, 64), pv_idesc = instr_desc(1, 1u, 128, D) | kBMnMajor;
        bool ok = mbar_wait_bounded(smem_u32(&q_full), 0, abort_ptr, p.wait_ns);
        // (a block's keys are use 2 j of the ring, its values use 2 j + 1)
        auto wait_use = [&](int slot, uint32_t ph) { return mbar_wait_bounded(smem_u32(&full[slot]), ph, abort_ptr, p.wait_ns); };
        auto scores = [&](int t, int slot, int h) {
          const uint32_t k_at = ring + static_cast<uint32_t>(slot) * kTile + h * 8192, a_at = q_at + t * kTile;
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {
            const uint32_t off = (n / 4) * kPanel + (n % 4) * 32;
            mma_f16(s_of(t) + 64u * h, smem_desc_kmajor(a_at + off, 128), smem_desc_kmajor(k_at + off, 128), s_idesc, n > 0);
          }
          tc_commit(smem_u32(&s_full[t][h]));
        };
        // four steps of 16 keys; the second terms lie 32 columns behind the first
        auto products = [&](int t, int slot, int h, bool first_ones) {
          const uint32_t v_at = ring + static_cast<uint32_t>(slot) * kTile + h * 8192;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint64_t v = smem_desc_mnmajor(v_at + i * 2048, kPanel, 1024);
            mma_f16_ts(o_of(t), s_of(t) + 64u * h + 8u * i, v, pv_idesc, !first_ones || i > 0);
            mma_f16_ts(o_of(t), s_of(t) + 64u * h + 32u + 8u * i, v, pv_idesc, 1u);
          }
          tc_commit(smem_u32(&o_done[t][h]));
        };
        ok = ok && wait_use(0, 0);
        if (ok) {
          tc_fence_after_sync();
          for (int h = 0; h < 2; ++h)
            for (int t = 0; t < tiles; ++t) scores(t, 0, h);
          tc_commit(smem_u32(&empty[0]));
        }
        int v_slot = 1;
        uint32_t v_ph = 0;
        for (int j = 0; ok && j < blocks; ++j) {
          const int k_slot = v_slot == kSlots - 1 ? 0 : v_slot + 1;
          const uint32_t k_ph = k_slot == 0 ? v_ph ^ 1u : v_ph;
          const bool more = j + 1 < blocks;
          ok = wait_use(v_slot, v_ph);
          for (int h = 0; ok && h < 2; ++h)
            for (int t = 0; t < tiles; ++t) {
              ok = mbar_wait_bounded(smem_u32(&p_full[t][h]), j & 1, abort_ptr, p.wait_ns);
              if (!ok) break;
              tc_fence_after_sync();
              products(t, v_slot, h, j == 0 && h == 0);
              if (h == 1 && t == tiles - 1) tc_commit(smem_u32(&empty[v_slot]));
              if (!more && h == 1) tc_commit(smem_u32(&o_full[t]));
              if (more) {
                if (h == 0 && t == 0) ok = wait_use(k_slot, k_ph);
                if (!ok) break;
                scores(t, k_slot, h);
                if (h == 1 && t == tiles - 1) tc_commit(smem_u32(&empty[k_slot]));
              }
            }
          v_slot = k_slot == kSlots - 1 ? 0 : k_slot + 1;
          v_ph = v_slot == 0 ? k_ph ^ 1u : k_ph;
        }
        if (!ok) gave_up();
        // MMAs under way are done before the CTA leaves, whoever gave up
        tc_commit(smem_u32(&drained));
        ring_landed(&drained, 1, 1);
      }
    }
  } else {
    // ---- softmaxes
    reg_alloc<Shape::kRegsSoftmax>();
    const int t = (warp - 8) >> 2;
    if (t < tiles) {
      const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // this warp's 32 lanes of tensor memory (lane in the upper half word)
      const uint32_t s_at = s_of(t) + lanes, o_at = o_of(t) + lanes;
      const int r = (warp & 3) * 32 + lane;  // row of the tile
      const long long row = row0 + t * 128 + r, token = first + row / G;
      const int head = kv_head * G + static_cast<int>(row % G);
      int position = -2;
      if (row < rows) {
        if (a.prefix) {
          const CachePlace place = cache_place(c, token);
          position = place.sequence < 0 ? -2 : place.position;
        } else {
          position = max(before + static_cast<int>(row / G), -1);
        }
      }
      const int least = __reduce_min_sync(~0u, position < -1 ? 0x7fffffff : position);
      // the row's query into the tile, as TMA would with a 128-byte swizzle
      const T* q = static_cast<const T*>(a.q) + token * a.q_token + head * a.q_head;
#pragma unroll 4
      for (int n = 0; n < D / 8; ++n) {
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (position > -2 && n * 8 < c.d) {
          if (p.q_wide) {
            w = __ldg(reinterpret_cast<const uint4*>(q + n * 8));
          } else {
            OpVec<T, 8> e{};
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (n * 8 + i < c.d) e.e[i] = q[n * 8 + i];
            w = *reinterpret_cast<const uint4*>(&e);
          }
        }
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(q_at + t * kTile + (n / 8) * kPanel + r * 128 + (((n & 7) ^ (r & 7)) << 4)), "r"(w.x), "r"(w.y),
                     "r"(w.z), "r"(w.w)
                     : "memory");
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&q_full));

      const float scale = a.scale_log2 * (HALF ? 1.0f : kBf16Integers);
      const uint64_t c2 = f32x2_make(__float_as_uint(scale), __float_as_uint(scale));
      float base = -INFINITY;  // of the exponentials: the maximum so far, or one up to 2^8 smaller
      float total = 0.0f;
      bool ok = true;
      // a half block: its 64 scores, and P in their place.  ALL: every row of the warp sees every key of it.
      auto half = [&](int j, int h, auto all, int there) {
        constexpr bool ALL = decltype(all)::value;
        const uint32_t steps = steps_at + static_cast<uint32_t>(j % kSteps) * 1024u + h * 256u, s_half = s_at + 64u * h;
        const int key0 = from + j * 128 + h * 64;
        uint32_t s[64];
        tmem_ld32(s_half, s);
        tmem_ld32(s_half + 32u, s + 32);
        tmem_ld_wait();
        float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        const int seen = min(position, to - 1) - key0;  // the last key of the half that the row sees
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          const uint4 k = lds_16(steps + i * 4);
          float2 x = f32x2_get(f32x2_mul(f32x2_make(s[i], s[i + 1]), f32x2_make(k.x, k.y)));
          float2 y = f32x2_get(f32x2_mul(f32x2_make(s[i + 2], s[i + 3]), f32x2_make(k.z, k.w)));
          if (!ALL) {
            const bool page = there >> (4 * h + i / 16) & 1;
            if (!page || i > seen) x.x = -INFINITY;
            if (!page || i + 1 > seen) x.y = -INFINITY;
            if (!page || i + 2 > seen) y.x = -INFINITY;
            if (!page || i + 3 > seen) y.y = -INFINITY;
          }
          s[i] = __float_as_uint(x.x);
          s[i + 1] = __float_as_uint(x.y);
          s[i + 2] = __float_as_uint(y.x);
          s[i + 3] = __float_as_uint(y.y);
          m[i / 4 & 3] = max3(m[i / 4 & 3], x.x, x.y);
          m[i / 4 & 3] = max3(m[i / 4 & 3], y.x, y.y);
        }
        const float top = max3(m[0], m[1], fmaxf(m[2], m[3])) * scale;
        const bool raise = top > base + 8.0f;  // (true for the first keys of a row: its base is -infinity)
        if (__any_sync(~0u, raise)) {
          const float next = raise ? top : base;
          const float keep = raise ? exp2_fast(base - next) : 1.0f;
          base = next;
          total *= keep;
          if (j > 0 || h > 0) {
            // the products of the half before this one are in O, and with them all others
            ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&o_done[t][h ^ 1]), (j + h + 1) & 1, abort_ptr, p.wait_ns));
            if (!ok) return;
            tc_fence_after_sync();
#pragma unroll
            for (int w = 0; w < D / 16; ++w) {
              uint32_t o[16];
              tmem_ld16(o_at + 16u * w, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
              tmem_st16(o_at + 16u * w, o);
            }
          }
        }
        const float zero = base == -INFINITY ? 0.0f : -base;
        const uint64_t from2 = f32x2_make(__float_as_uint(zero), __float_as_uint(zero));
        uint64_t sums[2] = {0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const int at = 16 * w + 2 * i;
            const uint4 v = lds_16(steps + 512u + at * 4);
            const uint32_t vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 x = f32x2_get(f32x2_fma3(f32x2_make(s[at + 2 * e], s[at + 2 * e + 1]), c2, from2));
              const uint64_t both = f32x2_make(__float_as_uint(exp2_fast(x.x)), __float_as_uint(exp2_fast(x.y)));
              f32x2_add(sums[e], sums[e], both);
              float2 y = f32x2_get(f32x2_mul(both, f32x2_make(vs[2 * e], vs[2 * e + 1])));
              if (!ALL) {  // (the step of a key that takes no part may be anything)
                if (s[at + 2 * e] == 0xff800000u) y.x = 0.0f;
                if (s[at + 2 * e + 1] == 0xff800000u) y.y = 0.0f;
              }
              hi[i + e] = pack2<__nv_bfloat16>(y.x, y.y);
              lo[i + e] = pack2<__nv_bfloat16>(y.x - __uint_as_float(hi[i + e] << 16), y.y - __uint_as_float(hi[i + e] & 0xffff0000u));
            }
          }
          tmem_st8(s_half + 8u * w, hi);
          tmem_st8(s_half + 32u + 8u * w, lo);
        }
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_full[t][h]));
        f32x2_add(sums[0], sums[0], sums[1]);
        const float2 sum = f32x2_get(sums[0]);
        total += sum.x + sum.y;
      };
      for (int j = 0; ok && j < blocks; ++j) {
        const int key0 = from + j * 128;
        ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&steps_full[j % kSteps]), (j / kSteps) & 1, abort_ptr, p.wait_ns));
        const int there = ok ? pages_there[j % kSteps] : 0;
        const bool whole = there == 0xff && key0 + 127 <= least && key0 + 127 < to;
        for (int h = 0; ok && h < 2; ++h) {
          // The products before these scores have ended, too; asked for so that no phase of their barrier is passed over: a parity
          // says only which of two neighbouring phases it is in.
          ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&s_full[t][h]), j & 1, abort_ptr, p.wait_ns) &&
                                   (j == 0 || mbar_wait_bounded(smem_u32(&o_done[t][h]), (j - 1) & 1, abort_ptr, p.wait_ns)));
          if (!ok) break;
          tc_fence_after_sync();
          if (whole) half(j, h, std::true_type{}, there);
          else half(j, h, std::false_type{}, there);
        }
      }
      if (ok && blocks > 0) {
        ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&o_full[t]), 0, abort_ptr, p.wait_ns));
        tc_fence_after_sync();
      }
      if (!ok) {
        if (lane == 0) gave_up();
      } else {
        const long long line = (a.first_range + range) * (c.tokens * a.heads) + token * a.heads + head;
        const float norm = a.part != nullptr ? kBf16Integers : total == 0.0f ? 0.0f : kBf16Integers / total;
        if (a.part != nullptr && position > -2) a.part_top[line] = make_float2(base, total);
        T* out = static_cast<T*>(a.o) + token * a.o_token + head * a.o_head;
#pragma unroll 1
        for (int w = 0; w < D / 16; ++w) {
          uint32_t o[16] = {};
          if (blocks > 0) {
            tmem_ld16(o_at + 16u * w, o);
            tmem_ld_wait();
          }
          if (position < -1 || 16 * w >= c.d) continue;
          if (a.part != nullptr) {
            float4* to_part = reinterpret_cast<float4*>(a.part + line * a.part_width + 16 * w);
#pragma unroll
            for (int i = 0; i < 4; ++i) to_part[i] = make_float4(__uint_as_float(o[4 * i]) * norm, __uint_as_float(o[4 * i + 1]) * norm, __uint_as_float(o[4 * i + 2]) * norm, __uint_as_float(o[4 * i + 3]) * norm);
          } else {
            OpVec<T, 4> y[4];
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i / 4].e[i % 4] = op_put<T>(total == 0.0f ? 0.0f : __uint_as_float(o[i]) * norm);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (a.o_wide) {
                if (16 * w + 4 * i < c.d) *reinterpret_cast<OpVec<T, 4>*>(out + 16 * w + 4 * i) = y[i];
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (16 * w + 4 * i + e < c.d) out[16 * w + 4 * i + e] = y[i].e[e];
              }
            }
          }
        }
      }
      tc_fence_before_sync();
    }
  }
  __syncthreads();
  if (warp == 7) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, Shape::kTmemCols);
  }
  grid_dependency_wait();
}

}  // namespace nb
