// Attention to at most 128 keys (the tokens of a text) on tensor cores: one block of scores, so no running maximum, and time goes
// into getting queries in and results out.
//
// One CTA to an SM walks a range of the call's tiles (128 queries of one head, heads in order); a head's keys and values stay in
// shared memory for its tiles, the next head's are loaded into the other half meanwhile, queries come through a ring.  The two
// groups of softmax warps take the tiles in turn: while one has its exponentials and its stores, the other's MMAs run, and the
// CTA's start (barriers, tensor memory, first loads: some 2 us) is paid once an SM instead of once for every two tiles.
// Measured (8 sequences of 4096 queries over 77 keys, 10 heads of 64, fp16): 28.6 us of device time, 3.0 TB/s; HBM would allow 13.  A tile takes
// a group some 4000 clocks, of which 1100 are exponentials and the rest the chain scores - maximum - products - results, of
// which the two groups hide half.
#pragma once

#include "tc_attend.cuh"

namespace nb {

template <int D>
struct TcShortShape {
  static constexpr int kPanel = kAttRows * 128;
  static constexpr int kTile = kPanel * (D / 64);
  static constexpr int kThreads = 384;
  static constexpr int kRegsLaunch = 168, kRegsControl = 56, kRegsSoftmax = 224;
  static constexpr int kQueries = D == 64 ? 6 : 3;  // tiles of the ring
  static constexpr int kSmem = 1024 + (4 + kQueries) * kTile;
};

struct TcShortParams {
  TcAttendParams t;
  int row_tiles;  // of a head
  int tiles;      // of the call
};

template <class T, int D>
__global__ void __launch_bounds__(TcShortShape<D>::kThreads, 1)
tc_attend_short_kernel(const __grid_constant__ TcShortParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o) {
  using namespace ptx;
  using Shape = TcShortShape<D>;
  constexpr int kTile = Shape::kTile, kPanel = Shape::kPanel, kQueries = Shape::kQueries;
  const AttendParams& a = p.t.a;
  extern __shared__ uint8_t attend_smem[];
  __shared__ __align__(8) uint64_t q_full[kQueries], q_empty[kQueries], kv_full[2], kv_empty[2], kv_fixed[2], s_full[2], p_full[2], o_full[2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int warp = __shfl_sync(~0u, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const uint32_t smem = (smem_u32(attend_smem) + 1023u) & ~1023u;
  const uint32_t kv_at = smem, q_at = smem + 4 * kTile;  // [half][keys, values], ring
  volatile int* abort_ptr = &abort_flag;
  const int first = static_cast<int>(static_cast<long long>(p.tiles) * blockIdx.x / gridDim.x);
  const int end = static_cast<int>(static_cast<long long>(p.tiles) * (blockIdx.x + 1) / gridDim.x);
  const int shared = a.heads / a.kv_heads;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kQueries; ++i) {
      mbar_init(smem_u32(&q_full[i]), 1);
      mbar_init(smem_u32(&q_empty[i]), 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&kv_full[i]), 1);
      mbar_init(smem_u32(&kv_empty[i]), 1);
      mbar_init(smem_u32(&kv_fixed[i]), 1);
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&p_full[i]), 4);
      mbar_init(smem_u32(&o_full[i]), 1);
    }
    mbar_init(smem_u32(&drained), 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(~0u, tmem_slot, 0);
  auto gave_up = [&] {
    if (atomicCAS(&abort_flag, 0, 1) == 0) atomicAdd(&g_attend_gave_up, 1u);
  };
  auto wait = [&](uint64_t& bar, int parity) { return mbar_wait_bounded(smem_u32(&bar), parity & 1, abort_ptr, p.t.wait_ns); };
  auto s_of = [&](int t) { return tmem + 128u * t; };
  auto o_of = [&](int t) { return tmem + 256u + static_cast<uint32_t>(D * t); };
  auto keys_of = [&](int b) { return a.lens == nullptr ? a.lk : min(max(__ldg(a.lens + b), 0), a.lk); };
  // The roles walk the same tiles.  `n` counts those of sequences with keys (others have no part in any barrier), `pair` the
  // (sequence, head) pairs with keys, whose keys and values take the halves in turn.
  auto walk = [&](auto&& f) {
    int n = 0, pair = -1;
    int at = first / p.row_tiles, row_tile = first - at * p.row_tiles, b = at / a.heads, h = at - b * a.heads;
    int keys = keys_of(b);
    bool fresh = true;
    for (int tile = first; tile < end; ++tile) {
      if (keys > 0 && fresh) ++pair;
      const bool ends = tile + 1 == end || row_tile + 1 == p.row_tiles;
      if (!f(row_tile, n, pair, b, h, keys, fresh, ends)) return false;
      if (keys > 0) ++n;
      fresh = false;
      if (++row_tile == p.row_tiles) {  // (no divisions: they took a sixth of a tile's time)
        row_tile = 0;
        fresh = true;
        if (++h == a.heads) {
          h = 0;
          if (tile + 1 < end) keys = keys_of(++b);
        }
      }
    }
    return true;
  };

  if (warp < 4) {
    reg_dealloc<Shape::kRegsControl>();
    if (warp == 0) {
      if (elect_one()) {
        int queries = 0, pairs = 0;
        const bool ok = walk([&](int row_tile, int n, int pair, int b, int h, int keys, bool fresh, bool) {
          if (keys == 0) return true;
          if (p.t.stall != 0) return true;
          if (fresh) {
            const int half = pair & 1;
            if (pair >= 2 && !wait(kv_empty[half], pair / 2 - 1)) return false;
            mbar_arrive_expect_tx(smem_u32(&kv_full[half]), 2 * kTile);
            const int kv = h / shared;
            for (int c = 0; c < D / 64; ++c) {
              const uint32_t to = kv_at + half * 2 * kTile + c * kPanel;
              tma_load_4d(to, &map_k, smem_u32(&kv_full[half]), c * 64, 0, kv * p.t.k_step[0], b * p.t.k_step[1]);
              tma_load_4d(to + kTile, &map_v, smem_u32(&kv_full[half]), c * 64, 0, kv * p.t.v_step[0], b * p.t.v_step[1]);
            }
            pairs = pair + 1;
          }
          const int slot = n % kQueries;
          if (n >= kQueries && !wait(q_empty[slot], n / kQueries - 1)) return false;
          mbar_arrive_expect_tx(smem_u32(&q_full[slot]), kTile);
          for (int c = 0; c < D / 64; ++c)
            tma_load_4d(q_at + slot * kTile + c * kPanel, &map_q, smem_u32(&q_full[slot]), c * 64, row_tile * kAttRows, h * p.t.q_step[0], b * p.t.q_step[1]);
          queries = n + 1;
          return true;
        });
        if (!ok) gave_up();
        // no copy may be under way when the CTA's shared memory is given back
        auto landed = [](uint32_t bar, int parity) {
          for (int tries = 0; tries < 1 << 20 && !mbar_try_wait(bar, parity & 1); ++tries) {
          }
        };
        for (int n = max(queries - kQueries, 0); n < queries; ++n) landed(smem_u32(&q_full[n % kQueries]), n / kQueries);
        for (int n = max(pairs - 2, 0); n < pairs; ++n) landed(smem_u32(&kv_full[n & 1]), n / 2);
      }
    } else if (warp == 1) {
      if (elect_one()) {
        constexpr uint32_t kFormat = std::is_same<T, __half>::value ? 0u : 1u;
        constexpr uint32_t kBMnMajor = 1u << 16;
        const uint32_t pv_idesc = instr_desc(1, kFormat, kAttRows, D) | kBMnMajor;
        // The products of a tile follow one tile behind its scores' turn: S(n) is issued before P(n - 1) V, so that both groups
        // of softmax warps have work.  `before`: the tile whose products are due.
        struct Due {
          int n = -1, half = 0, keys = 0, batch = 0;
          bool ends = false;
        } before;
        auto products = [&](const Due& d) {
          if (!wait(p_full[d.n & 1], d.n / 2)) return false;
          tc_fence_after_sync();
          const int steps = (d.keys + 15) >> 4;
          const uint32_t v_at = kv_at + d.half * 2 * kTile + kTile;
#pragma unroll
          for (int c = 0; c < 8; ++c)
            if (c < steps) mma_f16_ts(o_of(d.n & 1), s_of(d.n & 1) + 8u * c, smem_desc_mnmajor(v_at + c * 2048, kPanel, 1024), pv_idesc, c > 0);
          tc_commit(smem_u32(&o_full[d.n & 1]));
          if (d.ends) tc_commit(smem_u32(&kv_empty[d.half]));
          return true;
        };
        bool ok = walk([&](int, int n, int pair, int b, int, int keys, bool fresh, bool ends) {
          if (keys == 0) return true;
          const int half = pair & 1;
          if (fresh && (!wait(kv_full[half], pair / 2) || !wait(kv_fixed[half], pair / 2))) return false;
          if (!wait(q_full[n % kQueries], n / kQueries)) return false;
          tc_fence_after_sync();
          const uint32_t idesc = instr_desc(1, kFormat, kAttRows, (keys + 15) & ~15);
          const uint32_t k_at = kv_at + half * 2 * kTile, a_at = q_at + n % kQueries * kTile;
          // S(n) takes the place of P(n - 2), whose products were issued before it
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            const uint32_t off = (c / 4) * kPanel + (c % 4) * 32;
            mma_f16(s_of(n & 1), smem_desc_kmajor(a_at + off, 128), smem_desc_kmajor(k_at + off, 128), idesc, c > 0);
          }
          tc_commit(smem_u32(&s_full[n & 1]));
          if (before.n >= 0 && !products(before)) return false;
          before = Due{n, half, keys, b, ends};
          return true;
        });
        if (ok && before.n >= 0) ok = products(before);
        if (!ok) {
          gave_up();
          tc_commit(smem_u32(&drained));  // nor may MMAs be under way
          for (int tries = 0; tries < 1 << 20 && !mbar_try_wait(smem_u32(&drained), 0); ++tries) {
          }
        }
      }
    } else if (warp == 2) {
      // values that take no part are zeroed, up to the last step of the products
      const bool ok = walk([&](int, int, int pair, int b, int, int keys, bool fresh, bool) {
        if (keys == 0 || !fresh) return true;
        const int half = pair & 1;
        const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + static_cast<long long>(b) * a.lk;
        if (!__all_sync(~0u, wait(kv_full[half], pair / 2))) return false;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int r0 = 32 * w + lane;
          uint32_t bits = __ballot_sync(~0u, r0 < ((keys + 15) & ~15) && !(r0 < keys && (mask == nullptr || __ldg(mask + r0) != 0)));
          while (bits != 0) {
            const int r = 32 * w + __ffs(bits) - 1;
            bits &= bits - 1;
            for (int c = lane; c < D / 4; c += 32) {
              const uint32_t to = kv_at + half * 2 * kTile + kTile + (c / 16) * kPanel + r * 128 + (c % 16) * 8;
              asm volatile("st.shared.v2.b32 [%0], {%1, %1};" ::"r"(to), "r"(0u) : "memory");
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&kv_fixed[half]));
        return true;
      });
      if (!ok && lane == 0) gave_up();
    }
  } else {
    reg_alloc<Shape::kRegsSoftmax>();
    const int group = (warp - 4) >> 2;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
    const float c = p.t.scale_log2;
    const uint32_t s_at = s_of(group) + lanes, o_at = o_of(group) + lanes;
    // a tile's results leave through its queries' place in the ring, which is free once they have been read
    int leaving = -1;
    auto left = [&] {
      if (lane == 0 && leaving >= 0) {
        bulk_wait_read();
        mbar_arrive(smem_u32(&q_empty[leaving]));
      }
      leaving = -1;
    };
    const bool ok = walk([&](int row_tile, int n, int, int b, int h, int keys, bool, bool) {
      // tiles without keys go to the groups in turn, too
      if ((keys > 0 ? n & 1 : row_tile & 1) != group) return true;
      const int row0 = row_tile * kAttRows;
      if (keys == 0) {
        const int row = row0 + (warp & 3) * 32 + lane;
        if (row < a.lq)
          for (int i = 0; i < a.d; i += 8)
            *reinterpret_cast<uint4*>(static_cast<T*>(a.o) + b * a.o_batch + row * a.o_row + h * a.o_head + i) = make_uint4(0u, 0u, 0u, 0u);
        return true;
      }
      float total = 0.0f;
      {
        const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + static_cast<long long>(b) * a.lk;
        uint32_t part[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int r = 32 * w + lane;
          part[w] = mask == nullptr ? (keys >= 32 * (w + 1) ? ~0u : keys <= 32 * w ? 0u : (1u << (keys - 32 * w)) - 1u)
                                    : __ballot_sync(~0u, r < keys && __ldg(mask + r) != 0);
        }
        if (!__all_sync(~0u, wait(s_full[group], n / 2))) return false;
        tc_fence_after_sync();
        left();
        const int chunks = (keys + 15) >> 4;  // of 16 keys
        uint32_t s[128];
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (2 * w < chunks) tmem_ld32(s_at + 32u * w, s + 32 * w);
        tmem_ld_wait();
        float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int w = 0; w < 8; ++w)
          if (w < chunks) {
            const uint32_t bits = part[w / 2] >> (16 * (w & 1)) & 0xffffu;
            if (bits != 0xffffu) {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (!(bits >> i & 1u)) s[16 * w + i] = 0xff800000u;  // -infinity
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) m[i & 3] = fmaxf(m[i & 3], __uint_as_float(s[16 * w + i]));
          }
        const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * c;
        const float from = top == -INFINITY ? 0.0f : -top;
        const uint64_t c2 = f32x2_make(__float_as_uint(c), __float_as_uint(c)), from2 = f32x2_make(__float_as_uint(from), __float_as_uint(from));
        uint64_t sums[2] = {0, 0};
#pragma unroll
        for (int w = 0; w < 8; ++w)
          if (w < chunks) {
            uint32_t packed[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) packed[i] = exp_pair<T>(s[16 * w + 2 * i], s[16 * w + 2 * i + 1], c2, from2, sums[i & 1]);
            tmem_st8(s_at + 8u * w, packed);
          }
        f32x2_add(sums[0], sums[0], sums[1]);
        const float2 sum = f32x2_get(sums[0]);
        total = sum.x + sum.y;
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_full[group]));
        if (!__all_sync(~0u, wait(o_full[group], n / 2))) return false;
        tc_fence_after_sync();
      }
      const int slot = n % kQueries;
      attend_store<T, D>(o_at, true, total, q_at + slot * kTile, (warp & 3) * 32, &map_o, row0, a.lq, h, b, a.d);
      leaving = slot;
      tc_fence_before_sync();  // (the next tile's products take O's place once this group has said that its P is there)
      return true;
    });
    left();
    if (!ok && lane == 0) gave_up();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace nb
