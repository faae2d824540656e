// Attention of many queries on tensor cores, 16-bit types: tcgen05 MMAs over TMA tiles, softmax in registers.
//
// A CTA holds TILES tiles of 128 queries of one head and walks the keys in blocks of 128 with a running maximum and sum:
//   S = Q K^T        tcgen05.mma, both operands in shared memory, 128 x 128 fp32 in tensor memory
//   P = 2^(S c - m)  c = scale / ln 2; a thread owns a query's row: it loads the 128 scores, takes their maximum, and writes P,
//                    rounded to the type, over S (64 columns of packed pairs); fp16 times 2^7 (kProbabilityLift)
//   O += P V         tcgen05.mma with P out of tensor memory; V as TMA brings it is [key][component], the keys being the
//                    contraction: the descriptor's MN-major form
// O is divided by the sum of the unrounded P at the end.  When a row's maximum rises, O has to be scaled; up to 2^8 the old
// maximum is kept as the base instead (P and the sum grow by that factor, nothing is lost in floating point), so that O is
// touched a few times a row at most.  The MMAs of a tile run in order in one thread: scores of block j + 1 being complete
// means that the products of block j are in O.
//
// Roles: warp 0 issues the TMA loads (keys and values take turns in one ring), warp 1 the MMAs, warp 2 clears values that take
// no part; warps 4 to 7 are tile 0's softmax, warps 8 to 11 tile 1's.  While one tile's scores are in its softmax, the other
// tile's MMAs run: 512 clocks of MMAs a product of 128 x 128 x 128 against 1024 clocks of exponentials (16 a clock and SM).
// Keys that take no part have P = 0 exactly, but 0 times a NaN or an infinity is a NaN: their values are zeroed in shared
// memory before the product (the last block's up to the next multiple of 16, others only under a mask).
#pragma once

#include "op_attention.h"
#include "ptx_sm100.cuh"
#include "tc_gemm_common.cuh"

namespace nb {

__device__ unsigned g_attend_gave_up;  // CTAs in which a wait ran out, ever: ncnn_b200_op_check_status

constexpr int kAttRows = 128;  // queries of a tile, and keys of a block

struct TcAttendParams {
  AttendParams a;
  float scale_log2;
  int slots;             // ring of key and value blocks
  int q_step[2], k_step[2], v_step[2];  // 0 where all heads (0) or sequences (1) read the same keys
  int stall;             // tests of the time-out path: the first block of keys is never loaded
  unsigned long long wait_ns;
};

template <int D, int TILES>
struct TcAttendShape {
  static constexpr int kPanel = kAttRows * 128;  // 128 rows of 64 components
  static constexpr int kTile = kPanel * (D / 64);
  static constexpr int kThreads = 128 + 128 * TILES;
  static constexpr int kBlocksPerSm = TILES == 2 || D > 128 ? 1 : 2;
  static constexpr uint32_t kTmemCols = TILES == 2 || D > 128 ? 512 : 256;
  static_assert(TILES * (128 + D) <= static_cast<int>(kTmemCols), "scores and results in tensor memory");
  // 256 threads alone on an SM have 255 registers each anyway; otherwise the roles share what the CTA was launched with
  static constexpr bool kShareRegs = D <= 128;
  static constexpr int kRegsLaunch = 65536 / (kThreads * kBlocksPerSm) / 8 * 8;
  static constexpr int kRegsControl = TILES == 2 ? 56 : 40;
  static constexpr int kRegsSoftmax = TILES == 2 ? 224 : 216;
  static_assert(!kShareRegs || 128 * kRegsControl + 128 * TILES * kRegsSoftmax <= kThreads * kRegsLaunch, "registers of the roles");
  static constexpr int kSlots = D > 128 ? 2 : D == 128 ? (TILES == 2 ? 4 : 2) : (TILES == 2 ? 6 : 4);
  static_assert(kSlots % 2 == 0, "values always land in the same slots: `fixed` counts their phases");
  static constexpr int kSmem = 1024 + TILES * kTile + kSlots * kTile;
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
        "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
        "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
      "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
      "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
      : "memory");
}

// D[tmem] (+)= A[tmem, packed pairs] * B[smem]
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <class T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(taddr)
               : "memory");
}

// 2^(x c + from) and 2^(y c + from) packed, and added to a pair of sums: two values to an instruction where there is one
template <class T>
__device__ __forceinline__ uint32_t exp_pair(uint32_t x, uint32_t y, uint64_t c2, uint64_t from2, uint64_t& sums) {
  const float2 t = f32x2_get(f32x2_fma3(f32x2_make(x, y), c2, from2));
  const float e0 = exp2_fast(t.x), e1 = exp2_fast(t.y);
  f32x2_add(sums, sums, f32x2_make(__float_as_uint(e0), __float_as_uint(e1)));
  return pack2<T>(e0, e1);
}

// The same on the FMA pipe, for every eighth pair: the 16 exponentials a clock and SM take as long as the MMAs (4096 queries over
// 4500 keys, 16 heads of 128: 209 us, 215 without, 208 with every fourth pair, 234 with every second).
// 2^x = 2^n 2^f with n the nearest whole number (out of the sum with 1.5 2^23, whose last bits it is) and f in [-1/2, 1/2];
// 2^f by a polynomial through the Chebyshev points of that range, of relative error: degree 3 is good to 2^-13.3, an
// eighteenth of bf16's half step, degree 4 to 2^-18.  x is held to -127, where the exponent's bits are 0 and the term is exactly 0,
// as ex2 has it for a term below 2^-126: keys of score minus infinity add nothing, and a row of them has the sum 0.  A NaN stays one.
template <class T>
__device__ __forceinline__ uint32_t exp_pair_fma(uint32_t x, uint32_t y, uint64_t c2, uint64_t from2, uint64_t& sums) {
  auto both = [](float v) { return f32x2_make(__float_as_uint(v), __float_as_uint(v)); };
  float2 t = f32x2_get(f32x2_fma3(f32x2_make(x, y), c2, from2));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(t.x) : "f"(-127.0f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(t.y) : "f"(-127.0f));
  const uint64_t at = f32x2_make(__float_as_uint(t.x), __float_as_uint(t.y));
  uint64_t whole, n;
  f32x2_add(whole, at, both(12582912.0f));
  f32x2_add(n, whole, both(-12582912.0f));
  const uint64_t f = f32x2_fma3(n, both(-1.0f), at);
  uint64_t p;
  if constexpr (std::is_same<T, __half>::value) {
    p = f32x2_fma3(both(0.00966636836528778f), f, both(0.055921975523233414f));
    p = f32x2_fma3(p, f, both(0.2402234971523285f));
    p = f32x2_fma3(p, f, both(0.6931210160255432f));
    p = f32x2_fma3(p, f, both(1.0f));
  } else {
    p = f32x2_fma3(both(0.05583828315138817f), f, both(0.2426394820213318f));
    p = f32x2_fma3(p, f, both(0.6931367516517639f));
    p = f32x2_fma3(p, f, both(0.9999245405197144f));
  }
  const float2 w = f32x2_get(whole);
  const uint64_t power = f32x2_make((__float_as_uint(w.x) << 23) + 0x3f800000u, (__float_as_uint(w.y) << 23) + 0x3f800000u);
  uint64_t e;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(e) : "l"(p), "l"(power));
  f32x2_add(sums, sums, e);
  const float2 r = f32x2_get(e);
  return pack2<T>(r.x, r.y);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A warp's 32 rows of results, scaled, out of tensor memory into a tile of shared memory (panels of 64 components, 128-byte
// swizzle) and from there to global memory in whole lines (4096 queries over 77 keys: 36 us against 40 with 16-byte stores by
// rows).  `staged`: the tile; `warp_row`: the warp's first row in it.
template <class T, int D>
__device__ __forceinline__ void attend_store(uint32_t o_at, bool any, float total, uint32_t staged, int warp_row, const CUtensorMap* map, int row, int rows,
                                             int h, int b, int d) {
  using namespace ptx;
  const int lane = threadIdx.x & 31, r = warp_row + lane;
  const float scale = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    uint32_t o[32];
    if (any) {
      tmem_ld32(o_at + 32u * w, o);
      tmem_ld_wait();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        u[e] = total == 0.0f ? 0u : pack2<T>(__uint_as_float(o[8 * i + 2 * e]) * scale, __uint_as_float(o[8 * i + 2 * e + 1]) * scale);
      const uint32_t to = staged + (w / 2) * (kAttRows * 128) + r * 128 + (((w % 2 * 4 + i) ^ (r & 7)) << 4);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]) : "memory");
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0 && row + warp_row < rows) {
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      if (64 * c < d) tma_store_4d(map, staged + c * (kAttRows * 128) + warp_row * 128, 64 * c, row + warp_row, h, b);
    bulk_commit();
  }
}

template <class T, int D, int TILES>
__global__ void __launch_bounds__(TcAttendShape<D, TILES>::kThreads, TcAttendShape<D, TILES>::kBlocksPerSm)
tc_attend_kernel(const __grid_constant__ TcAttendParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o) {
  using namespace ptx;
  using Shape = TcAttendShape<D, TILES>;
  constexpr int kTile = Shape::kTile, kPanel = Shape::kPanel, kSlots = Shape::kSlots;
  extern __shared__ uint8_t attend_smem[];
  __shared__ __align__(8) uint64_t q_full, full[kSlots], empty[kSlots], fixed[kSlots], s_full[TILES], p_half[TILES], p_full[TILES], o_full[TILES], drained, to_fix;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, walked;  // walked: blocks of keys that the MMAs have begun with, in sixteens

  const int warp = __shfl_sync(~0u, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int head = blockIdx.y, batch = blockIdx.z;
  const int kv_head = head / (p.a.heads / p.a.kv_heads);
  const int row0 = blockIdx.x * (kAttRows * TILES);
  const int tiles = TILES == 2 && row0 + kAttRows < p.a.lq ? 2 : 1;
  const int keys = p.a.lens == nullptr ? p.a.lk : min(max(__ldg(p.a.lens + batch), 0), p.a.lk);
  const int blocks = (keys + kAttRows - 1) / kAttRows;
  const uint8_t* mask = p.a.mask == nullptr ? nullptr : p.a.mask + static_cast<long long>(batch) * p.a.lk;
  // values to clear: those of masked keys in any block, and those behind the sequence's end that the last block's product reads
  const bool fix_all = mask != nullptr;
  const bool fix_last = keys < p.a.lk && (keys & 15) != 0;
  const uint32_t smem = (smem_u32(attend_smem) + 1023u) & ~1023u;
  const uint32_t q_at = smem, ring = smem + TILES * kTile;
  volatile int* abort_ptr = &abort_flag;
  volatile int* walked_ptr = &walked;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    walked = 0;
    mbar_init(smem_u32(&q_full), 1);
    mbar_init(smem_u32(&drained), 1);
    mbar_init(smem_u32(&to_fix), 1);
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), 1);
      mbar_init(smem_u32(&fixed[i]), 1);
    }
    for (int t = 0; t < TILES; ++t) {
      mbar_init(smem_u32(&s_full[t]), 1);
      mbar_init(smem_u32(&p_half[t]), 4);
      mbar_init(smem_u32(&p_full[t]), 4);
      mbar_init(smem_u32(&o_full[t]), 1);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), Shape::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(~0u, tmem_slot, 0);
  auto gave_up = [&] {
    if (atomicCAS(&abort_flag, 0, 1) == 0) atomicAdd(&g_attend_gave_up, 1u);
  };
  auto s_of = [&](int t) { return tmem + 128u * t; };
  auto o_of = [&](int t) { return tmem + 128u * TILES + static_cast<uint32_t>(D * t); };

  if (warp < 4) {
    if constexpr (Shape::kShareRegs) reg_dealloc<Shape::kRegsControl>();
    if (warp == 0 && blocks > 0) {
      if (elect_one()) {
        bool ok = true;
        uint32_t used = 0;  // loads of the ring so far
        mbar_arrive_expect_tx(smem_u32(&q_full), static_cast<uint32_t>(tiles * kTile));
        for (int t = 0; t < tiles; ++t)
          for (int c = 0; c < D / 64; ++c)
            tma_load_4d(q_at + t * kTile + c * kPanel, &map_q, smem_u32(&q_full), c * 64, row0 + t * kAttRows, head * p.q_step[0], batch * p.q_step[1]);
        for (int j = 0; j < 2 * blocks; ++j) {
          const int slot = j % kSlots;
          if (j >= kSlots && !mbar_wait_bounded(smem_u32(&empty[slot]), (j / kSlots - 1) & 1, abort_ptr, p.wait_ns)) {
            ok = false;
            break;
          }
          if (p.stall != 0) break;
          const bool value = j & 1;
          const uint32_t bar = smem_u32(&full[slot]), to = ring + slot * kTile;
          const int h = kv_head * (value ? p.v_step[0] : p.k_step[0]), b = batch * (value ? p.v_step[1] : p.k_step[1]);
          mbar_arrive_expect_tx(bar, kTile);
          for (int c = 0; c < D / 64; ++c) tma_load_4d(to + c * kPanel, value ? &map_v : &map_k, bar, c * 64, (j >> 1) * kAttRows, h, b);
          used = j + 1;
        }
        if (!ok) gave_up();
        // no copy may be under way when the CTA's shared memory is given back
        auto landed = [](uint32_t bar, uint32_t parity) {
          for (int tries = 0; tries < 1 << 20 && !mbar_try_wait(bar, parity); ++tries) {
          }
        };
        landed(smem_u32(&q_full), 0);
        for (uint32_t j = used > kSlots ? used - kSlots : 0; j < used; ++j) landed(smem_u32(&full[j % kSlots]), (j / kSlots) & 1);
      }
    } else if (warp == 1 && blocks > 0) {
      if (elect_one()) {
        constexpr uint32_t kFormat = std::is_same<T, __half>::value ? 0u : 1u;
        constexpr uint32_t kBMnMajor = 1u << 16;
        const uint32_t pv_idesc = instr_desc(1, kFormat, kAttRows, D) | kBMnMajor;
        bool ok = mbar_wait_bounded(smem_u32(&q_full), 0, abort_ptr, p.wait_ns);
        auto scores = [&](int t, int j) {
          const int n = min(kAttRows, (keys - j * kAttRows + 15) & ~15);
          const uint32_t idesc = instr_desc(1, kFormat, kAttRows, n);
          const uint32_t k_at = ring + (2 * j) % kSlots * kTile, a_at = q_at + t * kTile;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            const uint32_t off = (c / 4) * kPanel + (c % 4) * 32;
            mma_f16(s_of(t), smem_desc_kmajor(a_at + off, 128), smem_desc_kmajor(k_at + off, 128), idesc, c > 0);
          }
        };
        auto products = [&](int t, int j, int from) {  // four steps of 16 keys
          const int steps = min(from + 4, (keys - j * kAttRows + 15) >> 4);
          const uint32_t v_at = ring + (2 * j + 1) % kSlots * kTile;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = from + i;
            if (c < steps) mma_f16_ts(o_of(t), s_of(t) + 8u * c, smem_desc_mnmajor(v_at + c * 2048, kPanel, 1024), pv_idesc, j > 0 || c > 0);
          }
        };
        auto wait_slot = [&](int at) { return mbar_wait_bounded(smem_u32(&full[at % kSlots]), (at / kSlots) & 1, abort_ptr, p.wait_ns); };
        ok = ok && wait_slot(0);
        if (ok) {
          tc_fence_after_sync();
          for (int t = 0; t < tiles; ++t) {
            scores(t, 0);
            tc_commit(smem_u32(&s_full[t]));
          }
          tc_commit(smem_u32(&empty[0]));
        }
        for (int j = 0; ok && j < blocks; ++j) {
          const int v_use = 2 * j + 1, k_next = 2 * j + 2;
          for (int t = 0; t < tiles; ++t) {
            if (t == 0) {
              ok = wait_slot(v_use);
              const bool last = !fix_all && fix_last && j == blocks - 1;
              if ((j & 15) == 0) *walked_ptr = j + 1;  // (every block: 0.5 % of 4096 queries over 4500 keys)
              if (ok && last) mbar_arrive(smem_u32(&to_fix));
              if (ok && (fix_all || last))
                ok = mbar_wait_bounded(smem_u32(&fixed[v_use % kSlots]), fix_all ? (v_use / kSlots) & 1 : 0, abort_ptr, p.wait_ns);
            }
            ok = ok && mbar_wait_bounded(smem_u32(&p_half[t]), j & 1, abort_ptr, p.wait_ns);
            if (!ok) break;
            tc_fence_after_sync();
            products(t, j, 0);
            ok = mbar_wait_bounded(smem_u32(&p_full[t]), j & 1, abort_ptr, p.wait_ns);
            if (!ok) break;
            tc_fence_after_sync();
            products(t, j, 4);
            if (t == tiles - 1) tc_commit(smem_u32(&empty[v_use % kSlots]));
            if (j + 1 < blocks) {
              if (t == 0) ok = wait_slot(k_next);
              if (!ok) break;
              scores(t, j + 1);
              tc_commit(smem_u32(&s_full[t]));
              if (t == tiles - 1) tc_commit(smem_u32(&empty[k_next % kSlots]));
            } else {
              tc_commit(smem_u32(&o_full[t]));
            }
          }
        }
        if (!ok) {
          gave_up();
          tc_commit(smem_u32(&drained));  // nor may MMAs be under way
          for (int tries = 0; tries < 1 << 20 && !mbar_try_wait(smem_u32(&drained), 0); ++tries) {
          }
        }
      }
    } else if (warp == 2 && blocks > 0 && (fix_all || fix_last)) {
      bool ok = true;
      for (int j = fix_all ? 0 : blocks - 1; ok && j < blocks; ++j) {
        const int use = 2 * j + 1, slot = use % kSlots;
        const int left = keys - j * kAttRows, rows = min(kAttRows, (left + 15) & ~15);
        uint32_t clear[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int r = 32 * w + lane;
          const bool part = r < left && (mask == nullptr || __ldg(mask + j * kAttRows + r) != 0);
          clear[w] = __ballot_sync(~0u, !part && r < rows);
        }
        // Under a mask the MMAs wait for this warp in every block, so that it sees every phase of the ring's barriers.  Without
        // one the ring runs ahead of it, and the issuing thread says when the last block has landed.  That is a wait for the whole
        // walk over the keys, whose time has no bound: its limit begins anew as long as the walk gets on.
        auto last_landed = [&] {
          while (true) {
            const int seen = *walked_ptr;
            if (mbar_wait_bounded(smem_u32(&to_fix), 0, abort_ptr, p.wait_ns)) return true;
            if (*abort_ptr != 0 || *walked_ptr == seen) return false;
          }
        };
        ok = __all_sync(~0u, fix_all ? mbar_wait_bounded(smem_u32(&full[slot]), (use / kSlots) & 1, abort_ptr, p.wait_ns) : last_landed());
        if (!ok) break;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t bits = clear[w];
          while (bits != 0) {
            const int r = 32 * w + __ffs(bits) - 1;
            bits &= bits - 1;
            // a row's 128 bytes of each panel (the swizzle moves 16-byte pieces inside them)
            for (int c = lane; c < D / 4; c += 32) {
              const uint32_t at = ring + slot * kTile + (c / 16) * kPanel + r * 128 + (c % 16) * 8;
              asm volatile("st.shared.v2.b32 [%0], {%1, %1};" ::"r"(at), "r"(0u) : "memory");
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&fixed[slot]));
      }
      if (!ok && lane == 0) gave_up();
    }
  } else {
    if constexpr (Shape::kShareRegs) reg_alloc<Shape::kRegsSoftmax>();
    const int t = (warp - 4) >> 2;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // this warp's 32 lanes of tensor memory (lane in the upper half word)
    if (t < tiles) {
      const uint32_t s_at = s_of(t) + lanes, o_at = o_of(t) + lanes;
      const float c = p.scale_log2;
      float base = -INFINITY;  // of the exponentials: the maximum so far, or one up to 2^8 smaller
      float total = 0.0f;
      bool ok = true;
      for (int j = 0; j < blocks; ++j) {
        const int left = keys - j * kAttRows;
        uint32_t part[4] = {~0u, ~0u, ~0u, ~0u};
        const bool whole = mask == nullptr && left >= kAttRows;
        if (!whole) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int r = 32 * w + lane;
            part[w] = __ballot_sync(~0u, r < left && (mask == nullptr || __ldg(mask + j * kAttRows + r) != 0));
          }
        }
        ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&s_full[t]), j & 1, abort_ptr, p.wait_ns));
        if (!ok) break;
        tc_fence_after_sync();
        uint32_t s[128];
#pragma unroll
        for (int w = 0; w < 4; ++w) tmem_ld32(s_at + 32u * w, s + 32 * w);
        tmem_ld_wait();
        if (!whole) {
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(part[w] >> i & 1u)) s[32 * w + i] = 0xff800000u;  // -infinity
        }
        float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 2) m[i / 2 & 3] = max3(m[i / 2 & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        const float top = max3(m[0], m[1], fmaxf(m[2], m[3])) * c;
        const bool raise = top > base + 8.0f;  // (true for the first keys of a row: its base is -infinity)
        if (__any_sync(~0u, raise)) {
          const float next = raise ? top : base;
          const float keep = raise ? exp2_fast(base - next) : 1.0f;
          base = next;
          total *= keep;
          if (j > 0) {
#pragma unroll
            for (int w = 0; w < D / 32; ++w) {
              uint32_t o[32];
              tmem_ld32(o_at + 32u * w, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
              tmem_st32(o_at + 32u * w, o);
            }
          }
        }
        const float from = base == -INFINITY ? 0.0f : kProbabilityLift<T> - base;
        const uint64_t c2 = f32x2_make(__float_as_uint(c), __float_as_uint(c)), from2 = f32x2_make(__float_as_uint(from), __float_as_uint(from));
        uint64_t sums[2] = {0, 0};
        // P leaves in halves: the first one's products begin while the second one's exponentials are taken
        auto half = [&](int h, auto fma) {
#pragma unroll
          for (int w = 2 * h; w < 2 * h + 2; ++w) {
            uint32_t packed[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
              packed[i] = decltype(fma)::value && i % 8 == 7 ? exp_pair_fma<T>(s[32 * w + 2 * i], s[32 * w + 2 * i + 1], c2, from2, sums[i & 1])
                                               : exp_pair<T>(s[32 * w + 2 * i], s[32 * w + 2 * i + 1], c2, from2, sums[i & 1]);
            tmem_st16(s_at + 16u * w, packed);
          }
          tmem_st_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(h == 0 ? &p_half[t] : &p_full[t]));
        };
        if (whole) {
          half(0, std::true_type{});
          half(1, std::true_type{});
        } else {
          half(0, std::false_type{});
          half(1, std::false_type{});
        }
        f32x2_add(sums[0], sums[0], sums[1]);
        const float2 sum = f32x2_get(sums[0]);
        total += sum.x + sum.y;
      }
      if (ok && blocks > 0) {
        ok = __all_sync(~0u, mbar_wait_bounded(smem_u32(&o_full[t]), 0, abort_ptr, p.wait_ns));
        tc_fence_after_sync();
      }
      if (!ok) {
        if (lane == 0) gave_up();
      } else {
        // (every product is done: the queries' tile is free)
        attend_store<T, D>(o_at, blocks > 0, total, q_at + t * kTile, (warp & 3) * 32, &map_o, row0 + t * kAttRows, p.a.lq, head, batch, p.a.d);
        if (lane == 0) bulk_wait_read();
      }
      tc_fence_before_sync();
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, Shape::kTmemCols);
  }
}

}  // namespace nb
