// Attention over a paged cache of 8-bit integers for few rows: a pass over the pages at HBM speed.
//
// A CTA has a tile of 8, 16 or 32 rows that read one key head (a row is a token and one of the head's query heads) and a range of keys;
// its warps take blocks of 16 keys in turn, each with a running maximum, sum and result.  The products are mma.sync m16n8k16 with the
// keys, and then the values' components, as the 16 and the rows as the 8: a decoding step has 4 to 8 rows, and the other way half of
// every instruction would be for rows that are not there.  HBM is the bound, not the tensor cores; tcgen05 would want 128 rows.
//
// Integers are exact in either 16-bit type (|q| is at most 127), so the steps stay out of the products: a key's multiplies its scores,
// a value's its probabilities.  No integer is exchanged between lanes.  The contraction's order is free: a lane takes 16 neighbouring
// bytes of "its" two keys as the operands of four products, and the queries are permuted to match; for values it takes the same
// components of four keys and picks one byte of each.  So a lane copies (cp.async) only what it reads itself, into a queue
// of its own in shared memory: no barriers, and every access of shared memory takes neighbouring 16 bytes for neighbouring lanes.
// Scores come out as [key][row] and probabilities go in as [row][key]: movmatrix turns them.
//
// Roundings: scores of 16-bit queries are exact products (f32 queries: three bf16 terms, 24 bits); probabilities times steps are
// split into two bf16 terms (16 bits), f32 three.
//
// 64 sequences of up to 8192 keys, 32 heads on 8 of 128: 139 us, 4.0 TB/s ragged; 223 us, 5.0 TB/s of one length (16 warps an SM, half of
// the issue slots: latency of the chain copy - scores - probabilities - products).
//
// The ranges' results go to the caller's workspace with their maximum (of scores in powers of two) and sum, and k_attend_cache_join
// puts them together in the order of the keys; one range alone writes its result itself.
#pragma once

#include "attend_few.cuh"
#include "ptx_sm100.cuh"
#include "op_cache.h"

namespace nb {

struct AttendCacheParams {
  CacheParams c;
  const void* q;
  void* o;
  long long q_token, q_head, o_token, o_head;
  int heads, rows_a_head;  // query heads; those of one key head
  float scale_log2;
  int shared;              // keys 0..shared-1 are the first table row's for all sequences
  int prefix;              // 1: this launch is about those keys, its rows are all tokens'
  int chunk;               // keys of a range
  int first_range;         // number of this launch's first range
  int prefix_ranges, prefix_chunk, own_ranges, own_chunk;  // for joining
  float* part;             // [range][token][head][part_width], or null: one range, results go to o
  float2* part_top;        // [range][token][head]: maximum, sum
  int part_width;
  int o_wide;              // four components of o can be stored at a time
};

// Integers as 16-bit floating point.  bf16 whose upper byte is 0 are u 2^-133 for every lower byte u: 0 to 127 as subnormal numbers, 128
// to 255 with the smallest exponent.  So a byte q + 128 becomes q / 64 in one fma, (q + 128) 2^-133 2^127 - 2, exactly; the 64 is made good
// for in the factor of the scores and in the results.  (Two masks, a permutation and a subtraction to a pair: 423 us where this takes 397,
// pieces of prompts in tiles of 128 rows.)
constexpr float kBf16Integers = 64.0f;
__device__ __forceinline__ uint32_t biased_pair(uint32_t x) {  // q + 128 in bytes 0 and 2, zeros in 1 and 3
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0x7f007f00u), "r"(0xc000c000u));
  return r;
}
// integers in bytes 0 and 2, anything in 1 and 3
__device__ __forceinline__ uint32_t bf16_pair(uint32_t x) {
  uint32_t u;
  asm("lop3.b32 %0, %1, 0x00ff00ff, 0x00800080, 0x6a;" : "=r"(u) : "r"(x));  // (x & mask) ^ bias
  return biased_pair(u);
}
// four integers as two pairs of T (the first in the lower half): fp16's as they are, bf16's over 64
template <class T>
__device__ __forceinline__ void int8_quad(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  if constexpr (std::is_same<T, __half>::value) {
    // 1024 + (q + 128), less 1152
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
  } else {
    lo = biased_pair(__byte_perm(u, 0u, 0x4140));
    hi = biased_pair(__byte_perm(u, 0u, 0x4342));
  }
}

__device__ __forceinline__ void queue_16(uint32_t to, const void* from, bool take) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void queue_8(uint32_t to, const void* from, bool take) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(take ? 8 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds_16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds_8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ uint32_t turn_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// NT: eights of rows
template <class T, int D, int NT, int WARPS, int STAGES>
struct CacheFewShared {
  static constexpr int kRows = 8 * NT;
  static constexpr int kQTerms = sizeof(T) == 4 ? 3 : 1;
  static constexpr int kValueBytes = D / 8;                    // of a key that a lane takes
  static constexpr int kKeyBytes = 2 * (D / 64) * 512;         // of a block, a warp
  static constexpr int kValues = 4 * kValueBytes * 32;
  static constexpr int kStage = kKeyBytes + kValues + 2 * 256;  // and the steps
  uint2 q[kQTerms][D / 16][NT][32];                            // fragments by lane
  union {
    uint8_t ring[WARPS][STAGES][kStage];
    struct {
      float part[WARPS][kRows][D + 4];
      float top[WARPS][kRows], total[WARPS][kRows];
    };
  };
};

template <class T, int D, int NT, int WARPS, int STAGES, int BLOCKS>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS) k_attend_cache_few(const __grid_constant__ AttendCacheParams p) {
  using Shared = CacheFewShared<T, D, NT, WARPS, STAGES>;
  using KT = typename std::conditional<std::is_same<T, __half>::value, __half, __nv_bfloat16>::type;
  using VT = __nv_bfloat16;
  constexpr int STEPS = D / 16, QTERMS = Shared::kQTerms, PTERMS = sizeof(T) == 4 ? 3 : 2, ROWS = Shared::kRows;
  constexpr int VB = Shared::kValueBytes;
  constexpr bool KEEP_Q = NT == 1 && QTERMS == 1 && D <= 128;  // queries in registers
  extern __shared__ __align__(128) uint8_t cache_few_smem[];
  Shared& sh = *reinterpret_cast<Shared*>(cache_few_smem);
  const CacheParams& c = p.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane >> 2, quad = lane & 3;
  const int range = blockIdx.z, kv_head = blockIdx.y, G = p.rows_a_head;
  ptx::grid_dependency_trigger();  // (whoever joins the ranges may be there, waiting)
  // rows of this tile: ROWS from row0 on, of a sequence or of all
  int sequence = 0;
  long long row0 = static_cast<long long>(blockIdx.x) * ROWS, first = 0, rows;
  int before = 0;  // position of a sequence's first row
  if (p.prefix) {
    rows = c.tokens * G;
  } else {
    const int tiles = static_cast<int>((static_cast<long long>(c.max_tokens) * G + ROWS - 1) / ROWS);
    sequence = blockIdx.x / tiles;
    row0 = static_cast<long long>(blockIdx.x % tiles) * ROWS;
    first = cache_start(c, sequence);
    const long long count = max(cache_start(c, sequence + 1) - first, 0ll);
    rows = min(count, static_cast<long long>(c.max_tokens)) * G;
    before = static_cast<int>(max(cache_len(c, sequence) - count, -(1ll << 30)));
  }
  // a lane's row: its token and position (-2: no row)
  const long long my_row = row0 + lane;
  int my_position = -2;
  if (lane < ROWS && my_row < rows) {
    if (p.prefix) {
      const CachePlace place = cache_place(c, my_row / G);
      my_position = place.sequence < 0 ? -2 : place.position;
    } else {
      my_position = max(before + static_cast<int>(my_row / G), -1);
    }
  }
  const int last = __reduce_max_sync(~0u, my_position);
  const int least = __reduce_min_sync(~0u, my_position < -1 ? 0x7fffffff : my_position);
  const int from = p.prefix ? range * p.chunk : p.shared + range * p.chunk;
  const int end = p.prefix ? min(p.shared, last + 1) : last + 1;
  const int to = min(from + p.chunk, end);
  // nothing to do (whoever joins knows), and before that the kernel that this one may have overtaken: its end is waited for through
  // this one's
  if (last == -2 || (from >= to && p.part != nullptr)) {
    ptx::grid_dependency_wait();
    return;
  }
  int position[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 2; ++e) position[t][e] = __shfl_sync(~0u, my_position, 8 * t + 2 * quad + e);

  const int table_row = p.prefix ? 0 : sequence;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(&sh.ring[warp][0][0])) + lane * 16;
  const uint32_t ring8 = ring - lane * 8;
  // pages of this warp's next 32 blocks, one to a lane
  int ahead = 0;
  uint32_t held = 0;  // of the blocks under way, the last one lowest: whether their page is there
  // this lane's bytes of a block's keys 2 group and 2 group + 1, and of the values 4 quad to 4 quad + 3
  const int k_byte = quad * 16, v_byte = group * VB;
  const long long k_from = static_cast<long long>(2 * group) * c.row + k_byte, v_from = static_cast<long long>(4 * quad) * c.row + v_byte;
  auto request = [&](int stage, int i) {
    const int key = from + (warp + i * WARPS) * 16;
    if ((i & 31) == 0) {
      const int mine = key + lane * WARPS * 16;
      ahead = mine < to ? cache_page(c, table_row, mine) : -1;
    }
    const int page = __shfl_sync(~0u, ahead, i & 31);
    const bool take = page >= 0;
    held = held << 1 | (take ? 1u : 0u);
    if (key < to) {
      const long long line = take ? ((static_cast<long long>(page) * c.kv_heads + kv_head) << c.page_shift) + (key & ((1 << c.page_shift) - 1)) : 0;
      const int8_t* k = c.k + (take ? line * c.row + k_from : 0);
      const int8_t* v = c.v + (take ? line * c.row + v_from : 0);
      const uint32_t at = ring + stage * Shared::kStage, at8 = ring8 + stage * Shared::kStage + Shared::kKeyBytes;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int cc = 0; cc < D / 64; ++cc) {
          const bool use = take && cc * 64 + k_byte < c.row;
          queue_16(at + (n * (D / 64) + cc) * 512, use ? k + n * c.row + cc * 64 : c.k, use);
        }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        if constexpr (VB == 8) {
          const bool use = take && v_byte < c.row;
          queue_8(at8 + n * 256, use ? v + n * c.row : c.v, use);
        } else {
#pragma unroll
          for (int h = 0; h < VB / 16; ++h) {
            const bool use = take && v_byte + h * 16 < c.row;
            queue_16(at + Shared::kKeyBytes + (n * (VB / 16) + h) * 512, use ? v + n * c.row + h * 16 : c.v, use);
          }
        }
      }
      queue_8(at8 + Shared::kValues, c.k_steps + (take ? line + 2 * group : 0), take);
      queue_8(at8 + Shared::kValues + 256, c.v_steps + (take ? line + 2 * group : 0), take);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int blocks = from < to ? ((to - from + 15) / 16 - warp + WARPS - 1) / WARPS : 0;
#pragma unroll
  for (int n = 0; n < STAGES - 1; ++n) request(n, n);

  // the queries as B fragments in the order of the keys' bytes: a warp makes every WARPS-th product's
  for (int s = warp; s < STEPS * NT; s += WARPS) {
    const int step = s / NT, t = s % NT;
    const int where = __shfl_sync(~0u, my_position, 8 * t + group);
    const long long row = row0 + 8 * t + group;
    const long long token = first + row / G;
    const int head = kv_head * G + static_cast<int>(row % G);
    const T* q = static_cast<const T*>(p.q) + token * p.q_token + head * p.q_head;
    uint32_t f[QTERMS][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int at = (step / 4) * 64 + quad * 16 + (step % 4) * 4 + 2 * e;
      const float x = where > -2 && at < c.d ? op_get(q[at]) : 0.0f, y = where > -2 && at + 1 < c.d ? op_get(q[at + 1]) : 0.0f;
      if constexpr (QTERMS == 1) {
        const OpVec<KT, 2> pair{{op_put<KT>(x), op_put<KT>(y)}};
        f[0][e] = *reinterpret_cast<const uint32_t*>(&pair);
      } else {
        uint32_t rest;
        split_pair<__nv_bfloat16>(x, y, f[0][e], rest);
        const float x1 = x - __bfloat162float(op_put<__nv_bfloat16>(x)), y1 = y - __bfloat162float(op_put<__nv_bfloat16>(y));
        split_pair<__nv_bfloat16>(x1, y1, f[1][e], f[2][e]);
      }
    }
#pragma unroll
    for (int w = 0; w < QTERMS; ++w) sh.q[w][step][t][lane] = make_uint2(f[w][0], f[w][1]);
  }
  __syncthreads();
  const uint32_t q_at = static_cast<uint32_t>(__cvta_generic_to_shared(&sh.q[0][0][0][0])) + lane * 8;
  uint2 q_held[KEEP_Q ? STEPS : 1];
  if constexpr (KEEP_Q)
#pragma unroll
    for (int s = 0; s < STEPS; ++s) q_held[s] = lds_8(q_at + s * 256);

  const float scale = p.scale_log2 * (std::is_same<KT, __half>::value ? 1.0f : kBf16Integers);
  float o[NT][STEPS][4] = {};
  float base[NT][2], total[NT][2] = {};
#pragma unroll
  for (int t = 0; t < NT; ++t) base[t][0] = base[t][1] = -INFINITY;
  int stage = 0;
  for (int i = 0; i < blocks; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    const bool there = held >> (STAGES - 2) & 1u;  // (before the next request's shift)
    request(stage == 0 ? STAGES - 1 : stage - 1, i + STAGES - 1);
    const uint32_t at = ring + stage * Shared::kStage, at8 = ring8 + stage * Shared::kStage + Shared::kKeyBytes;
    const int key = from + (warp + i * WARPS) * 16;
    float s[NT][4] = {};
#pragma unroll
    for (int cc = 0; cc < D / 64; ++cc) {
      const uint4 k0 = lds_16(at + cc * 512), k1 = lds_16(at + (D / 64 + cc) * 512);
      const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t a[4];
        int8_quad<KT>(w0[j], a[0], a[2]);
        int8_quad<KT>(w1[j], a[1], a[3]);
#pragma unroll
        for (int w = QTERMS - 1; w >= 0; --w)  // (small terms first)
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint2 b = KEEP_Q ? q_held[cc * 4 + j] : lds_8(q_at + ((w * STEPS + cc * 4 + j) * NT + t) * 256);
            mma_16x8x16<KT>(s[t], a, b.x, b.y);
          }
      }
    }
    // s[t][e]: key 2 group + e / 2, row 8 t + 2 quad + e % 2
    const uint2 ks = lds_8(at8 + Shared::kValues), vs = lds_8(at8 + Shared::kValues + 256);
    const float k_step[2] = {__uint_as_float(ks.x) * scale, __uint_as_float(ks.y) * scale};
    const float v_step[2] = {__uint_as_float(vs.x), __uint_as_float(vs.y)};
    const bool whole = there && key + 15 <= least && key + 15 < to;
    bool above = false;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[t][e] *= k_step[e >> 1];
        if (!whole) {
          const int at_key = key + 2 * group + (e >> 1);
          if (!there || at_key > position[t][e & 1] || at_key >= to) s[t][e] = -INFINITY;
        }
        above = above || s[t][e] > base[t][e & 1] + 8.0f;
      }
    // the base of the exponentials follows the maximum when that is 2^8 or more above it
    if (__any_sync(~0u, above)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float m = fmaxf(s[t][e], s[t][2 + e]);
          m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
          m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
          m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
          const float next = fmaxf(base[t][e], m);
          const float keep = next == -INFINITY ? 1.0f : exp2_approx(base[t][e] - next);
          base[t][e] = next;
          total[t][e] *= keep;
#pragma unroll
          for (int n = 0; n < STEPS; ++n) {
            o[t][n][e] *= keep;
            o[t][n][2 + e] *= keep;
          }
        }
    }
    uint32_t prob[PTERMS][NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float zero[2] = {base[t][0] == -INFINITY ? 0.0f : base[t][0], base[t][1] == -INFINITY ? 0.0f : base[t][1]};
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float e0 = exp2_approx(s[t][2 * n] - zero[0]), e1 = exp2_approx(s[t][2 * n + 1] - zero[1]);
        total[t][0] += e0;
        total[t][1] += e1;
        // (the step of a key that takes no part may be anything)
        const float y0 = !whole && s[t][2 * n] == -INFINITY ? 0.0f : e0 * v_step[n];
        const float y1 = !whole && s[t][2 * n + 1] == -INFINITY ? 0.0f : e1 * v_step[n];
        uint32_t term[PTERMS];
        split_pair<VT>(y0, y1, term[0], term[1]);
        if constexpr (PTERMS == 3) {
          const float r0 = y0 - __bfloat162float(op_put<VT>(y0)), r1 = y1 - __bfloat162float(op_put<VT>(y1));
          split_pair<VT>(r0, r1, term[1], term[2]);
        }
#pragma unroll
        for (int w = 0; w < PTERMS; ++w) prob[w][t][n] = turn_8x8(term[w]);
      }
    }
    // prob[.][t][n]: row 8 t + group, keys 4 quad + n and 4 quad + n + 2
    constexpr int WORDS = VB / 4;
    uint32_t v[4][WORDS];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if constexpr (VB == 8) {
        const uint2 w = lds_8(at8 + n * 256);
        v[n][0] = w.x;
        v[n][1] = w.y;
      } else {
#pragma unroll
        for (int h = 0; h < VB / 16; ++h) {
          const uint4 w = lds_16(at + Shared::kKeyBytes + (n * (VB / 16) + h) * 512);
          v[n][4 * h] = w.x;
          v[n][4 * h + 1] = w.y;
          v[n][4 * h + 2] = w.z;
          v[n][4 * h + 3] = w.w;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {
      // bytes 2 n and 2 n + 1 of two keys' words, in bytes 0 and 2
      const uint32_t even = 0x0400u + (2 * n % 4) * 0x0101u, odd = 0x0400u + ((2 * n + 1) % 4) * 0x0101u;
      const uint32_t a[4] = {bf16_pair(__byte_perm(v[0][n / 2], v[2][n / 2], even)), bf16_pair(__byte_perm(v[0][n / 2], v[2][n / 2], odd)),
                             bf16_pair(__byte_perm(v[1][n / 2], v[3][n / 2], even)), bf16_pair(__byte_perm(v[1][n / 2], v[3][n / 2], odd))};
#pragma unroll
      for (int w = PTERMS - 1; w >= 0; --w)
#pragma unroll
        for (int t = 0; t < NT; ++t) mma_16x8x16<VT>(o[t][n], a, prob[w][t][0], prob[w][t][1]);
    }
    stage = stage == STAGES - 1 ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // the results take the ring's place
  // o[t][n][e]: component group (D / 8) + 2 n + e / 2, row 8 t + 2 quad + e % 2
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 8 * t + 2 * quad + e;
      float sum = total[t][e];
      sum += __shfl_xor_sync(~0u, sum, 4);
      sum += __shfl_xor_sync(~0u, sum, 8);
      sum += __shfl_xor_sync(~0u, sum, 16);
      if (group == 0) {
        sh.top[warp][r] = base[t][e];
        sh.total[warp][r] = sum;
      }
      if (position[t][e] > -2)
#pragma unroll
        for (int n = 0; n < STEPS; n += 2)
          *reinterpret_cast<float4*>(&sh.part[warp][r][group * (D / 8) + 2 * n]) = make_float4(o[t][n][e], o[t][n][2 + e], o[t][n + 1][e], o[t][n + 1][2 + e]);
    }
  __syncthreads();
  const long long all_rows = c.tokens * p.heads;
  for (int i = threadIdx.x; i < ROWS * (D / 4); i += WARPS * 32) {
    const int r = i / (D / 4), at = i % (D / 4) * 4;
    const int where = __shfl_sync(~0u, my_position, r);
    if (where < -1 || at >= c.d) continue;
    float top = sh.top[0][r];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sh.top[w][r]);
    const float zero = top == -INFINITY ? 0.0f : top;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float all = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = exp2f(sh.top[w][r] - zero);
      const float4 y = *reinterpret_cast<const float4*>(&sh.part[w][r][at]);
      sum = make_float4(fmaf(f, y.x, sum.x), fmaf(f, y.y, sum.y), fmaf(f, y.z, sum.z), fmaf(f, y.w, sum.w));
      all = fmaf(f, sh.total[w][r], all);
    }
    sum = make_float4(sum.x * kBf16Integers, sum.y * kBf16Integers, sum.z * kBf16Integers, sum.w * kBf16Integers);
    const long long row = row0 + r, token = first + row / G;
    const int head = kv_head * G + static_cast<int>(row % G);
    if (p.part != nullptr) {
      const long long line = (p.first_range + range) * all_rows + token * p.heads + head;
      *reinterpret_cast<float4*>(p.part + line * p.part_width + at) = sum;
      if (at == 0) p.part_top[line] = make_float2(top, all);
    } else {
      const float scale = all == 0.0f ? 0.0f : 1.0f / all;
      T* out = static_cast<T*>(p.o) + token * p.o_token + head * p.o_head + at;
      const float y[4] = {sum.x * scale, sum.y * scale, sum.z * scale, sum.w * scale};
      if (p.o_wide) {
        OpVec<T, 4> w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w.e[e] = op_put<T>(all == 0.0f ? 0.0f : y[e]);
        *reinterpret_cast<OpVec<T, 4>*>(out) = w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (at + e < c.d) out[e] = op_put<T>(all == 0.0f ? 0.0f : y[e]);
      }
    }
  }
  ptx::grid_dependency_wait();
}

// The ranges' results of a row, joined: a warp to a row, ranges in the order of the keys.
template <class T>
__global__ void __launch_bounds__(256) k_attend_cache_join(const __grid_constant__ AttendCacheParams p) {
  ptx::grid_dependency_wait();  // (launched early)
  const CacheParams& c = p.c;
  const int lane = threadIdx.x & 31;
  const long long rows = c.tokens * p.heads, row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const long long token = row / p.heads;
  const int head = static_cast<int>(row - token * p.heads);
  const CachePlace place = cache_place(c, token);
  if (place.sequence < 0) return;
  // the ranges that hold keys of this row
  const int of_prefix = place.position < 0 || p.shared == 0 ? 0 : min(place.position, p.shared - 1) / p.prefix_chunk + 1;
  const int own = place.position < p.shared ? 0 : (place.position - p.shared) / p.own_chunk + 1;
  const int ranges = of_prefix + own;
  auto line_of = [&](int n) { return (n < of_prefix ? n : p.prefix_ranges + n - of_prefix) * rows + row; };
  float top = -INFINITY;
  for (int n = lane; n < ranges; n += 32) top = fmaxf(top, p.part_top[line_of(n)].x);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, w));
  const float zero = top == -INFINITY ? 0.0f : top;
  float all = 0.0f;
  float4 sum[2] = {};
  for (int n0 = 0; n0 < ranges; n0 += 32) {
    float2 mine = make_float2(-INFINITY, 0.0f);
    if (n0 + lane < ranges) mine = p.part_top[line_of(n0 + lane)];
    const float factor = exp2f(mine.x - zero);
    const int here = min(32, ranges - n0);
#pragma unroll 4
    for (int n = 0; n < here; ++n) {
      const float f = __shfl_sync(~0u, factor, n);
      all = fmaf(f, __shfl_sync(~0u, mine.y, n), all);
      const float* from = p.part + line_of(n0 + n) * p.part_width;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = h * 128 + lane * 4;
        if (at < c.d) {
          const float4 y = *reinterpret_cast<const float4*>(from + at);
          sum[h] = make_float4(fmaf(f, y.x, sum[h].x), fmaf(f, y.y, sum[h].y), fmaf(f, y.z, sum[h].z), fmaf(f, y.w, sum[h].w));
        }
      }
    }
  }
  const float scale = all == 0.0f ? 0.0f : 1.0f / all;
  T* out = static_cast<T*>(p.o) + token * p.o_token + head * p.o_head;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = h * 128 + lane * 4;
    const float y[4] = {sum[h].x * scale, sum[h].y * scale, sum[h].z * scale, sum[h].w * scale};
    if (at >= c.d) continue;
    if (p.o_wide) {
      OpVec<T, 4> w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w.e[e] = op_put<T>(all == 0.0f ? 0.0f : y[e]);
      *reinterpret_cast<OpVec<T, 4>*>(out + at) = w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (at + e < c.d) out[at + e] = op_put<T>(all == 0.0f ? 0.0f : y[e]);
    }
  }
}

}  // namespace nb
