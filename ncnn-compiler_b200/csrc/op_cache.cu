// A paged cache of keys and values in 8-bit integers on device arrays: quantised as they are written (ncnn_b200_op_cache_write),
// read back (ncnn_b200_op_cache_read), and attention over it (ncnn_b200_op_cache_attention).
#include <array>
#include <cmath>

#include "attend_cache.cuh"
#include "op_cache.h"
#include "row_int8.cuh"
#include "tc_attend_cache.cuh"

namespace nb {
namespace {

struct CacheRowsParams {
  CacheParams c;
  void *k, *v;  // the call's arrays (writing: read only)
  long long k_token, k_head, v_token, v_head;
  int kinds;    // 2: keys and values; 1: those that are not null
};

// PER rows (keys or values of neighbouring heads of a token) to LANES lanes, eight components of each row to a lane: what a lane reads of
// a row is one or two accesses of 16 bytes (WIDE) or eight elements.  Bound: instructions for many tokens (83 % of the issue slots when
// writing, 75 % when reading; HBM at 36 and 43 %), which wants several rows under way in each lane and their place found once; the chain of
// loads (starts, lens, table, row) for few, which wants many lanes.  36864 tokens of 8 heads of 128, f16: written in 64 us (3.6 TB/s),
// read in 47 (4.8); a row to a group of lanes 136 and 112.
template <class T, int LANES, int PER, bool WIDE, bool READ>
__global__ void __launch_bounds__(256) k_cache_rows(const __grid_constant__ CacheRowsParams p) {
  const CacheParams& c = p.c;
  constexpr int GROUPS = 256 / LANES, V = 16 / sizeof(T);
  const int lane = threadIdx.x % LANES;
  const int chunks = (c.kv_heads + PER - 1) / PER;
  const long long groups = c.tokens * p.kinds * chunks;
  const long long group = static_cast<long long>(blockIdx.x) * GROUPS + threadIdx.x / LANES;
  const bool there = group < groups;
  const long long rest = (there ? group : 0) / chunks, token = rest / p.kinds;
  const int head0 = static_cast<int>((there ? group : 0) - rest * chunks) * PER;
  const int rows = there ? min(PER, c.kv_heads - head0) : 0;
  const bool value = p.kinds == 2 ? rest % 2 == 1 : p.k == nullptr;
  const long long head_step = value ? p.v_head : p.k_head;
  const int at = lane * 8;
  T* row = static_cast<T*>(value ? p.v : p.k) + token * (value ? p.v_token : p.k_token) + head0 * head_step + at;
  OpVec<T, V> x[PER][8 / V];
  if constexpr (!READ) {
    // (asked for before the rows' place is known)
#pragma unroll
    for (int r = 0; r < PER; ++r)
#pragma unroll
      for (int i = 0; i < 8 / V; ++i) {
        x[r][i] = {};
        if constexpr (WIDE) {
          if (r < rows && at + i * V < c.d) x[r][i] = *reinterpret_cast<const OpVec<T, V>*>(row + r * head_step + i * V);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (r < rows && at + i * V + e < c.d) x[r][i].e[e] = row[r * head_step + i * V + e];
        }
      }
  }
  const CachePlace place = there ? cache_place(c, token) : CachePlace{-1, -1};
  const int page = place.sequence < 0 || place.position < 0 ? -1 : cache_page(c, place.sequence, place.position);
  const long long slot = (((page < 0 ? 0ll : page) * c.kv_heads + head0) << c.page_shift) + (place.position & ((1 << c.page_shift) - 1));
  int8_t* ints = (value ? c.v : c.k) + slot * c.row + at;
  float* steps = (value ? c.v_steps : c.k_steps) + slot;
  const long long line = 1ll << c.page_shift;  // rows from a head to the next
  if constexpr (READ) {
    uint2 w[PER];
    float step[PER];
#pragma unroll
    for (int r = 0; r < PER; ++r) {
      w[r] = make_uint2(0u, 0u);
      step[r] = 0.0f;
      if (r < rows && page >= 0 && at < c.row) {
        w[r] = *reinterpret_cast<const uint2*>(ints + r * line * c.row);
        step[r] = steps[r * line];
      }
    }
    if (place.sequence < 0) return;
#pragma unroll
    for (int r = 0; r < PER; ++r) {
      if (r >= rows) break;
#pragma unroll
      for (int i = 0; i < 8 / V; ++i) {
        OpVec<T, V> out;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int n = i * V + e;
          out.e[e] = op_put<T>(static_cast<float>(static_cast<int8_t>((n < 4 ? w[r].x : w[r].y) >> (8 * (n % 4)))) * step[r]);
        }
        if constexpr (WIDE) {
          if (at + i * V < c.d) *reinterpret_cast<OpVec<T, V>*>(row + r * head_step + i * V) = out;
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (at + i * V + e < c.d) row[r * head_step + i * V + e] = out.e[e];
        }
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < PER; ++r) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8 / V; ++i) top = row_top(x[r][i], top);
      top = row_top_bits<T>(top);
#pragma unroll
      for (int w = LANES / 2; w > 0; w >>= 1) top = max(top, __shfl_xor_sync(~0u, top, w));
      if (r >= rows || page < 0 || at >= c.row) continue;
      const RowScale scale = row_scale<T>(top);
      uint32_t w[2] = {0u, 0u};
      if (scale.factor != 0.0f) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          uint32_t b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) b[e] = row_integer<T>(op_get(x[r][(4 * g + e) / V].e[(4 * g + e) % V]), scale);
          w[g] = low_bytes(b[0], b[1], b[2], b[3]);
        }
      }
      *reinterpret_cast<uint2*>(ints + r * line * c.row) = make_uint2(w[0], w[1]);
      if (lane == 0) steps[r * line] = scale.step;
    }
  }
}

template <class T, bool READ>
cudaError_t cache_rows(const CacheRowsParams& p, bool wide, int sms, cudaStream_t st) {
  const int pieces = p.c.row / 8;
  auto go = [&](auto lanes, auto per) {
    constexpr int LANES = decltype(lanes)::value, PER = decltype(per)::value;
    const long long groups = p.c.tokens * p.kinds * ((p.c.kv_heads + PER - 1) / PER);
    const dim3 grid(static_cast<unsigned>((groups + 256 / LANES - 1) / (256 / LANES)));
    return wide ? op_launch(k_cache_rows<T, LANES, PER, true, READ>, grid, 256, 0, st, 0, p) : op_launch(k_cache_rows<T, LANES, PER, false, READ>, grid, 256, 0, st, 0, p);
  };
  auto by_lanes = [&](auto per) {
    if (pieces <= 8) return go(std::integral_constant<int, 8>{}, per);
    return pieces <= 16 ? go(std::integral_constant<int, 16>{}, per) : go(std::integral_constant<int, 32>{}, per);
  };
  // four rows to a lane where there are enough of them for the whole device
  const long long rows = p.c.tokens * p.kinds * p.c.kv_heads;
  return p.c.kv_heads > 1 && rows * pieces >= 4096ll * sms ? by_lanes(std::integral_constant<int, 4>{}) : by_lanes(std::integral_constant<int, 1>{});
}

// ------------------------------------------------------------------ arguments
// What a cache and a batch say, checked: 0, or a status (the message is set).
int cache_params(const char* op, const ncnn_b200_cache* cache, const ncnn_b200_cache_batch* batch, CacheParams* p) {
  auto bad = [&](const char* what) { return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, std::string(op) + ": " + what); };
  if (cache == nullptr || batch == nullptr) return op_fail(NCNN_B200_STATUS_NULL_POINTER, std::string(op) + ": NULL cache or batch");
  if (cache->page_size < 16 || cache->page_size > 1024 || (cache->page_size & (cache->page_size - 1)) != 0)
    return bad("page_size is a power of two from 16 to 1024");
  if (cache->head_dim < 1 || cache->head_dim > 256 || cache->kv_heads < 1 || cache->kv_heads > 65535 || cache->pages < 0 || cache->pages > 0x7fffffffll)
    return bad("head_dim 1 to 256, kv_heads 1 to 65535, pages 0 to 2^31 - 1");
  if (batch->sequences < 0 || batch->sequences > (1 << 24) || batch->tokens < 0 || batch->tokens > 0x7fffffffll || batch->table_width < 0 || batch->max_tokens < 0 ||
      batch->max_len < 0)
    return bad("sequences 0 to 2^24, tokens 0 to 2^31 - 1, and no negative table_width, max_tokens or max_len");
  const long long room = static_cast<long long>(batch->table_width) * cache->page_size;
  if (room > (1 << 30)) return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, std::string(op) + ": a row of the table holds more than 2^30 positions");
  if (batch->max_len > room) return bad("max_len is more than a row of the table holds");
  if (batch->sequences > 0 && batch->tokens > 0) {
    if (cache->k == nullptr || cache->v == nullptr || cache->k_steps == nullptr || cache->v_steps == nullptr || batch->lens == nullptr ||
        (batch->table == nullptr && batch->table_width > 0))
      return op_fail(NCNN_B200_STATUS_NULL_POINTER, std::string(op) + ": NULL array in the cache or the batch");
    if (!op_starts(cache->k, 16) || !op_starts(cache->v, 16) || !op_starts(cache->k_steps, 16) || !op_starts(cache->v_steps, 16))
      return bad("the cache's arrays start at multiples of 16 bytes");
    if (!op_starts(batch->table, 4) || !op_starts(batch->lens, 4) || !op_starts(batch->starts, 4)) return bad("an array does not start at a multiple of its elements' size");
    for (const void* ints : {cache->k, cache->v})
      if (ints == cache->k_steps || ints == cache->v_steps) return bad("integers and steps need memory of their own");
    if (cache->k == cache->v || cache->k_steps == cache->v_steps) return bad("keys and values need memory of their own");
  }
  p->k = cache->k;
  p->v = cache->v;
  p->k_steps = cache->k_steps;
  p->v_steps = cache->v_steps;
  p->pages = cache->pages;
  p->page_shift = 0;
  while ((1 << p->page_shift) < cache->page_size) ++p->page_shift;
  p->kv_heads = cache->kv_heads;
  p->d = cache->head_dim;
  p->row = (cache->head_dim + 15) / 16 * 16;
  p->table = batch->table;
  p->lens = batch->lens;
  p->starts = batch->starts;
  p->sequences = static_cast<int>(batch->sequences);
  p->width = batch->table_width;
  p->tokens = batch->tokens;
  p->max_tokens = static_cast<int>(batch->max_tokens == 0 ? batch->tokens : std::min<int64_t>(batch->max_tokens, batch->tokens));
  if (batch->starts == nullptr) p->max_tokens = std::min(p->max_tokens, 1);
  p->max_len = static_cast<int>(batch->max_len == 0 ? room : batch->max_len);
  return 0;
}

// {token, head} strides of an array of `heads` rows of d at each token; `written`: rows must not overlap.
int row_strides(const char* op, const int64_t* given, long long tokens, int heads, int d, bool written, long long* token, long long* head) {
  if (given == nullptr) {
    *token = static_cast<long long>(heads) * d;
    *head = d;
    return 0;
  }
  *token = given[0];
  *head = given[1];
  for (int i = 0; i < 2; ++i) {
    if (given[i] < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, std::string(op) + ": a stride is negative");
    if (given[i] > (1ll << 50) / std::max<int64_t>({tokens, heads, 1})) return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, std::string(op) + ": a stride is too large");
  }
  if (written) {
    std::array<std::pair<int64_t, int64_t>, 2> axes = {{{*token, tokens}, {*head, heads}}};
    std::sort(axes.begin(), axes.end());
    int64_t extent = d;
    for (const auto& a : axes) {
      if (a.second == 1) continue;
      if (a.first < extent) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, std::string(op) + ": the result's rows overlap");
      extent = a.first * (a.second - 1) + extent;
    }
  }
  return 0;
}

// Whether `count` elements can be moved at a time in all rows of an array.
bool moves(const void* base, int count, int size, int d, long long tokens, long long token, int heads, long long head) {
  return base == nullptr || (d % count == 0 && reinterpret_cast<uintptr_t>(base) % (count * size) == 0 && (tokens == 1 || token % count == 0) &&
                             (heads == 1 || head % count == 0));
}

int cache_rows_call(const char* op, bool read, const ncnn_b200_cache* cache, const ncnn_b200_cache_batch* batch, void* k, void* v, int32_t type,
                    const int64_t* strides, void* stream) {
  return op_guarded(op, [&]() -> int {
    auto bad = [&](const char* what) { return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, std::string(op) + ": " + what); };
    if (!op_type_ok(type)) return bad("unknown element type");
    CacheRowsParams p{};
    if (const int e = cache_params(op, cache, batch, &p.c); e != 0) return e;
    const int size = op_elem_bytes(type);
    if (const int e = row_strides(op, strides, p.c.tokens, p.c.kv_heads, p.c.d, read && k != nullptr, &p.k_token, &p.k_head); e != 0) return e;
    if (const int e = row_strides(op, strides == nullptr ? nullptr : strides + 2, p.c.tokens, p.c.kv_heads, p.c.d, read && v != nullptr, &p.v_token, &p.v_head); e != 0)
      return e;
    if (p.c.tokens * 2 * p.c.kv_heads > (1ll << 33)) return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, std::string(op) + ": more than 2^33 rows");
    if (p.c.tokens == 0 || p.c.sequences == 0) return NCNN_B200_STATUS_SUCCESS;
    if (read ? k == nullptr && v == nullptr : k == nullptr || v == nullptr) return op_fail(NCNN_B200_STATUS_NULL_POINTER, std::string(op) + ": NULL argument");
    if (!op_starts(k, size) || !op_starts(v, size)) return bad("an array does not start at a multiple of its elements' size");
    for (const void* a : {static_cast<const void*>(k), static_cast<const void*>(v)}) {
      if (a == nullptr) continue;
      if (a == p.c.k || a == p.c.v || a == p.c.k_steps || a == p.c.v_steps) return bad("the arrays must not lie over the cache");
      if (a == p.c.table || a == p.c.lens || a == p.c.starts) return bad("the arrays must not lie over the batch's");
    }
    if (read && k == v) return bad("keys and values need memory of their own");
    p.k = k;
    p.v = v;
    p.kinds = k != nullptr && v != nullptr ? 2 : 1;
    std::string why;
    const int device = op_common_device(op, {k, v, p.c.k, p.c.v, p.c.k_steps, p.c.v_steps, p.c.table, p.c.lens, p.c.starts}, &why);
    if (device < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, why);
    DeviceGuard guard(device);
    const int count = 16 / size;
    const bool wide = moves(k, count, size, p.c.d, p.c.tokens, p.k_token, p.c.kv_heads, p.k_head) &&
                      moves(v, count, size, p.c.d, p.c.tokens, p.v_token, p.c.kv_heads, p.v_head);
    return op_by_type(type, [&](auto t) {
      using T = decltype(t);
      const cudaStream_t st = static_cast<cudaStream_t>(stream);
      const int sms = op_sm_count(device);
      return op_launched(op, read ? cache_rows<T, true>(p, wide, sms, st) : cache_rows<T, false>(p, wide, sms, st));
    });
  });
}

// ------------------------------------------------------------------ attention
// How the keys of a call, of its shared prefix and of the sequences' own, are walked: by which kernel, and in ranges of how many.
struct AttendCachePart {
  int wide, ranges, chunk;
};
struct AttendCachePlan {
  AttendCachePart prefix, own;
  int ranges() const { return prefix.ranges + own.ranges; }
};

int up(long long x, int to) { return static_cast<int>((x + to - 1) / to * to); }

// Rows of a tile: eights, sixteens or, of heads up to 128, thirty-twos.
int few_rows(long long rows, int d) { return rows <= 8 ? 8 : rows <= 16 || d > 128 ? 16 : 32; }

// More rows to a key head than this go through tiles of 128 rows (32 heads over 8 key heads of 128, one sequence of 16000 keys: 68 rows
// 32 us, 64 rows in thirty-twos 47; 16 sequences of 2000: 96 rows 40, 64 rows in thirty-twos 47).
constexpr int kWideRows = 32;

AttendCachePlan attend_cache_plan(const CacheParams& c, int heads, long long shared, int sms, bool halves) {
  const int G = heads / c.kv_heads;
  auto part = [&](long long keys, long long sequences, long long rows) {
    AttendCachePart p{0, 0, 128};
    if (keys <= 0) return p;
    p.wide = halves && c.d <= 128 && rows > kWideRows ? 1 : 0;
    const int height = p.wide ? 256 : few_rows(rows, c.d);
    const long long tiles = std::max<long long>(1, sequences * c.kv_heads * ((rows + height - 1) / height));
    // Ranges, 64 at most.  Tiles of 128 rows: as many as give each SM a CTA, of 512 keys or more.  Few rows: where there are no more tiles
    // than SMs, as many as fill the device once (two CTAs to an SM), of 256 keys or more: a CTA has 3 to 4 us of its own (8 sequences of
    // 8192 keys, 64 tiles: 4 ranges 40 us, 9 46, 18 54; one of 60001: 37 ranges 45, 64 57).  Otherwise up to eight CTAs to an SM, of
    // 1024 keys or more, which evens out sequences of different lengths (64 of up to 8192, 512 tiles: 1 range 156 us, 2 140, 9 155).
    const long long most = std::max<long long>(1, p.wide          ? std::min<long long>({64, (keys + 511) / 512, sms / tiles})
                                                  : tiles <= sms ? std::min<long long>({64, (keys + 255) / 256, 2ll * sms / tiles})
                                                                 : std::min<long long>({64, (keys + 1023) / 1024, 8ll * sms / tiles}));
    p.chunk = up((keys + most - 1) / most, p.wide ? 128 : 64);
    p.ranges = static_cast<int>((keys + p.chunk - 1) / p.chunk);
    return p;
  };
  AttendCachePlan plan{};
  const long long in_prefix = std::min<long long>(shared, c.max_len);
  plan.prefix = part(in_prefix, 1, c.tokens * G);
  plan.own = part(c.max_len - in_prefix, c.sequences, static_cast<long long>(c.max_tokens) * G);
  return plan;
}

long long attend_cache_bytes(const CacheParams& c, int heads, const AttendCachePlan& plan) {
  if (plan.ranges() <= 1) return 0;
  return plan.ranges() * c.tokens * heads * (c.row * 4ll + 8);
}
// (for any type)
long long attend_cache_workspace(const CacheParams& c, int heads, long long shared, int sms) {
  return std::max(attend_cache_bytes(c, heads, attend_cache_plan(c, heads, shared, sms, true)),
                  attend_cache_bytes(c, heads, attend_cache_plan(c, heads, shared, sms, false)));
}

template <class T, int D>
cudaError_t launch_cache_wide(const AttendCacheParams& a, int ranges, bool early, bool q_wide, int device, cudaStream_t st) {
  using Shape = TcCacheShape<D>;
  TcCacheParams p{};
  p.a = a;
  p.q_wide = q_wide ? 1 : 0;
  p.stall = op_stalled() ? 1 : 0;
  p.wait_ns = op_wait_ns(kTcWaitLimitNs);
  static std::atomic<uint64_t> granted{0};
  const auto kernel = tc_attend_cache_kernel<T, D>;
  if (const cudaError_t e = op_grant_smem(kernel, Shape::kSmem, device, &granted, Shape::kRegsLaunch); e != cudaSuccess) return e;
  const long long G = a.rows_a_head;
  const long long tiles = a.prefix ? (a.c.tokens * G + 255) / 256 : static_cast<long long>(a.c.sequences) * ((a.c.max_tokens * G + 255) / 256);
  if (tiles * a.c.kv_heads > 0x7fffffffll) return cudaErrorInvalidValue;
  op_will_wait_on(device);
  return op_launch_early(early, kernel, dim3(static_cast<unsigned>(tiles * a.c.kv_heads), ranges), Shape::kThreads, Shape::kSmem, st, 0, p);
}

template <class T, int D, int NT, int WARPS, int STAGES, int BLOCKS>
cudaError_t launch_cache_few(const AttendCacheParams& p, int ranges, bool early, int device, cudaStream_t st) {
  constexpr int smem = sizeof(CacheFewShared<T, D, NT, WARPS, STAGES>), ROWS = 8 * NT;
  static_assert(BLOCKS * (smem + 1024) <= 228 * 1024, "shared memory of an SM");
  static std::atomic<uint64_t> granted{0};
  const auto kernel = k_attend_cache_few<T, D, NT, WARPS, STAGES, BLOCKS>;
  if (const cudaError_t e = op_grant_smem(kernel, smem, device, &granted); e != cudaSuccess) return e;
  const long long G = p.rows_a_head;
  const long long tiles = p.prefix ? (p.c.tokens * G + ROWS - 1) / ROWS : static_cast<long long>(p.c.sequences) * ((p.c.max_tokens * G + ROWS - 1) / ROWS);
  if (tiles > 0x7fffffffll) return cudaErrorInvalidValue;
  return op_launch_early(early, kernel, dim3(static_cast<unsigned>(tiles), p.c.kv_heads, ranges), WARPS * 32, smem, st, 0, p);
}

template <class T>
cudaError_t attend_cache_few(const AttendCacheParams& p, int ranges, bool early, int device, cudaStream_t st) {
  const int rows = few_rows((p.prefix ? p.c.tokens : p.c.max_tokens) * static_cast<long long>(p.rows_a_head), p.c.d);
  if (p.c.d <= 64) {
    if (rows == 8) return launch_cache_few<T, 64, 1, 4, 5, 4>(p, ranges, early, device, st);
    return rows == 16 ? launch_cache_few<T, 64, 2, 4, 4, 4>(p, ranges, early, device, st) : launch_cache_few<T, 64, 4, 4, 4, 3>(p, ranges, early, device, st);
  }
  if (p.c.d <= 128) {
    if (rows == 8) return launch_cache_few<T, 128, 1, 8, 3, sizeof(T) == 4 ? 1 : 2>(p, ranges, early, device, st);
    return rows == 16 ? launch_cache_few<T, 128, 2, 4, 4, 2>(p, ranges, early, device, st) : launch_cache_few<T, 128, 4, 4, 3, 2>(p, ranges, early, device, st);
  }
  return rows == 8 ? launch_cache_few<T, 256, 1, 4, 3, sizeof(T) == 4 ? 1 : 2>(p, ranges, early, device, st) : launch_cache_few<T, 256, 2, 4, 3, 1>(p, ranges, early, device, st);
}

template <class T>
cudaError_t attend_cache_part(AttendCacheParams p, const AttendCachePart& part, bool early, bool q_wide, int device, cudaStream_t st) {
  p.chunk = part.chunk;
  const int ranges = std::max(part.ranges, 1);
  if constexpr (sizeof(T) == 2)
    if (part.wide) return p.c.d <= 64 ? launch_cache_wide<T, 64>(p, ranges, early, q_wide, device, st) : launch_cache_wide<T, 128>(p, ranges, early, q_wide, device, st);
  return attend_cache_few<T>(p, ranges, early, device, st);
}

int attend_cache_args(const char* op, const ncnn_b200_cache* cache, const ncnn_b200_cache_batch* batch, int32_t heads, int64_t shared, CacheParams* c) {
  if (const int e = cache_params(op, cache, batch, c); e != 0) return e;
  auto bad = [&](const char* what) { return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, std::string(op) + ": " + what); };
  if (heads <= 0 || heads > 65535 || heads % c->kv_heads != 0) return bad("heads is a multiple of kv_heads up to 65535");
  if (shared < 0 || shared % cache->page_size != 0 || shared > static_cast<long long>(c->width) * cache->page_size)
    return bad("shared is a multiple of page_size, and no more than a row of the table holds");
  if (c->tokens * heads > (1ll << 31)) return op_fail(NCNN_B200_STATUS_SHAPE_OVERFLOW, std::string(op) + ": more than 2^31 rows");
  return 0;
}

}  // namespace

cudaError_t cache_gave_up(unsigned* count) {
  return cudaMemcpyFromSymbol(count, g_cache_gave_up, sizeof *count);
}

}  // namespace nb

extern "C" int ncnn_b200_op_cache_write(const ncnn_b200_cache* cache, const ncnn_b200_cache_batch* batch, const void* k, const void* v, int32_t type,
                                        const int64_t* strides, void* stream) {
  return nb::cache_rows_call("op_cache_write", false, cache, batch, const_cast<void*>(k), const_cast<void*>(v), type, strides, stream);
}

extern "C" int ncnn_b200_op_cache_read(const ncnn_b200_cache* cache, const ncnn_b200_cache_batch* batch, void* k, void* v, int32_t type,
                                       const int64_t* strides, void* stream) {
  return nb::cache_rows_call("op_cache_read", true, cache, batch, k, v, type, strides, stream);
}

extern "C" int64_t ncnn_b200_op_cache_attention_workspace(const ncnn_b200_cache* cache, const ncnn_b200_cache_batch* batch, int32_t heads, int64_t shared) {
  using namespace nb;
  static const char* kOp = "op_cache_attention_workspace";
  int64_t bytes = -1;
  op_guarded(kOp, [&]() -> int {
    CacheParams c{};
    if (const int e = attend_cache_args(kOp, cache, batch, heads, shared, &c); e != 0) return e;
    if (c.tokens == 0 || c.sequences == 0) {
      bytes = 0;
      return 0;
    }
    std::string why;
    const int device = op_common_device(kOp, {c.k}, &why);
    if (device < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, why);
    bytes = attend_cache_workspace(c, heads, shared, op_sm_count(device));
    return 0;
  });
  return bytes;
}

extern "C" int ncnn_b200_op_cache_attention(const ncnn_b200_cache* cache, const ncnn_b200_cache_batch* batch, const void* q, void* o, int32_t type, int32_t heads,
                                            const int64_t* strides, int64_t shared, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace nb;
  static const char* kOp = "op_cache_attention";
  return op_guarded(kOp, [&]() -> int {
    auto bad = [&](const char* what) { return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, std::string(kOp) + ": " + what); };
    if (!op_type_ok(type)) return bad("unknown element type");
    AttendCacheParams p{};
    if (const int e = attend_cache_args(kOp, cache, batch, heads, shared, &p.c); e != 0) return e;
    if (!(scale >= 0.0f) || std::isinf(scale * 1.44269504088896340736f)) return bad("scale must not be negative, and scale / ln 2 finite");
    if (const int e = row_strides(kOp, strides, p.c.tokens, heads, p.c.d, false, &p.q_token, &p.q_head); e != 0) return e;
    if (const int e = row_strides(kOp, strides == nullptr ? nullptr : strides + 2, p.c.tokens, heads, p.c.d, true, &p.o_token, &p.o_head); e != 0) return e;
    if (p.c.tokens == 0 || p.c.sequences == 0) return NCNN_B200_STATUS_SUCCESS;
    if (q == nullptr || o == nullptr) return op_fail(NCNN_B200_STATUS_NULL_POINTER, "op_cache_attention: NULL argument");
    const int size = op_elem_bytes(type);
    if (!op_starts(q, size) || !op_starts(o, size) || !op_starts(workspace, 16))
      return bad("an array does not start at a multiple of its elements' size (workspace: of 16 bytes)");
    for (const void* a : {static_cast<const void*>(p.c.k), static_cast<const void*>(p.c.v), static_cast<const void*>(p.c.k_steps),
                          static_cast<const void*>(p.c.v_steps), static_cast<const void*>(p.c.table), static_cast<const void*>(p.c.lens),
                          static_cast<const void*>(p.c.starts), q})
      if (a != nullptr && (a == o || a == workspace)) return bad("the result and the workspace must not lie over an input");
    if (o == workspace) return bad("the result and the workspace must not lie over each other");
    std::string why;
    const int device = op_common_device(kOp, {q, o, p.c.k, p.c.v, p.c.k_steps, p.c.v_steps, p.c.table, p.c.lens, p.c.starts, workspace}, &why);
    if (device < 0) return op_fail(NCNN_B200_STATUS_INVALID_SHAPE, why);
    DeviceGuard guard(device);
    const int sms = op_sm_count(device);
    const AttendCachePlan plan = attend_cache_plan(p.c, heads, shared, sms, type != NCNN_B200_F32);
    const long long bytes = attend_cache_workspace(p.c, heads, shared, sms);
    if (bytes > 0 && workspace == nullptr) return op_fail(NCNN_B200_STATUS_NULL_POINTER, "op_cache_attention: this call needs a workspace");
    if (bytes > workspace_bytes && bytes > 0) return op_fail(NCNN_B200_STATUS_OUTPUT_CAPACITY, "op_cache_attention: the workspace is too small");
    p.q = q;
    p.o = o;
    p.heads = heads;
    p.rows_a_head = heads / p.c.kv_heads;
    p.scale_log2 = (scale == 0.0f ? 1.0f / std::sqrt(static_cast<float>(p.c.d)) : scale) * 1.44269504088896340736f;
    p.shared = static_cast<int>(shared);
    p.prefix_ranges = plan.prefix.ranges;
    p.prefix_chunk = plan.prefix.chunk;
    p.own_ranges = plan.own.ranges;
    p.own_chunk = plan.own.chunk;
    p.part_width = p.c.row;
    if (plan.ranges() > 1) {
      p.part = static_cast<float*>(workspace);
      p.part_top = reinterpret_cast<float2*>(p.part + static_cast<long long>(plan.ranges()) * p.c.tokens * heads * p.part_width);
    }
    p.o_wide = moves(o, 4, size, p.c.d, p.c.tokens, p.o_token, heads, p.o_head) ? 1 : 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return op_by_type(type, [&](auto t) {
      using T = decltype(t);
      cudaError_t e = cudaSuccess;
      const bool q_wide = moves(q, 16 / size, size, p.c.d, p.c.tokens, p.q_token, heads, p.q_head);
      if (plan.prefix.ranges > 0) {
        AttendCacheParams first = p;
        first.prefix = 1;
        e = attend_cache_part<T>(first, plan.prefix, false, q_wide, device, st);
      }
      // The sequences' own keys.  (Without any keys there is still a result: zeros.)  Beside the prefix's: the kernel waits for that one's
      // end before its own.
      if (e == cudaSuccess && (plan.own.ranges > 0 || plan.prefix.ranges == 0)) {
        AttendCacheParams own = p;
        own.first_range = plan.prefix.ranges;
        e = attend_cache_part<T>(own, plan.own, plan.prefix.ranges > 0, q_wide, device, st);
      }
      if (e == cudaSuccess && p.part != nullptr)
        e = op_launch_early(true, k_attend_cache_join<T>, dim3(static_cast<unsigned>((p.c.tokens * heads + 7) / 8)), 256, 0, st, 0, p);
      return op_launched(kOp, e);
    });
  });
}
