// What the kernels on the paged cache (ncnn_b200_op_cache_write, _read, _attention) share.
#pragma once

#include "op_common.cuh"

namespace nb {

struct CacheParams {
  int8_t *k, *v;
  float *k_steps, *v_steps;
  long long pages;
  int page_shift, kv_heads, d, row;  // row: bytes of a row
  const int *table, *lens, *starts;
  int sequences, width;
  long long tokens;
  int max_tokens, max_len;
};

struct CachePlace {
  int sequence;  // -1: the row is no sequence's, and is left as it is
  int position;  // negative: no place
};

__device__ __forceinline__ long long cache_start(const CacheParams& p, int s) {
  return p.starts == nullptr ? min(static_cast<long long>(s), p.tokens) : min(max(static_cast<long long>(__ldg(p.starts + s)), 0ll), p.tokens);
}
__device__ __forceinline__ int cache_len(const CacheParams& p, int s) { return min(max(__ldg(p.lens + s), 0), p.max_len); }

// The sequence and position of a row of the call's arrays.
__device__ __forceinline__ CachePlace cache_place(const CacheParams& p, long long token) {
  int s = 0;
  if (p.starts == nullptr) {
    s = static_cast<int>(min(token, static_cast<long long>(p.sequences)));
  } else {
    // the last sequence that starts at the row or before it (a search inside 0..sequences whatever the array holds)
    int most = p.sequences;
    if (cache_start(p, 0) > token) return {-1, -1};
    while (s < most) {
      const int mid = (s + most + 1) >> 1;
      if (cache_start(p, mid) <= token) s = mid;
      else most = mid - 1;
    }
  }
  if (s >= p.sequences) return {-1, -1};
  const long long first = cache_start(p, s), count = cache_start(p, s + 1) - first, at = token - first;
  if (at < 0 || at >= count || at >= p.max_tokens) return {-1, -1};
  return {s, static_cast<int>(max(cache_len(p, s) - count + at, -1ll))};
}

// The page of a position below the table's end, or -1.
__device__ __forceinline__ int cache_page(const CacheParams& p, int sequence, int position) {
  const int page = __ldg(p.table + static_cast<long long>(sequence) * p.width + (position >> p.page_shift));
  return page >= 0 && page < p.pages ? page : -1;
}

}  // namespace nb
