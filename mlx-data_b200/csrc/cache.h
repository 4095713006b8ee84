// A cache of keys and values in pages, as its kernels see it.
#pragma once

#include "attention.h"

namespace mlxd {

struct CacheParams {
  const void* table;
  const void* lengths;
  const void* counts;           // null: every token of a call
  int64_t table_stride;
  int table_width, pages, page_size, page_shift, capacity;   // capacity: places that a row of the table has
  int table_dtype, lengths_dtype, counts_dtype;
};

constexpr int kMaxPlaces = 1 << 30;

inline Heads pages_of(const mlxd_pages& x) {
  return Heads{static_cast<char*>(x.data), x.stride_page, x.stride_row, x.stride_head};
}

// Checks a cache and takes what its kernels need; the pools themselves are the caller's to check.
int cache_of(const char* entry, const mlxd_cache& c, int batch, CacheParams* p);

#ifdef __CUDACC__
__device__ __forceinline__ int64_t integer_at(const void* x, int dtype, int64_t i) {
  return dtype == MLXD_I64 ? static_cast<const int64_t*>(x)[i] : static_cast<const int32_t*>(x)[i];
}

// Tokens that lie in the cache before the call.
__device__ __forceinline__ int length_of(const CacheParams& p, int b) {
  const int64_t n = integer_at(p.lengths, p.lengths_dtype, b);
  return static_cast<int>(n < 0 ? 0 : n > kMaxPlaces ? kMaxPlaces : n);
}

// New ones.
__device__ __forceinline__ int count_of(const CacheParams& p, int b, int tokens) {
  if (!p.counts) return tokens;
  const int64_t n = integer_at(p.counts, p.counts_dtype, b);
  return static_cast<int>(n < 0 ? 0 : n > tokens ? tokens : n);
}

// The page of an entry of the table, -1 where it is none.
__device__ __forceinline__ int page_at(const CacheParams& p, int b, int entry) {
  const int64_t page = integer_at(p.table, p.table_dtype, b * p.table_stride + entry);
  return page < 0 || page >= p.pages ? -1 : static_cast<int>(page);
}

__device__ __forceinline__ int page_of(const CacheParams& p, int b, int place) {
  return place < p.capacity ? page_at(p, b, place >> p.page_shift) : -1;
}
#endif

}  // namespace mlxd
