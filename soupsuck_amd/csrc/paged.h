// Shared parts of the paged key-value cache kernels: element types, the cache's
// rows, and the host checks that every entry point makes before it launches.
#pragma once

#include "common.h"

namespace ss {

typedef __bf16 bhalf_t;

constexpr int kCacheDim = 128;  // head dimension

// A cache as the kernels see it: element strides, rows found through a block table.
struct CacheView {
  char* k;
  int64_t k_page, k_head, k_row;  // bytes
  char* v;
  int64_t v_page, v_head, v_row;
  int pages, page_size, kv_heads;
};

struct TableView {
  const int32_t* table;
  int64_t stride;
  int row_pages;
  const int32_t* lengths;

  // Rows that sequence b holds, at most `limit`.
  __device__ __forceinline__ int64_t length(int b, int page_size, int64_t limit) const {
    const int64_t cap = (int64_t)row_pages * page_size;
    const int64_t n = lengths[b];
    const int64_t top = cap < limit ? cap : limit;
    return n < 0 ? 0 : n < top ? n : top;
  }
  // Page of table entry i of sequence b, or -1 where it holds none.
  __device__ __forceinline__ int page(int b, int64_t i, int pages) const {
    if (i < 0 || i >= row_pages) return -1;
    const int p = table[(int64_t)b * stride + i];
    return p >= 0 && p < pages ? p : -1;
  }
};

// Sequence of packed token t: cu[b] <= t < cu[b + 1], or -1 (offsets that are not
// nondecreasing find a sequence that does not contain t, or one that does).
__device__ __forceinline__ int sequence_of(const int32_t* cu, int rows, int64_t t) {
  int lo = 0, hi = rows - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return cu[lo] <= t && t < cu[lo + 1] ? lo : -1;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

inline CacheView cache_view(const ss_paged_cache* c) {
  return CacheView{(char*)c->k, c->k_page * 2, c->k_head * 2, c->k_row * 2,
                   (char*)c->v, c->v_page * 2, c->v_head * 2, c->v_row * 2,
                   c->pages,    c->page_size,  c->kv_heads};
}

// What every cache entry point asks of the cache and the table.
inline int check_cache(const char* who, const ss_paged_cache* c) {
  SS_CHECK_ARG(c && c->k && c->v, "%s: null cache", who);
  SS_CHECK_ARG(c->dtype == SS_F16 || c->dtype == SS_BF16, "%s: cache dtype must be fp16 or bf16",
               who);
  SS_CHECK_ARG(c->head_dim == kCacheDim, "%s: head_dim %d, expected 128", who, c->head_dim);
  SS_CHECK_ARG(c->pages > 0 && c->kv_heads > 0, "%s: cache without pages or heads", who);
  SS_CHECK_ARG(c->page_size > 0 && c->page_size % 16 == 0,
               "%s: page_size %d must be a multiple of 16", who, c->page_size);
  SS_CHECK_ARG(aligned16(c->k) && aligned16(c->v) &&
                   ((c->k_page | c->k_head | c->k_row | c->v_page | c->v_head | c->v_row) & 7) == 0,
               "%s: cache needs 16-byte aligned bases and strides that are multiples of 8", who);
  return SS_OK;
}

inline int check_table(const char* who, const ss_paged_cache* c, const int32_t* table,
                       int64_t stride, int row_pages, const int32_t* lengths, int rows) {
  SS_CHECK_ARG(rows >= 0 && row_pages > 0 && stride >= row_pages,
               "%s: bad block table sizes (rows %d, pages a row %d, stride %lld)", who, rows,
               row_pages, (long long)stride);
  SS_CHECK_ARG(rows == 0 || (table && lengths), "%s: null block table or lengths", who);
  SS_CHECK_ARG((int64_t)row_pages * c->page_size <= INT32_MAX - 2048, "%s: a row holds %lld rows", who,
               (long long)row_pages * c->page_size);
  return SS_OK;
}

}  // namespace ss
