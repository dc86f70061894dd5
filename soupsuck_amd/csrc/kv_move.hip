// Rows of paged caches read back, and block tables that follow chosen beams.
//
// kv_read: the last rows of every sequence, as packed tokens: what append wrote, as the cache
// holds it.  Eight threads a (token, head), each with columns 8 c .. + 7 and 64 + 8 c .. + 7 of the
// key and of the value: 16-byte stores, and for a 4-bit cache one word of codes each.
//
// kv_fork: new row i continues old row p = parents[i].  Its full pages are p's own (shared from
// then on: nothing is appended to them), the page that p's next token goes to is spare[i], and
// the rows that p has there already are copied, for all layers in one launch: a workgroup
// takes 16 rows of one head, 8 KiB (16 bits) or a group (4 bits), in some of the layers.
// Parent, length and table entry are three dependent loads, and that latency is what a small
// fork costs: 28 layers of 4 beams 4.0 us; 32 beams of 4 heads (43 MB) 12 us.  Reading those
// rows back (98 MB) takes 21 us, 4.7 TB/s, in a workgroup for every layer: two of them one after
// the other took the same, and one layer's read longer.  Of 16 bits: four layers of 42976 tokens (704
// MB) 124 us, 5.7 TB/s; one of 6042 tokens (25 MB) 6.3.
#include "paged4.h"

namespace ss {
namespace {

constexpr int kCaches = 64;  // of a launch: their bases are arguments

struct Bases {
  char* k[kCaches];
  char* v[kCaches];
};

template <class T>
using Vec8 = T __attribute__((ext_vector_type(8)));

struct ReadArgs {
  CacheView cache;
  TableView rows;
  const int32_t* cu;
  int sequences;
  uint32_t items;  // tokens * kv heads
  char* k;         // [caches][tokens][kv heads][128]
  char* v;
  int64_t each;    // bytes of one cache's k
  Bases bases;
};

template <class T, bool FOUR>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a) {
  const uint32_t item = blockIdx.x * 32 + (threadIdx.x >> 3);
  if (item >= a.items) return;
  const int c = threadIdx.x & 7;
  const int hk = a.cache.kv_heads;
  const uint32_t t = item / (uint32_t)hk;
  const int h = (int)(item - t * (uint32_t)hk);
  u32x4 k[2] = {}, v[2] = {};
  const int b = a.sequences ? sequence_of(a.cu, a.sequences, t) : -1;
  const int64_t row = b < 0 ? -1 : (int64_t)a.rows.lengths[b] - a.cu[b + 1] + t;
  if (row >= 0) {
    const int64_t entry = row / a.cache.page_size, r = row - entry * a.cache.page_size;
    const int page = a.rows.page(b, entry, a.cache.pages);
    if (page >= 0) {
      const char* from = a.bases.k[blockIdx.y] + page * a.cache.k_page + h * a.cache.k_head;
      if constexpr (FOUR) {
        from += (r >> 4) * a.cache.k_row;
        const int in = (int)(r & 15);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int chunk = c + 8 * half, block = chunk >> 2;
          const auto* bytes = reinterpret_cast<const uint8_t*>(from);
          k[half] = decoded<T>(
              *reinterpret_cast<const uint32_t*>(from + key_at(in, block) + (chunk & 3) * 4),
              scale_of(bytes[kKeyScales + scale_at(in, block)]));
          v[half] = decoded<T>(*reinterpret_cast<const uint32_t*>(from + value_at(in, chunk)),
                               scale_of(bytes[kValueScales + scale_at(in, block)]));
        }
      } else {
        const char* from_v = a.bases.v[blockIdx.y] + page * a.cache.v_page + h * a.cache.v_head;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          k[half] = reinterpret_cast<const u32x4*>(from + r * a.cache.k_row)[c + 8 * half];
          v[half] = reinterpret_cast<const u32x4*>(from_v + r * a.cache.v_row)[c + 8 * half];
        }
      }
    }
  }
  const int64_t at = blockIdx.y * a.each + (int64_t)item * kCacheDim * 2;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    reinterpret_cast<u32x4*>(a.k + at)[c + 8 * half] = k[half];
    reinterpret_cast<u32x4*>(a.v + at)[c + 8 * half] = v[half];
  }
}

struct ForkArgs {
  CacheView cache;
  TableView rows;
  int old_rows;
  const int32_t* parents;
  const int32_t* spare;
  int32_t* out_table;
  int32_t* out_lengths;
  int new_rows;
  Bases bases;
};

template <bool FOUR>
__global__ __launch_bounds__(256) void kv_fork_kernel(ForkArgs a, int caches, int each,
                                                      bool tables) {
  const int pieces = a.cache.page_size / kGroupRows, hk = a.cache.kv_heads;
  const uint32_t unit = blockIdx.x / (uint32_t)pieces;
  const int piece = (int)(blockIdx.x - unit * pieces);
  const int i = (int)(unit / (uint32_t)hk), h = (int)(unit - (uint32_t)i * hk);
  const int parent = a.parents[i];
  const bool holds = parent >= 0 && parent < a.old_rows;
  const int length = holds ? (int)a.rows.length(parent, a.cache.page_size, INT64_MAX) : 0;
  const int full = length / a.cache.page_size, open = length - full * a.cache.page_size;
  const int spare = a.spare[i];
  const int from = open ? a.rows.page(parent, full, a.cache.pages) : -1;
  if (tables && blockIdx.y == 0 && h == 0 && piece == 0) {
    // Rows on a page that the parent does not hold are not held by its successor either.
    const int next = open && from < 0 ? -1 : spare;
    for (int e = threadIdx.x; e < a.rows.row_pages; e += 256)
      a.out_table[(int64_t)i * a.rows.row_pages + e] =
          e < full ? a.rows.table[parent * a.rows.stride + e] : e == full ? next : -1;
    if (threadIdx.x == 0) a.out_lengths[i] = length;
  }
  if (from < 0 || spare < 0 || spare >= a.cache.pages || piece * kGroupRows >= open) return;
  const int first = blockIdx.y * each, last = min(first + each, caches);
  if constexpr (FOUR) {
    constexpr int kParts = kGroupBytes / 16;
    const int64_t at = h * a.cache.k_head + piece * a.cache.k_row;
    const int64_t source = at + from * a.cache.k_page, target = at + spare * a.cache.k_page;
#pragma unroll 4
    for (int item = threadIdx.x; item < (last - first) * kParts; item += 256) {
      char* base = a.bases.k[first + item / kParts] + item % kParts * 16;
      *reinterpret_cast<u32x4*>(base + target) = *reinterpret_cast<const u32x4*>(base + source);
    }
  } else {
    const int r = piece * kGroupRows + (threadIdx.x >> 4), c = (threadIdx.x & 15) * 16;
    if (r >= open) return;
    const int64_t at_k = h * a.cache.k_head + r * a.cache.k_row + c;
    const int64_t at_v = h * a.cache.v_head + r * a.cache.v_row + c;
#pragma unroll 4
    for (int cache = first; cache < last; ++cache) {
      char *k = a.bases.k[cache] + at_k, *v = a.bases.v[cache] + at_v;
      const u32x4 x = *reinterpret_cast<const u32x4*>(k + from * a.cache.k_page);
      const u32x4 y = *reinterpret_cast<const u32x4*>(v + from * a.cache.v_page);
      *reinterpret_cast<u32x4*>(k + spare * a.cache.k_page) = x;
      *reinterpret_cast<u32x4*>(v + spare * a.cache.v_page) = y;
    }
  }
}

bool alike(const CacheView& a, const CacheView& b) {
  return a.k_page == b.k_page && a.k_head == b.k_head && a.k_row == b.k_row &&
         a.v_page == b.v_page && a.v_head == b.v_head && a.v_row == b.v_row &&
         a.pages == b.pages && a.page_size == b.page_size && a.kv_heads == b.kv_heads;
}

// The checks of the caches of a call: each by itself, and alike.
template <class Cache>
int check_caches(const char* who, const Cache* const* caches, int count) {
  SS_CHECK_ARG(caches && count > 0, "%s: needs a cache", who);
  for (int i = 0; i < count; ++i) {
    if (const int rc = check_cache(who, caches[i])) return rc;
    SS_CHECK_ARG(caches[i]->dtype == caches[0]->dtype &&
                     alike(cache_view(caches[i]), cache_view(caches[0])),
                 "%s: cache %d is not like the first", who, i);
  }
  return SS_OK;
}

// Calls f(bases, first cache, caches) for as many caches as a launch takes, and then the next.
template <class Cache, class F>
int in_launches(const Cache* const* caches, int count, F f) {
  for (int first = 0; first < count; first += kCaches) {
    const int n = count - first < kCaches ? count - first : kCaches;
    Bases bases{};
    for (int i = 0; i < n; ++i) {
      const CacheView view = cache_view(caches[first + i]);
      bases.k[i] = view.k;
      bases.v[i] = view.v;
    }
    if (const int rc = f(bases, first, n)) return rc;
  }
  return SS_OK;
}

template <bool FOUR, class Cache>
int read(const char* who, const Cache* const* caches, int count, const int32_t* table,
         int64_t table_stride, int row_pages, const int32_t* lengths, const int32_t* cu_seqlens,
         int rows, int64_t tokens, void* k, void* v, void* stream) {
  if (const int rc = check_caches(who, caches, count)) return rc;
  const Cache* cache = caches[0];
  if (const int rc = check_table(who, cache, table, table_stride, row_pages, lengths, rows))
    return rc;
  SS_CHECK_ARG(tokens >= 0, "%s: negative token count", who);
  if (tokens == 0) return SS_OK;
  SS_CHECK_ARG(k && v && (rows == 0 || cu_seqlens), "%s: null pointer", who);
  SS_CHECK_ARG(aligned16(k) && aligned16(v), "%s: needs 16-byte aligned outputs", who);
  SS_CHECK_ARG(tokens <= INT64_MAX / cache->kv_heads &&
                   fits_grid(tokens * cache->kv_heads, 32, 256),
               "%s: too many rows in one call", who);
  const int64_t each = tokens * cache->kv_heads * kCacheDim * 2;
  const hipStream_t st = (hipStream_t)stream;
  return in_launches(caches, count, [&](const Bases& bases, int first, int n) -> int {
    ReadArgs a{cache_view(cache), TableView{table, table_stride, row_pages, lengths}, cu_seqlens,
               rows, (uint32_t)(tokens * cache->kv_heads), (char*)k + first * each,
               (char*)v + first * each, each, bases};
    const dim3 grid((unsigned)cdiv(a.items, 32), (unsigned)n), block(256);
    if (cache->dtype == SS_F16)
      hipLaunchKernelGGL((kv_read_kernel<half_t, FOUR>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((kv_read_kernel<bhalf_t, FOUR>), grid, block, 0, st, a);
    SS_CHECK_LAUNCH("kv_read_kernel");
    return SS_OK;
  });
}

template <bool FOUR, class Cache>
int fork(const char* who, const Cache* const* caches, int count, const int32_t* table,
         int64_t table_stride, int row_pages, const int32_t* lengths, int rows,
         const int32_t* parents, const int32_t* spare, int new_rows, int32_t* out_table,
         int32_t* out_lengths, void* stream) {
  if (const int rc = check_caches(who, caches, count)) return rc;
  const Cache* cache = caches[0];
  if (const int rc = check_table(who, cache, table, table_stride, row_pages, lengths, rows))
    return rc;
  SS_CHECK_ARG(new_rows >= 0, "%s: negative row count", who);
  if (new_rows == 0) return SS_OK;
  SS_CHECK_ARG(parents && spare && out_table && out_lengths, "%s: null pointer", who);
  const int64_t units = (int64_t)new_rows * cache->kv_heads * (cache->page_size / kGroupRows);
  SS_CHECK_ARG(fits_grid(units, 1, 256), "%s: too many rows in one call", who);
  const hipStream_t st = (hipStream_t)stream;
  return in_launches(caches, count, [&](const Bases& bases, int first, int n) -> int {
    ForkArgs a{cache_view(cache), TableView{table, table_stride, row_pages, lengths}, rows,
               parents, spare, out_table, out_lengths, new_rows, bases};
    // Four caches a workgroup, whose loads are on their way at once, where that leaves every CU
    // eight: 32 beams of 28 layers 20.7, 12.0, 13.8, 14.8 and 16.4 us with 1, 4, 7, 14 and 28.
    const int64_t most = units * n / (8 * (int64_t)device_cu_count());
    const int each = (int)(most < 1 ? 1 : most < 4 ? most : 4);
    hipLaunchKernelGGL((kv_fork_kernel<FOUR>), dim3((unsigned)units, (unsigned)cdiv(n, each)),
                       dim3(256), 0, st, a, n, each, first == 0);
    SS_CHECK_LAUNCH("kv_fork_kernel");
    return SS_OK;
  });
}

}  // namespace
}  // namespace ss

extern "C" int ss_kv_read(const ss_paged_cache* const* caches, int count, const int32_t* table,
                          int64_t table_stride, int row_pages, const int32_t* lengths,
                          const int32_t* cu_seqlens, int rows, int64_t tokens, void* k, void* v,
                          void* stream) {
  return ss::read<false>("ss_kv_read", caches, count, table, table_stride, row_pages, lengths,
                         cu_seqlens, rows, tokens, k, v, stream);
}

extern "C" int ss_kv_read4(const ss_paged_cache4* const* caches, int count, const int32_t* table,
                           int64_t table_stride, int row_pages, const int32_t* lengths,
                           const int32_t* cu_seqlens, int rows, int64_t tokens, void* k, void* v,
                           void* stream) {
  return ss::read<true>("ss_kv_read4", caches, count, table, table_stride, row_pages, lengths,
                        cu_seqlens, rows, tokens, k, v, stream);
}

extern "C" int ss_kv_fork(const ss_paged_cache* const* caches, int count, const int32_t* table,
                          int64_t table_stride, int row_pages, const int32_t* lengths, int rows,
                          const int32_t* parents, const int32_t* spare, int new_rows,
                          int32_t* out_table, int32_t* out_lengths, void* stream) {
  return ss::fork<false>("ss_kv_fork", caches, count, table, table_stride, row_pages, lengths,
                         rows, parents, spare, new_rows, out_table, out_lengths, stream);
}

extern "C" int ss_kv_fork4(const ss_paged_cache4* const* caches, int count, const int32_t* table,
                           int64_t table_stride, int row_pages, const int32_t* lengths, int rows,
                           const int32_t* parents, const int32_t* spare, int new_rows,
                           int32_t* out_table, int32_t* out_lengths, void* stream) {
  return ss::fork<true>("ss_kv_fork4", caches, count, table, table_stride, row_pages, lengths,
                        rows, parents, spare, new_rows, out_table, out_lengths, stream);
}
