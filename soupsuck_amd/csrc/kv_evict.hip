// Eviction from a paged cache by accumulated attention weight.
//
// Per (sequence, kv head): rows below lo = min(sinks, length) and from hi = max(lo, length
// - recent) on stay, and of the rows between them the m = budget - lo - (length - hi)
// heaviest, equal weights from the lowest row up.
//
// Selection (one workgroup of 16 waves per (sequence, kv head)): the m-th largest weight
// by its bits, 11 at a time from the top: a histogram of the digit among the rows that
// agree with the digits found so far, then the bin that holds the m-th, found by one wave
// (32 bins a lane, then the lane's own 32).  Counts are whole numbers, so LDS atomics give
// the same result in any order.  Then each wave counts the rows above and at the threshold
// in its part, a scan over the waves gives its first place, and a second walk over its part
// writes the kept rows' numbers in order.  The five walks are latency: 5.5 us for 1281 rows
// (37.7 with 8-bit digits and a serial search), 12 us for 128 lines of up to 8191; up to
// kStaged rows they read keys that the first one left in LDS.
// Copy: 16 lanes a kept row, 16 bytes of k and of v each, HBM-bound: 490 MB in 99 us, the
// rate of a large copy.
#include "paged.h"

namespace ss {
namespace {

constexpr int kWaves = 16;
constexpr int kBins = 2048;
constexpr int kStaged = 16384;  // rows whose keys LDS holds (64 KiB)

struct EvictArgs {
  CacheView cache;
  TableView rows;
  int sequences;
  int64_t max_length;
  const float* w;
  const int32_t* out_table;
  int64_t out_stride;
  int out_pages;
  int64_t budget, sinks, recent;
  int32_t* out_lengths;
  float* out_w;
  int32_t* kept;  // [sequences][kv_heads][budget]
};

// Order of the weights as whole numbers; NaN is the heaviest, the zeros are equal.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sums over the lanes up to and with each.
template <int CTRL, int ROWS>
__device__ __forceinline__ int add_moved(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int lanes_upto(int v) {
  v = add_moved<0x111, 0xf>(v);  // lanes 1, 2, 4, 8 below in the row
  v = add_moved<0x112, 0xf>(v);
  v = add_moved<0x114, 0xf>(v);
  v = add_moved<0x118, 0xf>(v);
  v = add_moved<0x142, 0xa>(v);  // the last lane of rows 0 and 2 to rows 1 and 3
  return add_moved<0x143, 0xc>(v);  // and of row 1 to rows 2 and 3
}

struct Digit {
  int bin, above;  // the need-th row from the top lies in this bin, with so many in higher ones
};
// By one wave: lane l takes the 32 bins below bin 2048 - 32 l, then those of the lane that
// the row lies in.
__device__ __forceinline__ Digit find_digit(const uint32_t* bins, int need) {
  const int lane = threadIdx.x & 63;
  int sum = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const u32x4 v = reinterpret_cast<const u32x4*>(bins)[(63 - lane) * 8 + i];
    sum += (int)(v[0] + v[1] + v[2] + v[3]);
  }
  const int upto = lanes_upto(sum);
  const int at = __ffsll((long long)__ballot(upto >= need)) - 1;
  const int before = __builtin_amdgcn_readlane(upto - sum, at);
  const int bin = (63 - at) * 32 + 31 - (lane & 31);
  const int mine = lane < 32 ? (int)bins[bin] : 0;
  const int inside = before + lanes_upto(mine);
  const int hit = __ffsll((long long)__ballot(inside >= need)) - 1;
  return Digit{__builtin_amdgcn_readlane(bin, hit), __builtin_amdgcn_readlane(inside - mine, hit)};
}

__global__ __launch_bounds__(kWaves * 64) void kv_select_kernel(EvictArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t bins[kBins];
  __shared__ uint32_t keys[kStaged];
  __shared__ Digit found;
  __shared__ int counts[2][kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int head = blockIdx.x % a.cache.kv_heads;
  const int b = blockIdx.x / a.cache.kv_heads;
  const int len = (int)a.rows.length(b, a.cache.page_size, a.max_length);
  const int keep = (int)(len < a.budget ? len : a.budget);
  if (head == 0 && threadIdx.x == 0) a.out_lengths[b] = keep;
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.budget;
  if (len <= a.budget) {
    for (int j = threadIdx.x; j < len; j += kWaves * 64) kept[j] = j;
    return;
  }
  // sinks + recent <= budget < len
  const int lo = (int)a.sinks, hi = len - (int)a.recent;
  const int want = keep - lo - (len - hi);
  const float* w = a.w + (int64_t)blockIdx.x * a.rows.row_pages * a.cache.page_size;
  const bool staged = hi - lo <= kStaged;
  auto key_of = [&](int j) { return staged ? keys[j - lo] : weight_key(w[j]); };
  uint32_t threshold = 0;
  int need = want;  // of the rows that agree with the digits found
  if (want == 0) {
    threshold = 0xFFFFFFFFu;  // no key is larger, and none at it is needed
  } else {
    // Digits of 11, 11 and 10 bits.
#pragma unroll
    for (int shift = 21; shift >= 0; shift -= shift == 21 ? 11 : 10) {
      for (int i = threadIdx.x; i < kBins; i += kWaves * 64) bins[i] = 0;
      __syncthreads();
      const uint32_t mask = shift == 21 ? 0u : ~0u << (shift == 10 ? 21 : 10);
      const uint32_t digit = shift == 0 ? 1023u : 2047u;
      for (int j = lo + threadIdx.x; j < hi; j += kWaves * 64) {
        uint32_t key;
        if (shift == 21) {
          key = weight_key(w[j]);
          if (staged) keys[j - lo] = key;
        } else {
          key = key_of(j);
        }
        if ((key & mask) == threshold) atomicAdd(&bins[(key >> shift) & digit], 1u);
      }
      __syncthreads();
      if (wave == 0) {
        const Digit d = find_digit(bins, need);
        if (lane == 0) found = d;
      }
      __syncthreads();
      threshold |= (uint32_t)found.bin << shift;
      need -= found.above;
    }
  }
  // Rows above the threshold, and the first `need` at it.
  const int span = (int)cdiv(cdiv(hi - lo, kWaves), 64) * 64;
  const int from = lo + wave * span, to = min(hi, from + span);
  int above = 0, equal = 0;
  if (want > 0)
    for (int j0 = from; j0 < to; j0 += 64) {
      const uint32_t key = j0 + lane < to ? key_of(j0 + lane) : 0;
      above += __popcll(__ballot(j0 + lane < to && key > threshold));
      equal += __popcll(__ballot(j0 + lane < to && key == threshold));
    }
  if (lane == 0) counts[0][wave] = above, counts[1][wave] = equal;
  __syncthreads();
  int above_before = 0, equal_before = 0;
  for (int i = 0; i < wave; ++i) {
    above_before += counts[0][i];
    equal_before += counts[1][i];
  }
  const uint64_t below = (1ull << lane) - 1;
  if (want > 0)
    for (int j0 = from; j0 < to; j0 += 64) {
      const int j = j0 + lane;
      const uint32_t key = j < to ? key_of(j) : 0;
      const uint64_t gt = __ballot(j < to && key > threshold);
      const uint64_t eq = __ballot(j < to && key == threshold);
      const int ga = above_before + __popcll(gt & below), ea = equal_before + __popcll(eq & below);
      if (j < to && (key > threshold || (key == threshold && ea < need)))
        kept[lo + ga + min(ea, need)] = j;
      above_before += __popcll(gt);
      equal_before += __popcll(eq);
    }
  for (int j = threadIdx.x; j < lo; j += kWaves * 64) kept[j] = j;
  for (int j = threadIdx.x; j < len - hi; j += kWaves * 64) kept[lo + want + j] = hi + j;
}

__global__ __launch_bounds__(256) void kv_copy_kernel(EvictArgs a) {
  const int64_t cap = (int64_t)a.out_pages * a.cache.page_size;
  const int64_t item = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int c = threadIdx.x & 15;
  if (item >= cap * a.sequences * a.cache.kv_heads) return;
  const int64_t i = item % cap;
  const int64_t line = item / cap;
  const int head = (int)(line % a.cache.kv_heads);
  const int b = (int)(line / a.cache.kv_heads);
  const int64_t len = a.rows.length(b, a.cache.page_size, a.max_length);
  const int64_t keep = len < a.budget ? len : a.budget;
  if (i >= keep) {
    if (c == 0) a.out_w[item] = 0.f;
    return;
  }
  const int size = a.cache.page_size;
  const int j = a.kept[line * a.budget + i];
  if (c == 0) a.out_w[item] = a.w[line * a.rows.row_pages * size + j];
  const int from = a.rows.page(b, j / size, a.cache.pages);
  const int to = a.out_table[(int64_t)b * a.out_stride + i / size];
  if (to < 0 || to >= a.cache.pages) return;
  // Past the caches both ways (a row is moved once): 32 sequences halved 109 -> 98 us.
  u32x4 k{}, v{};
  if (from >= 0) {
    const char* row = a.cache.k + from * a.cache.k_page + head * a.cache.k_head;
    k = __builtin_nontemporal_load(
        &reinterpret_cast<const u32x4*>(row + j % size * a.cache.k_row)[c]);
    row = a.cache.v + from * a.cache.v_page + head * a.cache.v_head;
    v = __builtin_nontemporal_load(
        &reinterpret_cast<const u32x4*>(row + j % size * a.cache.v_row)[c]);
  }
  char* row = a.cache.k + to * a.cache.k_page + head * a.cache.k_head;
  __builtin_nontemporal_store(k, &reinterpret_cast<u32x4*>(row + i % size * a.cache.k_row)[c]);
  row = a.cache.v + to * a.cache.v_page + head * a.cache.v_head;
  __builtin_nontemporal_store(v, &reinterpret_cast<u32x4*>(row + i % size * a.cache.v_row)[c]);
}

}  // namespace
}  // namespace ss

extern "C" size_t ss_kv_evict_workspace_size(int rows, int kv_heads, int64_t budget) {
  if (rows <= 0 || kv_heads <= 0 || budget <= 0) return 0;
  return (size_t)rows * kv_heads * budget * sizeof(int32_t);
}

extern "C" int ss_kv_evict(const ss_paged_cache* cache, const int32_t* table,
                           int64_t table_stride, int row_pages, const int32_t* lengths, int rows,
                           int64_t max_length, const float* weights, const int32_t* out_table,
                           int64_t out_stride, int out_pages, int64_t budget, int64_t sinks,
                           int64_t recent, int32_t* out_lengths, float* out_weights,
                           void* workspace, size_t workspace_bytes, void* stream) {
  using namespace ss;
  const char* who = "ss_kv_evict";
  if (const int rc = check_cache(who, cache)) return rc;
  if (const int rc = check_table(who, cache, table, table_stride, row_pages, lengths, rows))
    return rc;
  SS_CHECK_ARG(max_length >= 0, "%s: negative max_length", who);
  SS_CHECK_ARG(sinks >= 0 && recent >= 0 && budget > 0 && sinks <= budget &&
                   recent <= budget - sinks,
               "%s: sinks %lld and recent %lld must fit the budget %lld", who, (long long)sinks,
               (long long)recent, (long long)budget);
  SS_CHECK_ARG(out_pages > 0 && out_stride >= out_pages &&
                   (int64_t)out_pages * cache->page_size >= budget &&
                   (int64_t)out_pages * cache->page_size <= INT32_MAX,
               "%s: %d pages a row do not hold the budget %lld", who, out_pages,
               (long long)budget);
  if (rows == 0) return SS_OK;
  SS_CHECK_ARG(weights && out_table && out_lengths && out_weights, "%s: null pointer", who);
  const size_t need = ss_kv_evict_workspace_size(rows, cache->kv_heads, budget);
  SS_CHECK_ARG(need <= workspace_bytes && workspace && aligned16(workspace),
               "%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, need);
  const int64_t lines = (int64_t)rows * cache->kv_heads;
  const int64_t items = (int64_t)out_pages * cache->page_size * lines;
  SS_CHECK_ARG(fits_grid(lines, 1, kWaves * 64) && fits_grid(items, 16, 256), "%s: too many rows",
               who);
  EvictArgs a{cache_view(cache), TableView{table, table_stride, row_pages, lengths}, rows,
              max_length, weights, out_table, out_stride, out_pages, budget, sinks, recent,
              out_lengths, out_weights, (int32_t*)workspace};
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(kv_select_kernel, dim3((unsigned)lines), dim3(kWaves * 64), 0, st, a);
  SS_CHECK_LAUNCH("kv_select_kernel");
  hipLaunchKernelGGL(kv_copy_kernel, dim3((unsigned)cdiv(items, 16)), dim3(256), 0, st, a);
  SS_CHECK_LAUNCH("kv_copy_kernel");
  return SS_OK;
}
