// New tokens into the paged cache: keys rotated, values copied, queries rotated.
//
// Rows are (token, head), q heads first, then k, then v: one launch does what the
// rotation, two scattered copies and their index arithmetic would do in several.
// Rotation: y[c] = x[c] cos[c] - x[c + 64] sin[c], y[c + 64] = x[c + 64] cos[c + 64]
// + x[c] sin[c + 64], products and sum in fp32, rounded once to the cache's type (the
// training rotation rounds each product as well; here a key is stored once and read
// for the rest of the sequence).
//
// Eight threads a row, each with 8 columns of the low half and the 8 that they turn
// with (16-byte loads and stores).  HBM-bound for prompts: 6042 tokens of 28 / 4 heads (114
// MB) in 21.5 us, 5.3 TB/s.  A single token is latency (2.7 us): offsets, length and table
// entry are three dependent loads.
#include "paged.h"

namespace ss {
namespace {

struct AppendArgs {
  CacheView cache;
  TableView rows;
  const int32_t* cu;
  int sequences;
  uint32_t items;  // tokens * heads
  const char* k; int64_t k_tok, k_head;  // bytes
  const char* v; int64_t v_tok, v_head;
  const char* q; int64_t q_tok, q_head;
  const char* cos; int64_t cos_tok;
  const char* sin; int64_t sin_tok;
  char* qo; int64_t qo_tok, qo_head;
  int hq, heads;  // q heads (0: none); q + 2 kv heads
};

template <class T>
using Vec8 = T __attribute__((ext_vector_type(8)));

template <class CS>
__device__ __forceinline__ void load_angles(const char* p, int c, float (&out)[8]) {
  const Vec8<CS> v = *reinterpret_cast<const Vec8<CS>*>(p + c * sizeof(CS));
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = (float)v[e];
}

template <class T, class CS>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
  const uint32_t item = blockIdx.x * 32 + (threadIdx.x >> 3);
  if (item >= a.items) return;
  const int c = (threadIdx.x & 7) * 8;
  const uint32_t t = item / (uint32_t)a.heads;
  const int head = (int)(item - t * (uint32_t)a.heads);
  const int hk = a.cache.kv_heads;
  const bool is_q = head < a.hq, is_k = !is_q && head < a.hq + hk;
  const int h = is_q ? head : is_k ? head - a.hq : head - a.hq - hk;
  const char* from = is_q   ? a.q + t * a.q_tok + h * a.q_head
                     : is_k ? a.k + t * a.k_tok + h * a.k_head
                            : a.v + t * a.v_tok + h * a.v_head;
  Vec8<T> lo = reinterpret_cast<const Vec8<T>*>(from)[c / 8];
  Vec8<T> hi = reinterpret_cast<const Vec8<T>*>(from)[c / 8 + 8];
  if (a.cos && (is_q || is_k)) {
    float c1[8], c2[8], s1[8], s2[8];
    load_angles<CS>(a.cos + t * a.cos_tok, c, c1);
    load_angles<CS>(a.cos + t * a.cos_tok, c + 64, c2);
    load_angles<CS>(a.sin + t * a.sin_tok, c, s1);
    load_angles<CS>(a.sin + t * a.sin_tok, c + 64, s2);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = (float)lo[e], y = (float)hi[e];
      lo[e] = (T)(x * c1[e] - y * s1[e]);
      hi[e] = (T)(y * c2[e] + x * s2[e]);
    }
  }
  char* to;
  if (is_q) {
    to = a.qo + t * a.qo_tok + h * a.qo_head;
  } else {
    if (a.sequences == 0) return;
    const int b = sequence_of(a.cu, a.sequences, t);
    if (b < 0) return;
    // Row of the token: the sequence's own tokens are its last ones.
    const int64_t row = (int64_t)a.rows.lengths[b] - a.cu[b + 1] + t;
    if (row < 0) return;
    const int64_t entry = row / a.cache.page_size;
    const int page = a.rows.page(b, entry, a.cache.pages);
    if (page < 0) return;
    const int64_t r = row - entry * a.cache.page_size;
    to = is_k ? a.cache.k + page * a.cache.k_page + h * a.cache.k_head + r * a.cache.k_row
              : a.cache.v + page * a.cache.v_page + h * a.cache.v_head + r * a.cache.v_row;
  }
  reinterpret_cast<Vec8<T>*>(to)[c / 8] = lo;
  reinterpret_cast<Vec8<T>*>(to)[c / 8 + 8] = hi;
}

}  // namespace
}  // namespace ss

extern "C" int ss_kv_append(const ss_paged_cache* cache, const void* k, int64_t k_tok,
                            int64_t k_head, const void* v, int64_t v_tok, int64_t v_head,
                            const void* q, int64_t q_tok, int64_t q_head, int q_heads,
                            const void* cos, int64_t cos_tok, const void* sin, int64_t sin_tok,
                            int cs_dtype, const int32_t* table, int64_t table_stride,
                            int row_pages, const int32_t* lengths, const int32_t* cu_seqlens,
                            int rows, int64_t tokens, void* q_out, int64_t qo_tok,
                            int64_t qo_head, void* stream) {
  using namespace ss;
  const char* who = "ss_kv_append";
  if (const int rc = check_cache(who, cache)) return rc;
  if (const int rc = check_table(who, cache, table, table_stride, row_pages, lengths, rows))
    return rc;
  SS_CHECK_ARG(tokens >= 0, "%s: negative token count", who);
  if (tokens == 0) return SS_OK;
  SS_CHECK_ARG(k && v && (rows == 0 || cu_seqlens), "%s: null pointer", who);
  SS_CHECK_ARG((q == nullptr) == (q_out == nullptr) && (!q || q_heads > 0),
               "%s: q and q_out go together", who);
  SS_CHECK_ARG((cos == nullptr) == (sin == nullptr), "%s: cos and sin go together", who);
  SS_CHECK_ARG(!q || cos, "%s: q is given only to be rotated", who);
  SS_CHECK_ARG(!cos || cs_dtype == SS_F32 || cs_dtype == cache->dtype,
               "%s: cos / sin must be fp32 or of the cache's type", who);
  SS_CHECK_ARG(aligned16(k) && aligned16(v) && aligned16(q) && aligned16(q_out) &&
                   aligned16(cos) && aligned16(sin) &&
                   ((k_tok | k_head | v_tok | v_head) & 7) == 0 &&
                   (!q || ((q_tok | q_head | qo_tok | qo_head) & 7) == 0) &&
                   (!cos || ((cos_tok | sin_tok) & (cs_dtype == SS_F32 ? 3 : 7)) == 0),
               "%s: needs 16-byte aligned bases and strides that are multiples of 8", who);
  const int hq = q ? q_heads : 0;
  const int64_t heads = (int64_t)hq + 2 * (int64_t)cache->kv_heads;
  SS_CHECK_ARG(heads <= INT32_MAX && tokens <= (int64_t)INT32_MAX / heads,
               "%s: too many rows in one call", who);
  const int cs = cs_dtype == SS_F32 ? 4 : 2;
  AppendArgs a{cache_view(cache), TableView{table, table_stride, row_pages, lengths},
               cu_seqlens, rows, (uint32_t)(tokens * heads),
               (const char*)k, k_tok * 2, k_head * 2, (const char*)v, v_tok * 2, v_head * 2,
               (const char*)q, q_tok * 2, q_head * 2, (const char*)cos, cos_tok * cs,
               (const char*)sin, sin_tok * cs, (char*)q_out, qo_tok * 2, qo_head * 2, hq,
               (int)heads};
  const dim3 grid((unsigned)cdiv(tokens * heads, 32)), block(256);
  const hipStream_t st = (hipStream_t)stream;
  const bool wide = cos && cs_dtype == SS_F32;
  if (cache->dtype == SS_F16) {
    if (wide) hipLaunchKernelGGL((kv_append_kernel<half_t, float>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((kv_append_kernel<half_t, half_t>), grid, block, 0, st, a);
  } else {
    if (wide) hipLaunchKernelGGL((kv_append_kernel<bhalf_t, float>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((kv_append_kernel<bhalf_t, bhalf_t>), grid, block, 0, st, a);
  }
  SS_CHECK_LAUNCH("kv_append_kernel");
  return SS_OK;
}
