// Attention of new tokens over a paged key-value cache.
//
// o = sum_j softmax_j(scale q . k_j) v_j over the rows j that the token at row p sees
// (j <= p, and inside the window or among the sinks), with a running maximum and sum in
// fp32: m' = max(m, s), l' = l 2^(m - m') + 2^(s - m'), o' likewise, in base-2 scores.
//
// One workgroup per (token, q head): its four waves take every fourth visible row, a
// lane holds two of the 128 columns; the waves' (m, l, o) are joined at the end.  The
// weights are a second pass over the keys with the joined statistics.
#include "paged.h"
#include "elementwise.h"

namespace ss {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct CachedAttnArgs {
  CacheView cache;
  TableView rows;
  const int32_t* cu;
  int sequences;
  int64_t tokens, max_length;
  const char* q; int64_t q_tok, q_head;  // bytes
  char* o; int64_t o_tok, o_head;
  int hq, group;
  float scale_log2;
  int64_t window, sinks;
  const float* w_in;
  float* w_out;
  float* lse2;  // [tokens][hq], base 2
};

__device__ __forceinline__ bool visible(const CachedAttnArgs& a, int64_t j, int64_t at) {
  return j <= at && (a.window == 0 || j > at - a.window || j < a.sinks);
}

template <class T>
__device__ __forceinline__ float dot_row(const char* row, int lane, float q0, float q1) {
  const T* p = reinterpret_cast<const T*>(row) + 2 * lane;
  return wave_sum((float)p[0] * q0 + (float)p[1] * q1);
}

template <class T>
__global__ __launch_bounds__(256) void cached_attention_kernel(CachedAttnArgs a) {
  __shared__ float part[4][130];
  const int64_t t = blockIdx.x / a.hq;
  const int head = (int)(blockIdx.x - t * a.hq);
  const int kv = head / a.group;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = sequence_of(a.cu, a.sequences, t);
  const int64_t len = b < 0 ? 0 : a.rows.length(b, a.cache.page_size, a.max_length);
  const int64_t at = b < 0 ? -1 : (int64_t)a.rows.lengths[b] - a.cu[b + 1] + t;
  const T* q = reinterpret_cast<const T*>(a.q + t * a.q_tok + head * a.q_head) + 2 * lane;
  const float q0 = (float)q[0], q1 = (float)q[1];
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int64_t j = wave; j < len; j += 4) {
    if (!visible(a, j, at)) continue;
    const int64_t entry = j / a.cache.page_size;
    const int page = a.rows.page(b, entry, a.cache.pages);
    if (page < 0) continue;
    const int64_t r = j - entry * a.cache.page_size;
    const float s = a.scale_log2 * dot_row<T>(a.cache.k + page * a.cache.k_page +
                                                  kv * a.cache.k_head + r * a.cache.k_row,
                                              lane, q0, q1);
    const T* v = reinterpret_cast<const T*>(a.cache.v + page * a.cache.v_page +
                                            kv * a.cache.v_head + r * a.cache.v_row) + 2 * lane;
    const float top = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : exp2f(m - top);
    const float p = s == -INFINITY ? 0.f : exp2f(s - top);
    o0 = o0 * keep + p * (float)v[0];
    o1 = o1 * keep + p * (float)v[1];
    l = l * keep + p;
    m = top;
  }
  part[wave][2 * lane] = o0;
  part[wave][2 * lane + 1] = o1;
  if (lane == 0) part[wave][128] = m, part[wave][129] = l;
  __syncthreads();
  if (wave) return;
  float top = -INFINITY;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, part[w][128]);
  float sum = 0.f, x0 = 0.f, x1 = 0.f;
  for (int w = 0; w < 4; ++w) {
    const float f = part[w][128] == -INFINITY ? 0.f : exp2f(part[w][128] - top);
    sum += f * part[w][129];
    x0 += f * part[w][2 * lane];
    x1 += f * part[w][2 * lane + 1];
  }
  T* o = reinterpret_cast<T*>(a.o + t * a.o_tok + head * a.o_head) + 2 * lane;
  o[0] = (T)(sum > 0.f || sum != sum ? x0 / sum : 0.f);
  o[1] = (T)(sum > 0.f || sum != sum ? x1 / sum : 0.f);
  if (lane == 0 && a.lse2) a.lse2[t * a.hq + head] = top + log2f(sum);
}

template <class T>
__global__ __launch_bounds__(256) void cached_weights_kernel(CachedAttnArgs a) {
  const int64_t cap = (int64_t)a.rows.row_pages * a.cache.page_size;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (item >= cap * a.sequences * a.cache.kv_heads) return;
  const int64_t j = item % cap;
  const int kv = (int)(item / cap % a.cache.kv_heads);
  const int b = (int)(item / cap / a.cache.kv_heads);
  float sum = 0.f;
  const int64_t entry = j / a.cache.page_size;
  const int page = a.rows.page(b, entry, a.cache.pages);
  if (j < a.rows.length(b, a.cache.page_size, a.max_length) && page >= 0) {
    const char* k = a.cache.k + page * a.cache.k_page + kv * a.cache.k_head +
                    (j - entry * a.cache.page_size) * a.cache.k_row;
    const int64_t last = min((int64_t)a.cu[b + 1], a.tokens);
    for (int64_t t = max(a.cu[b], 0); t < last; ++t) {
      if (!visible(a, j, (int64_t)a.rows.lengths[b] - a.cu[b + 1] + t)) continue;
      for (int h = kv * a.group; h < (kv + 1) * a.group; ++h) {
        const T* q = reinterpret_cast<const T*>(a.q + t * a.q_tok + h * a.q_head) + 2 * lane;
        sum += exp2f(a.scale_log2 * dot_row<T>(k, lane, (float)q[0], (float)q[1]) -
                     a.lse2[t * a.hq + h]);
      }
    }
  }
  if (lane == 0) a.w_out[item] = (a.w_in ? a.w_in[item] : 0.f) + sum;
}

template <class T>
int launch(const CachedAttnArgs& a, hipStream_t st) {
  if (a.tokens > 0) {
    hipLaunchKernelGGL(cached_attention_kernel<T>, dim3((unsigned)(a.tokens * a.hq)), dim3(256), 0,
                       st, a);
    SS_CHECK_LAUNCH("cached_attention_kernel");
  }
  if (a.w_out) {
    const int64_t items =
        (int64_t)a.rows.row_pages * a.cache.page_size * a.sequences * a.cache.kv_heads;
    hipLaunchKernelGGL(cached_weights_kernel<T>, dim3((unsigned)cdiv(items, 4)), dim3(256), 0, st,
                       a);
    SS_CHECK_LAUNCH("cached_weights_kernel");
  }
  return SS_OK;
}

}  // namespace
}  // namespace ss

extern "C" size_t ss_cached_attention_workspace_size(int rows, int64_t tokens, int q_heads,
                                                     int kv_heads, int max_new,
                                                     int64_t max_length, int weights) {
  if (rows <= 0 || tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || !weights) return 0;
  return (size_t)tokens * q_heads * sizeof(float);
}

extern "C" int ss_cached_attention(const ss_paged_cache* cache, const void* q, int64_t q_tok,
                                   int64_t q_head, int q_heads, const int32_t* table,
                                   int64_t table_stride, int row_pages, const int32_t* lengths,
                                   const int32_t* cu_seqlens, int rows, int64_t tokens,
                                   int max_new, int64_t max_length, float scale, int64_t window,
                                   int64_t sinks, const float* weights_in, float* weights_out,
                                   void* o, int64_t o_tok, int64_t o_head, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  using namespace ss;
  const char* who = "ss_cached_attention";
  if (const int rc = check_cache(who, cache)) return rc;
  if (const int rc = check_table(who, cache, table, table_stride, row_pages, lengths, rows))
    return rc;
  SS_CHECK_ARG(tokens >= 0 && max_new >= 0 && max_length >= 0, "%s: negative size", who);
  SS_CHECK_ARG(window >= 0 && sinks >= 0, "%s: negative window or sinks", who);
  SS_CHECK_ARG(q_heads > 0 && q_heads % cache->kv_heads == 0,
               "%s: %d q heads are no multiple of %d kv heads", who, q_heads, cache->kv_heads);
  if (rows == 0 || (tokens == 0 && !weights_out)) return SS_OK;
  SS_CHECK_ARG(cu_seqlens && (tokens == 0 || (q && o)), "%s: null pointer", who);
  SS_CHECK_ARG(aligned16(q) && aligned16(o) && ((q_tok | q_head | o_tok | o_head) & 7) == 0,
               "%s: needs 16-byte aligned bases and strides that are multiples of 8", who);
  SS_CHECK_ARG(tokens <= (int64_t)INT32_MAX / q_heads, "%s: too many tokens in one call", who);
  const size_t need = ss_cached_attention_workspace_size(rows, tokens, q_heads, cache->kv_heads,
                                                         max_new, max_length, weights_out != 0);
  SS_CHECK_ARG(need <= workspace_bytes && (need == 0 || (workspace && aligned16(workspace))),
               "%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, need);
  CachedAttnArgs a{cache_view(cache), TableView{table, table_stride, row_pages, lengths},
                   cu_seqlens, rows, tokens, max_length, (const char*)q, q_tok * 2, q_head * 2,
                   (char*)o, o_tok * 2, o_head * 2, q_heads, q_heads / cache->kv_heads,
                   scale * kLog2e, window, sinks, weights_in, weights_out,
                   need ? (float*)workspace : nullptr};
  const hipStream_t st = (hipStream_t)stream;
  return cache->dtype == SS_F16 ? launch<half_t>(a, st) : launch<bhalf_t>(a, st);
}
