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
//
// Into a 4-bit cache (paged4.h) the same eight threads find each block's scale (four threads
// have its 32 values) and write four bytes of codes a half.  Codes are decided next to
// borders, half way between two steps, so the rotated key is taken without a rounding before
// its own: products of 24 and 11 bits are exact in fp64, their sum is rounded to odd in fp32
// (a last bit of 1 stands for whatever was cut off), which orders against every border as the
// sum in fp64 does.  The queries' rotation stays in fp32.  6042 tokens (108 MB) 23.4 us, 4.6 TB/s.
// Queries are sets of four heads for eight threads, which load the angles once for them: a head at
// a time 25.4 us, its angles four times its own bytes; with heads of both kinds in a wave 24.9.
#include "paged4.h"

namespace ss {
namespace {

struct AppendArgs {
  CacheView cache;
  TableView rows;
  const int32_t* cu;
  int sequences;
  uint32_t items;  // tokens * heads
  uint32_t query_items;  // 4-bit cache: tokens * sets of query heads, the first of the items
  const char* k; int64_t k_tok, k_head;  // bytes
  const char* v; int64_t v_tok, v_head;
  const char* q; int64_t q_tok, q_head;
  const char* cos; int64_t cos_tok;
  const char* sin; int64_t sin_tok;
  char* qo; int64_t qo_tok, qo_head;
  int hq, heads;  // q heads (0: none); q + 2 kv heads
};

constexpr int kQueryHeads = 4;  // of a set

template <class T>
using Vec8 = T __attribute__((ext_vector_type(8)));

template <class CS>
__device__ __forceinline__ void load_angles(const char* p, int c, float (&out)[8]) {
  const Vec8<CS> v = *reinterpret_cast<const Vec8<CS>*>(p + c * sizeof(CS));
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = (float)v[e];
}

// fp32 with a last bit of 1 wherever y is not one itself, and the smaller size then: never an
// infinity from a number.
__device__ __forceinline__ float rounded_to_odd(double y) {
  const float f = (float)y;
  uint32_t bits = __builtin_bit_cast(uint32_t, f);
  const double back = f;
  if (back != y && y == y) {
    if (fabs(back) > fabs(y)) --bits;
    bits |= 1;
  }
  return __builtin_bit_cast(float, bits);
}

// Codes of eight values of a block, the others of which the next three threads have, and its
// scale byte: the least power of two with which no code is past 6.
template <class T>
__device__ __forceinline__ uint32_t encoded(const float (&x)[8], uint32_t* scale_byte) {
  uint32_t top = 0;  // as bits, which order sizes, NaN above all
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1, kWave));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2, kWave));
  *scale_byte = kNotFinite;
  if (top >= 0x7f800000u) return 0;
  // 6 2^e is 1.5 2^(e + 2): a mantissa past 1.5 carries into the exponent.
  const int byte = min(max((int)((top + 0x3fffffu) >> 23) - 2, Exponents<T>::lowest + 127),
                       Exponents<T>::highest + 127);
  *scale_byte = byte;
  const float scale = scale_of(byte);
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
}

// The row of token t's sequence that it goes to: its page, or -1, and the row in it.
__device__ __forceinline__ int page_of(const AppendArgs& a, uint32_t t, int64_t* r) {
  if (a.sequences == 0) return -1;
  const int b = sequence_of(a.cu, a.sequences, t);
  if (b < 0) return -1;
  // The sequence's own tokens are its last ones.
  const int64_t row = (int64_t)a.rows.lengths[b] - a.cu[b + 1] + t;
  if (row < 0) return -1;
  const int64_t entry = row / a.cache.page_size;
  *r = row - entry * a.cache.page_size;
  return a.rows.page(b, entry, a.cache.pages);
}

// Some heads of a token's queries by eight threads, which load its angles once.
template <class T, class CS>
__device__ __forceinline__ void turn_queries(const AppendArgs& a, uint32_t item, int c) {
  const uint32_t sets = (uint32_t)(a.hq + kQueryHeads - 1) / kQueryHeads, t = item / sets;
  const int first = (int)(item - t * sets) * kQueryHeads;
  Vec8<T> lo[kQueryHeads], hi[kQueryHeads];
#pragma unroll
  for (int i = 0; i < kQueryHeads; ++i) {
    const char* from = a.q + t * a.q_tok + min(first + i, a.hq - 1) * a.q_head;
    lo[i] = reinterpret_cast<const Vec8<T>*>(from)[c / 8];
    hi[i] = reinterpret_cast<const Vec8<T>*>(from)[c / 8 + 8];
  }
  float c1[8], c2[8], s1[8], s2[8];
  load_angles<CS>(a.cos + t * a.cos_tok, c, c1);
  load_angles<CS>(a.cos + t * a.cos_tok, c + 64, c2);
  load_angles<CS>(a.sin + t * a.sin_tok, c, s1);
  load_angles<CS>(a.sin + t * a.sin_tok, c + 64, s2);
#pragma unroll
  for (int i = 0; i < kQueryHeads; ++i) {
    if (first + i >= a.hq) break;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = (float)lo[i][e], y = (float)hi[i][e];
      lo[i][e] = (T)(x * c1[e] - y * s1[e]);
      hi[i][e] = (T)(y * c2[e] + x * s2[e]);
    }
    char* to = a.qo + t * a.qo_tok + (first + i) * a.qo_head;
    reinterpret_cast<Vec8<T>*>(to)[c / 8] = lo[i];
    reinterpret_cast<Vec8<T>*>(to)[c / 8 + 8] = hi[i];
  }
}

template <class T, class CS, bool FOUR>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
  const uint32_t item = blockIdx.x * 32 + (threadIdx.x >> 3);
  if (item >= a.items) return;
  const int c = (threadIdx.x & 7) * 8;
  const int hk = a.cache.kv_heads;
  uint32_t t;
  int head;
  if constexpr (FOUR) {
    if (item < a.query_items) {
      turn_queries<T, CS>(a, item, c);
      return;
    }
    const uint32_t row = item - a.query_items;
    t = row / (2 * (uint32_t)hk);
    head = (int)(row - t * 2 * (uint32_t)hk) + a.hq;
  } else {
    t = item / (uint32_t)a.heads;
    head = (int)(item - t * (uint32_t)a.heads);
  }
  const bool is_q = head < a.hq, is_k = !is_q && head < a.hq + hk;
  const int h = is_q ? head : is_k ? head - a.hq : head - a.hq - hk;
  const char* from = is_q   ? a.q + t * a.q_tok + h * a.q_head
                     : is_k ? a.k + t * a.k_tok + h * a.k_head
                            : a.v + t * a.v_tok + h * a.v_head;
  Vec8<T> lo = reinterpret_cast<const Vec8<T>*>(from)[c / 8];
  Vec8<T> hi = reinterpret_cast<const Vec8<T>*>(from)[c / 8 + 8];
  float x[8], y[8];
  if constexpr (FOUR) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)lo[e], y[e] = (float)hi[e];
  }
  if (a.cos && (is_k || (!FOUR && is_q))) {
    float c1[8], c2[8], s1[8], s2[8];
    load_angles<CS>(a.cos + t * a.cos_tok, c, c1);
    load_angles<CS>(a.cos + t * a.cos_tok, c + 64, c2);
    load_angles<CS>(a.sin + t * a.sin_tok, c, s1);
    load_angles<CS>(a.sin + t * a.sin_tok, c + 64, s2);
    if constexpr (FOUR) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double u = x[e], w = y[e];
        x[e] = rounded_to_odd(u * (double)c1[e] - w * (double)s1[e]);
        y[e] = rounded_to_odd(w * (double)c2[e] + u * (double)s2[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float u = (float)lo[e], w = (float)hi[e];
        lo[e] = (T)(u * c1[e] - w * s1[e]);
        hi[e] = (T)(w * c2[e] + u * s2[e]);
      }
    }
  }
  char* to;
  if (!FOUR && is_q) {
    to = a.qo + t * a.qo_tok + h * a.qo_head;
  } else {
    int64_t r = 0;
    const int page = page_of(a, t, &r);
    if (page < 0) return;
    if constexpr (FOUR) {
      char* group = a.cache.k + page * a.cache.k_page + h * a.cache.k_head +
                    (r >> 4) * a.cache.k_row;
      const int row = (int)(r & 15), part = threadIdx.x & 7, block = part >> 2;
      uint32_t scale_lo, scale_hi;
      const uint32_t codes_lo = encoded<T>(x, &scale_lo), codes_hi = encoded<T>(y, &scale_hi);
      const int at_lo = is_k ? key_at(row, block) + (part & 3) * 4 : value_at(row, part);
      const int at_hi = is_k ? key_at(row, block + 2) + (part & 3) * 4 : value_at(row, part + 8);
      *reinterpret_cast<uint32_t*>(group + at_lo) = codes_lo;
      *reinterpret_cast<uint32_t*>(group + at_hi) = codes_hi;
      char* scales = group + (is_k ? kKeyScales : kValueScales);
      if ((part & 3) == 0) {
        scales[scale_at(row, block)] = (char)scale_lo;
        scales[scale_at(row, block + 2)] = (char)scale_hi;
      }
      return;
    }
    to = is_k ? a.cache.k + page * a.cache.k_page + h * a.cache.k_head + r * a.cache.k_row
              : a.cache.v + page * a.cache.v_page + h * a.cache.v_head + r * a.cache.v_row;
  }
  reinterpret_cast<Vec8<T>*>(to)[c / 8] = lo;
  reinterpret_cast<Vec8<T>*>(to)[c / 8 + 8] = hi;
}

template <bool FOUR, class Cache>
int append(const char* who, const Cache* cache, const void* k, int64_t k_tok, int64_t k_head,
           const void* v, int64_t v_tok, int64_t v_head, const void* q, int64_t q_tok,
           int64_t q_head, int q_heads, const void* cos, int64_t cos_tok, const void* sin,
           int64_t sin_tok, int cs_dtype, const int32_t* table, int64_t table_stride, int row_pages,
           const int32_t* lengths, const int32_t* cu_seqlens, int rows, int64_t tokens,
           void* q_out, int64_t qo_tok, int64_t qo_head, void* stream) {
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
  const int64_t sets = FOUR ? cdiv(hq, kQueryHeads) : 0;
  const int64_t items = tokens * (FOUR ? sets + 2 * (int64_t)cache->kv_heads : heads);
  SS_CHECK_ARG(fits_grid(items, 32, 256), "%s: too many rows in one call", who);
  AppendArgs a{cache_view(cache), TableView{table, table_stride, row_pages, lengths},
               cu_seqlens, rows, (uint32_t)items, (uint32_t)(tokens * sets),
               (const char*)k, k_tok * 2, k_head * 2, (const char*)v, v_tok * 2, v_head * 2,
               (const char*)q, q_tok * 2, q_head * 2, (const char*)cos, cos_tok * cs,
               (const char*)sin, sin_tok * cs, (char*)q_out, qo_tok * 2, qo_head * 2, hq,
               (int)heads};
  const dim3 grid((unsigned)cdiv(items, 32)), block(256);
  const hipStream_t st = (hipStream_t)stream;
  const bool wide = cos && cs_dtype == SS_F32;
  if (cache->dtype == SS_F16) {
    if (wide) hipLaunchKernelGGL((kv_append_kernel<half_t, float, FOUR>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((kv_append_kernel<half_t, half_t, FOUR>), grid, block, 0, st, a);
  } else {
    if (wide) hipLaunchKernelGGL((kv_append_kernel<bhalf_t, float, FOUR>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((kv_append_kernel<bhalf_t, bhalf_t, FOUR>), grid, block, 0, st, a);
  }
  SS_CHECK_LAUNCH("kv_append_kernel");
  return SS_OK;
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
  return ss::append<false>("ss_kv_append", cache, k, k_tok, k_head, v, v_tok, v_head, q, q_tok,
                                           q_head, q_heads, cos, cos_tok, sin, sin_tok, cs_dtype,
                                           table, table_stride, row_pages, lengths, cu_seqlens,
                                           rows, tokens, q_out, qo_tok, qo_head, stream);
}

extern "C" int ss_kv_append4(const ss_paged_cache4* cache, const void* k, int64_t k_tok,
                             int64_t k_head, const void* v, int64_t v_tok, int64_t v_head,
                             const void* q, int64_t q_tok, int64_t q_head, int q_heads,
                             const void* cos, int64_t cos_tok, const void* sin, int64_t sin_tok,
                             int cs_dtype, const int32_t* table, int64_t table_stride,
                             int row_pages, const int32_t* lengths, const int32_t* cu_seqlens,
                             int rows, int64_t tokens, void* q_out, int64_t qo_tok,
                             int64_t qo_head, void* stream) {
  return ss::append<true>("ss_kv_append4", cache, k, k_tok, k_head, v, v_tok, v_head, q, q_tok,
                                           q_head, q_heads, cos, cos_tok, sin, sin_tok, cs_dtype,
                                           table, table_stride, row_pages, lengths, cu_seqlens,
                                           rows, tokens, q_out, qo_tok, qo_head, stream);
}
