// The 4-bit paged cache: its bytes and host checks.
//
// A row has 128 keys and 128 values of one kv head, in blocks of 32 that share a scale 2^e.  A
// value is a code of 4 bits (sign, two bits exponent, one mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6)
// times that scale, so two significant bits: exact in fp16 and bf16 as long as e keeps away
// from the ends of their range (Exponents' lowest .. highest; past 6 2^highest codes saturate).  The
// scale is the byte e + 127; 255 makes the block NaN (one that held an infinity or NaN).
//
// 16 rows of a page are a group of 2176 bytes, 17 lines of 128, laid out so that a wave of 64
// loads each part as it stands, 16 bytes a lane side by side:
//   [block 4][row 16][16 bytes]          key codes: lane (row, block) has a row of the
//                                        product's operand, 32 of its 128 dimensions
//   [row / 4][dims / 8][row % 4][4 bytes] value codes: lane (c, quad) has dimensions 8 c .. + 7
//                                        of four rows
//   [block 4][row 16]                    key scales, a byte each
//   [block 4][row 16]                    value scales
// Of two codes in a byte the lower dimension's is the low one.
#pragma once

#include "paged.h"

namespace ss {

constexpr int kGroupRows = 16;
constexpr int kGroupBytes = 2176;
constexpr int kValues = 1024, kKeyScales = 2048, kValueScales = 2112;  // offsets in a group
constexpr uint32_t kNotFinite = 255;  // scale byte

template <class T>
struct Exponents;
template <>
struct Exponents<half_t> {
  static constexpr int lowest = -13, highest = 13;
};
template <>
struct Exponents<bhalf_t> {
  static constexpr int lowest = -125, highest = 125;
};

__host__ __device__ constexpr int key_at(int row, int block) { return block * 256 + row * 16; }
// Of dimensions 8 chunk .. + 7.
__host__ __device__ constexpr int value_at(int row, int chunk) {
  return kValues + (row >> 2) * 256 + chunk * 16 + (row & 3) * 4;
}
__host__ __device__ constexpr int scale_at(int row, int block) { return block * 16 + row; }

__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __builtin_bit_cast(float, byte << 23);
}

// The two values of byte B of eight codes, as two 16-bit numbers.
template <class T, int B>
__device__ __forceinline__ uint32_t decoded(uint32_t codes, float scale) {
  if constexpr (sizeof(T) == 2 && Exponents<T>::highest == 13)
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, B));
  else
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
}
template <class T>
__device__ __forceinline__ u32x4 decoded(uint32_t codes, float scale) {
  return u32x4{decoded<T, 0>(codes, scale), decoded<T, 1>(codes, scale),
               decoded<T, 2>(codes, scale), decoded<T, 3>(codes, scale)};
}

// k of the view is the cache's bytes, k_row the stride between groups; there is no v.
inline CacheView cache_view(const ss_paged_cache4* c) {
  return CacheView{(char*)c->data, c->page, c->head, c->group, nullptr, 0, 0, 0,
                   c->pages, c->page_size, c->kv_heads};
}

inline int check_cache(const char* who, const ss_paged_cache4* c) {
  SS_CHECK_ARG(c && c->data, "%s: null cache", who);
  SS_CHECK_ARG(c->dtype == SS_F16 || c->dtype == SS_BF16, "%s: cache dtype must be fp16 or bf16",
               who);
  SS_CHECK_ARG(c->head_dim == kCacheDim, "%s: head_dim %d, expected 128", who, c->head_dim);
  SS_CHECK_ARG(c->pages > 0 && c->kv_heads > 0, "%s: cache without pages or heads", who);
  SS_CHECK_ARG(c->page_size > 0 && c->page_size % 16 == 0,
               "%s: page_size %d must be a multiple of 16", who, c->page_size);
  SS_CHECK_ARG(aligned16(c->data) && ((c->page | c->head | c->group) & 15) == 0,
               "%s: cache needs a 16-byte aligned base and strides that are multiples of 16", who);
  return SS_OK;
}

}  // namespace ss
