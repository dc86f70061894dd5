// Attention of new tokens over a paged cache that holds its rows in 4 bits (paged4.h).
//
// o = sum_j softmax_j(scale q . k_j) v_j with a running maximum and sum in fp32, units of work and
// their split over the keys as over a 16-bit cache (cached_units.h).  Keys and values
// become 16-bit numbers in registers, exactly (two significant bits times a power of two), on
// v_cvt_scalef32_pk, which takes the block's scale with it; all products are 16-bit MFMAs,
// so that the result is that of a 16-bit cache with the same rows.  As there P is rounded to the
// cache's type, its product's operand, while its sum is of what was not rounded: bf16 outputs
// lie 2.0e-3 of their norm from 64 bits, 1.7e-3 of it their own rounding, fp16 ones 2.2e-4 and
// 2.1e-4 of that.
//
// Products (v_mfma_f32_16x16x32): S^T = K Q^T and O^T += V^T P^T, operands as over a 16-bit
// cache.  A group of 16 rows is laid out for it: 16 bytes a lane are one key's 32
// dimensions of one block, the operands of four products as they stand (the queries' dimensions
// are taken in the same order: lane group g has 32 g + 8 s .. + 7 of product s), and 16 bytes
// are four keys' values in eight columns, which permutes pair by key.
//
// What bounds it: a tile of 32 keys and 16 query rows takes a SIMD 1400 cycles (170 vector
// instructions, 64 of them conversions, 32 permutes, 12 for the values' scales, some 50 for the
// softmax, and 16 MFMAs, which overlap little), and HBM's rate leaves 1500 for its 4352 bytes,
// so a large batch is near both: 64 sequences of 5860 .. 8191 keys (245 MB) 50 us, 4.9 TB/s, the
// vector units busy 60 of 100 cycles and the matrix cores 15.
// Tiles on their way in the loop's order count more than their number: with the first ones' loads
// in another order the loop's first wait was for all of them (53.7 us); 2, 3 and 4 tiles 51.5
// (12 waves), 50.0 and 51.9 us; two workgroups a CU 60.2 (128 registers, some spilled).  Longer
// blocks are bound by vector instructions (373 a tile of 32 rows, conversions for each wave by itself
// among them) that its products do not run beside: 64 tokens of 4 sequences (13.7 GFLOP) 37 us, of
// whose 73700 cycles the vector units are busy 41400 and the matrix cores 13200.  They go by ranges
// (parts of 55 tiles would be 308), 92 of which hold the end of one unit and the start of another.
// Decoded by one wave for four of 32 rows, through LDS with a barrier for two tiles, 45.4, when
// this took 39.  One sequence is latency: 518 keys 7.7 us, 131071 keys (71 MB) 19 us, of which
// 5 pass before the first tile is there and 2 to 3 after the last one, and 5 for the join.

#include "cached_units.h"
#include "paged4.h"

namespace ss {
namespace {

constexpr int kDeep = 3;       // tiles of a wave on their way
constexpr int kSteps = 27;     // tiles of a wave whose pages are looked up at once
static_assert(kSteps % kDeep == 0 && 2 * (kSteps + kDeep) <= kWave, "a lane for every half tile");

template <int QT, int W>
struct Shared4 : Results<QT, W> {
  struct alignas(16) {
    float o[16 * QT][kPadDim];
  } wave[W];
};

// A row's sums stay where they are until a tile's maximum is more than this power of two above the
// one that they refer to.  A wave of a long call has few tiles, and in most of the first ones some
// row has a new maximum: 4 sequences of 64 tokens (bf16) 38.9 us, without 40.2.
template <class T>
constexpr float kRise = std::is_same<T, half_t>::value ? 0.99f : 8.f;

// Powers of two that P is raised by.  fp16: as over a 16-bit cache, and P, up to 2^0.99 above its
// lift then, stays below 65504 (2^15.99 is 65070).  bf16: lowered by what sums may rise, so that P
// is 1 at most and sums of values next to fp32's end (the cache holds up to 6 2^125) do not pass
// it; P of at least 2^-8 at the top leaves the least value, 2^-126, 15 bits in fp32's subnormals.
template <class T>
constexpr float kLift4 = std::is_same<T, half_t>::value ? kLift<T> : -kRise<T>;

// 32 rows of one kv head: two groups' parts, as the lanes load them.
struct Tile4 {
  u32x4 k[2], v[2];
  uint32_t ks[2], vs[2];  // a key's scale; those of four values' rows
};

// NaN for the rows that see a value block that is, which a wave's products left out: its tiles
// again, rarely (two columns a lane).
template <int QT>
__device__ __noinline__ void add_left_out4(LateArgs* late, float (*o)[kPadDim], int b, Sequence seq,
                                           Span span, int kv, int r0, int x, int x_end,
                                           int stripes) {
  CachedAttnArgs a;
  __builtin_memcpy(&a, (const void*)late, sizeof a);
  const int lane = threadIdx.x & 63, size = a.cache.page_size;
  const int rows = min(16 * QT, min(seq.n, a.max_new) * a.group - r0);
  const char* base = a.cache.k + (int64_t)kv * a.cache.k_head + kValueScales;
  for (; x < x_end; x += stripes) {
    const int j0 = span.tile(x) * kKeys;
    for (int j = j0; j < min(j0 + kKeys, seq.len); ++j) {
      const int entry = j / size, row = j - entry * size;
      const int page = a.rows.page(b, entry, a.cache.pages);
      if (page < 0) continue;
      const uint8_t scale = *reinterpret_cast<const uint8_t*>(
          base + (int64_t)page * a.cache.k_page + (int64_t)(row >> 4) * a.cache.k_row +
          scale_at(row & 15, lane >> 4));
      if (scale != kNotFinite) continue;
      for (int r = 0; r < rows; ++r) {
        const int i = (r0 + r) / a.group;
        if (j > seq.last(i) || (j < seq.low(a, i) && j >= a.sinks)) continue;
        o[r][2 * lane] = o[r][2 * lane + 1] = NAN;
      }
    }
  }
}

// The tiles [x0, x1) of a unit by the waves of the workgroup, and their join.
template <class T, int QT, int W, int RW, bool ONCE>
__device__ __forceinline__ void attend4(const CachedAttnArgs& a, Shared4<QT, W>& lds, int b,
                                        int block, int kv, const Sequence& seq, const Span& span,
                                        int x0, int x1, bool whole, int slot) {
  // Opaque, so that what follows from them is not kept in registers through the segments' loop.
  int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
  asm volatile("" : "+v"(lane), "+s"(wave));
  const int thread = 64 * wave + lane;
  const int col = lane & 15, grp = lane >> 4;
  const int size = a.cache.page_size;
  const int rows = min(seq.n, a.max_new) * a.group;
  const int block_row = block * 16 * QT * RW;
  const int r0 = block_row + wave % RW * 16 * QT;
  const int stripe = wave / RW;
  constexpr int kStripes = W / RW;
  const int x_end = r0 < rows ? x1 : x0;  // the waves behind the last row have nothing

  Vec8<T> q[QT][4];  // Q[row][32 grp + 8 s ..]
  int last[QT], low[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = min(r0 + 16 * t + col, rows - 1);
    const int token = r / a.group;
    const char* p = a.q + (int64_t)(seq.start + token) * a.q_tok +
                    (int64_t)(kv * a.group + r - token * a.group) * a.q_head + grp * 64;
#pragma unroll
    for (int s = 0; s < 4; ++s) q[t][s] = *reinterpret_cast<const Vec8<T>*>(p + s * 16);
    last[t] = seq.last(token);
    low[t] = seq.low(a, token);
  }
  // The maximum and the masks want a positive scale: a negative one changes the queries' sign
  // (exact), a zero one makes them zeros.
  const float scale = a.scale_log2;
  if (a.q_sign != 1.f) {
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int s = 0; s < 4; ++s) q[t][s] *= (T)a.q_sign;
  }
  const int sinks = span.sinks;
  const char* base = a.cache.k + (int64_t)kv * a.cache.k_head;
  const uint32_t lane16 = lane * 16, value_scales = scale_at(4 * grp, col >> 2);

  // Tokens of this wave's rows.
  const int t0 = uniform(min(r0, rows - 1) / a.group);
  const int t1 = uniform(min(r0 + 16 * QT - 1, rows - 1) / a.group);
  const int see_low = seq.low(a, t0), see_high = seq.last(t1) + 1;
  const bool several = t0 != t1;
  bool left_out = false;
  {
    float4v acc[QT][8];
    float m[QT], l[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[t][e] = float4v{0.f, 0.f, 0.f, 0.f};
      m[t] = -INFINITY;
      l[t] = 0.f;
    }
    // Some of this wave's tiles at a time: their groups' addresses in one load, the lanes behind
    // them none.
#pragma unroll 1
    for (int x = x0 + stripe; x < x_end; x += kSteps * kStripes) {
      const int steps = uniform(min((x_end - x + kStripes - 1) / kStripes, kSteps));
      Halves at;
      {
        int page = -1, row = 0;
        const int j = span.tile(x + (lane >> 1) * kStripes) * kKeys + (lane & 1) * 16;
        if ((lane >> 1) < steps && j < seq.len) {
          const int entry = j / size;
          page = a.rows.page(b, entry, a.cache.pages);
          row = j - entry * size;
        }
        at.set(base + (int64_t)max(page, 0) * a.cache.k_page +
                   (int64_t)(row >> 4) * a.cache.k_row,
               page >= 0);
      }
      // Of a group that no page holds, or behind the last tile, nothing is fetched: zeros.
      auto fetch = [&](Tile4& tile, int s) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const Rsrc group = at.rows(2 * s + u);
          tile.k[u] = load16<ONCE>(group, lane16, 0);
          tile.v[u] = load16<ONCE>(group, lane16, kValues);
          tile.ks[u] = __builtin_amdgcn_raw_buffer_load_b8(group, lane, kKeyScales, ONCE * 2);
          tile.vs[u] =
              __builtin_amdgcn_raw_buffer_load_b32(group, value_scales, kValueScales, ONCE * 2);
        }
      };
      auto attend_tile = [&](Tile4& tile, int s) {
        const int j0 = span.tile(x + s * kStripes) * kKeys;
        const bool held0 = at.held(2 * s), held1 = at.held(2 * s + 1);
        float sc[QT][8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float ks = scale_of(tile.ks[u]);
          float4v c[QT] = {};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const Vec8<T> k = __builtin_bit_cast(Vec8<T>, decoded<T>(tile.k[u][w], ks));
#pragma unroll
            for (int t = 0; t < QT; ++t) c[t] = mfma(k, q[t][w], c[t]);
          }
#pragma unroll
          for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[t][4 * u + i] = c[t][i];
        }
        if (!(held0 && held1 && span.clear(j0))) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int j = j0 + 4 * grp + (i & 3) + 16 * (i >> 2);
            const bool held = i < 4 ? held0 : held1;
#pragma unroll
            for (int t = 0; t < QT; ++t)
              sc[t][i] = held & (j <= last[t]) & ((j >= low[t]) | (j < sinks)) ? sc[t][i] : -INFINITY;
            // Values that no row of the wave sees become zeros, and so do NaN ones that some
            // see and others do not.
            const bool seen = held & (j < see_high) & ((j >= see_low) | (j < sinks));
            uint32_t& scales = tile.vs[i >> 2];
            const uint32_t byte = 255u << 8 * (i & 3);
            const bool odd = seen & several & ((scales & byte) == byte);
            left_out |= odd;
            const bool counts = seen & !odd;
            tile.v[i >> 2][i & 3] = counts ? tile.v[i >> 2][i & 3] : 0u;
            scales = counts ? scales : (scales & ~byte) | 127u << 8 * (i & 3);
          }
        }
        Vec8<T> p[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          float top = sc[t][0];
#pragma unroll
          for (int i = 1; i < 8; ++i) top = fmaxf(top, sc[t][i]);
          top = group_max(top);
          const bool rises = (top - m[t]) * scale > kRise<T>;
          if (__any(rises)) {
            const float next = rises ? top : m[t];
            const float keep =
                __builtin_amdgcn_exp2f((m[t] - (next == -INFINITY ? 0.f : next)) * scale);
            l[t] *= keep;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[t][e] *= keep;
            m[t] = next;
          }
          const float base_score = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float w =
                __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i] - base_score, scale, kLift4<T>));
            l[t] += w;
            p[t][i] = (T)w;
          }
        }
        u32x4 vf[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          vf[i] = decoded<T>(tile.v[i >> 2][i & 3],
                             scale_of(tile.vs[i >> 2] >> 8 * (i & 3) & 255u));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const Vec8<T> v = __builtin_bit_cast(Vec8<T>, turned(vf, e));
#pragma unroll
          for (int t = 0; t < QT; ++t) acc[t][e] = mfma(v, p[t], acc[t][e]);
        }
      };
      Tile4 tiles[kDeep];
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        fetch(tiles[d], d);
        __builtin_amdgcn_sched_barrier(0);  // in the order of the loop's, for its waits
      }
#pragma unroll 1
      for (int s = 0; s < steps; s += kDeep)
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
          if (s + d < steps) attend_tile(tiles[d], s + d);
          // Not before the products, which the registers' old contents are for.
          __builtin_amdgcn_sched_barrier(0);
          fetch(tiles[d], s + d + kDeep);
          __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const float sum = group_sum(l[t]);
      const int r = 16 * t + col;
      if (grp == 0) lds.m[wave][r] = m[t], lds.l[wave][r] = sum;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          *reinterpret_cast<float4v*>(&lds.wave[wave].o[r][32 * grp + 8 * i + 4 * u]) =
              float4v{acc[t][4 * u][i], acc[t][4 * u + 1][i], acc[t][4 * u + 2][i],
                      acc[t][4 * u + 3][i]};
    }
  }
  if (__any(left_out))
    add_left_out4<QT>(late_args(), lds.wave[wave].o, b, seq, span, kv, r0, x0 + stripe, x_end,
                      kStripes);
  finish_unit<T, QT, W, RW>(lds, lds.wave, thread, block, block_row, rows, kv, seq, span, x1,
                            whole, slot);
}

template <class T, int QT, int W, int RW, bool SPLIT, bool ONCE>
__global__ __launch_bounds__(64 * W, 2) void cached_attention4_kernel(CachedAttnArgs a) {
  __shared__ Shared4<QT, W> lds;
  auto unit = [&](int b, int block, int kv, const Sequence& seq, const Span& span, int x0, int x1,
                  bool whole, int slot) {
    attend4<T, QT, W, RW, ONCE>(a, lds, b, block, kv, seq, span, x0, x1, whole, slot);
  };
  if constexpr (SPLIT) for_ranges<QT, W, RW, true>(a, lds, unit);
  else for_unit<QT, RW>(a, unit);
  if (blockIdx.x == 0) clear_outside<W>(a);
}

// The join of long blocks where a unit has few parts: a workgroup takes eight rows at once, 32
// lanes of 4 columns each, part by part, or, of a unit that has more (a long sequence among short
// ones), one after the other.  112 units of 64 rows, up to five parts each (ranges): 5.4 us, with a
// workgroup a row 8.4 (7168 of them, most of whose threads have no part).  Of 16 rows it is no
// faster (64 units, 15 rows, four parts: the call 19.0 us against 17.7).
constexpr int kFewParts = 8, kJoinRows = 8;
template <class T, int ROWS>
__global__ __launch_bounds__(32 * kJoinRows) void cached_join_rows_kernel(CachedAttnArgs a) {
  __shared__ JoinShared lds;
  const int hk = a.cache.kv_heads;
  const int line = (int)(blockIdx.x / hk), kv = (int)(blockIdx.x - line * hk);
  const int b = line / a.blocks, block = line - b * a.blocks;
  const int4 unit = a.units[blockIdx.x];
  const Sequence seq(a, b);
  const int first = blockIdx.y * kJoinRows;
  const int rows = min(kJoinRows, min(seq.n, a.max_new) * a.group - block * ROWS - first);
  if (rows <= 0 || unit.x == unit.y) return;
  const int count = unit.y - unit.x + 1;
  if (count > kFewParts) {
    for (int r = 0; r < rows; ++r) {
      join_row<T, ROWS>(a, lds, seq, unit, block, kv, first + r);
      __syncthreads();
    }
    return;
  }
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
  if (r >= rows) return;
  auto part = [&](int i) {
    return (int64_t)(2 * (unit.x + i) + (i ? 0 : unit.z)) * ROWS + first + r;
  };
  float2v s{-INFINITY, 0.f};  // of the lane's part
  if (c < count) s = *reinterpret_cast<const float2v*>(a.part_ml + part(c) * 2);
  float m = s[0];
#pragma unroll
  for (int d = kFewParts / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, kFewParts));
  m = __shfl(m, 0, 32);
  const float base = m == -INFINITY ? 0.f : m;
  const float f = __builtin_amdgcn_exp2f((s[0] - base) * a.scale_log2);
  float sum = 0.f;
  float4v o{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = 0; i < count; ++i) {
    const float fi = __shfl(f, i, 32);
    sum += fi * __shfl(s[1], i, 32);
    o += fi * *reinterpret_cast<const float4v*>(a.part_o + part(i) * kCacheDim + 4 * c);
  }
  store_joined<T>(a, seq, kv, block * ROWS + first + r, c, o, sum, base);
}

// One workgroup a unit, or the split: whole, the units that there are leave the other CUs without
// work, a tile of a wave 0.9 us long (16 rows) or 1.5; split, the join comes after, 5.5 us and
// one more for 1100 rows.  Past 16 tiles the lengths, which the bound says little of, matter more.
// So and so, whole and split, us: 28 / 4 heads, one token, 1 / 8 / 32 sequences of 1500 keys 11.7
// 12.7 / 11.8 13.1 / 12.8 16.8, of 3000 17.5 12.7 / 17.6 13.7 / 18.8 19.9; 12 / 2 heads, 5 tokens,
// of 1500 15.9 13.5 / 16.0 14.4 / 16.3 17.0; 28 / 4 heads, 8 tokens, of 600 14.7 15.4 / 15.0 16.9 /
// 15.6 29.5, of 1500 24.1 15.4 / 24.3 19.4 / 25.0 33.4.
bool whole(int unit_rows, int64_t units, int cus, int64_t tiles) {
  const double idle = units < cus ? 1.0 - (double)units / cus : 0.0;
  const double tile = unit_rows <= 16 ? 0.9 : 1.5;
  return tiles <= 16 && tiles * tile * idle <= 5.5 + (double)units * unit_rows / 1100;
}

// Blocks of 64 rows at most: 64 tokens of 4 sequences (448 rows a kv head) 42.9 us, in blocks of
// 128 45.7 and of 32 54.7.
Layout layout4(int rows, int64_t tokens, int q_heads, int kv_heads, int max_new,
               int64_t max_length) {
  return Layout(rows, tokens, q_heads, kv_heads, max_new, max_length, false, whole, 64);
}

template <class T, int QT, int W, int RW, bool ONCE>
int launch_whole4(const CachedAttnArgs& a, const Layout& p, hipStream_t st) {
  hipLaunchKernelGGL((cached_attention4_kernel<T, QT, W, RW, false, ONCE>),
                     dim3((unsigned)p.units), dim3(64 * W), 0, st, a);
  SS_CHECK_LAUNCH("cached_attention4_kernel");
  return SS_OK;
}

template <class T, int QT, int RW, bool ONCE>
int launch_attention4(const CachedAttnArgs& a, const Layout& p, hipStream_t st) {
  if (!p.workers) {
    // More units than CUs: workgroups of four waves, of which a CU holds two, so that one's start
    // and end pass while another multiplies.  More than those hold at once: of two waves, where
    // the work of a unit is little.  With 8, 4 and 2 waves, us: 320 units of 24 rows, 40 keys
    // 14.2 9.0, 600 20.7 16.7, 2000 38.7 32.2; 640 of 24 rows, 40 keys - 14.2 9.4, 600 - 24.2
    // 23.0; 800 of up to 64 rows, 40 keys - 19.9 14.0, 600 - 42.5 42.0; 448 of 64 rows, 600 keys
    // 77.7 57.5 63.3, 2000 164.5 136 175; 1024 of one row, 40 keys - 11.1 7.3, 600 - 20.6 18.8,
    // 2000 - 48.8 49.9; 2000 of seven rows, 40 keys - 17.4 12.2, 2000 - 97.9 103.  (Blocks of 16
    // rows take two at any length, which costs those 2 and 5 % where sequences are long.)
    const int64_t cus = device_cu_count();
    const bool little = QT == 1 || a.max_length <= 16 * kKeys * (2 / RW);
    if (p.units > 2 * cus && little) return launch_whole4<T, QT, 2, RW, ONCE>(a, p, st);
    if (p.units > cus) return launch_whole4<T, QT, 4, RW, ONCE>(a, p, st);
    return launch_whole4<T, QT, kWaves, RW, ONCE>(a, p, st);
  }
  hipLaunchKernelGGL((cached_attention4_kernel<T, QT, kWaves, RW, true, ONCE>),
                     dim3((unsigned)p.workers), dim3(64 * kWaves), 0, st, a);
  SS_CHECK_LAUNCH("cached_attention4_kernel");
  const int64_t rows = (int64_t)a.max_new * a.group;
  const unsigned block = (unsigned)(rows < p.block_rows ? rows : p.block_rows);
  if constexpr (QT > 1) {
    if (p.units * kFewParts >= p.workers) {
      hipLaunchKernelGGL((cached_join_rows_kernel<T, 16 * QT * RW>),
                         dim3((unsigned)p.units, (block + kJoinRows - 1) / kJoinRows), dim3(256), 0,
                         st, a);
      SS_CHECK_LAUNCH("cached_join_rows_kernel");
      return SS_OK;
    }
  }
  hipLaunchKernelGGL((cached_join_kernel<T, 16 * QT * RW>), dim3((unsigned)p.units, block),
                     dim3(256), 0, st, a);
  SS_CHECK_LAUNCH("cached_join_kernel");
  return SS_OK;
}

// Bytes of rows that the bounds allow from which on they are loaded past the caches (nt), as over
// a 16-bit cache.
constexpr int64_t kOnceBytes = (int64_t)32 << 20;

template <class T>
int launch4(const CachedAttnArgs& a, const Layout& p, hipStream_t st) {
  if (a.sequences == 0) {
    hipLaunchKernelGGL(cached_zeros_kernel, dim3((unsigned)cdiv(a.tokens * a.hq, kZeroRows)),
                       dim3(256), 0, st, a);
    SS_CHECK_LAUNCH("cached_zeros_kernel");
    return SS_OK;
  }
  if (p.block_rows > 32) return launch_attention4<T, 2, 2, false>(a, p, st);
  int64_t keys = a.max_length;
  if (a.window && a.window < keys && a.sinks < keys)
    keys = std::min(keys, a.window + a.sinks + a.max_new);
  const bool once = keys >= kOnceBytes * kGroupRows / kGroupBytes /
                                ((int64_t)a.sequences * a.cache.kv_heads);
  if (p.block_rows == 16)
    return once ? launch_attention4<T, 1, 1, true>(a, p, st)
                : launch_attention4<T, 1, 1, false>(a, p, st);
  return once ? launch_attention4<T, 2, 1, true>(a, p, st)
              : launch_attention4<T, 2, 1, false>(a, p, st);
}

}  // namespace
}  // namespace ss

extern "C" size_t ss_cached_attention4_workspace_size(int rows, int64_t tokens, int q_heads,
                                                      int kv_heads, int max_new,
                                                      int64_t max_length) {
  if (rows <= 0 || tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || max_new < 0 ||
      max_length < 0 || q_heads % kv_heads)
    return 0;
  return ss::layout4(rows, tokens, q_heads, kv_heads, max_new, max_length).bytes;
}

extern "C" int ss_cached_attention4(const ss_paged_cache4* cache, const void* q, int64_t q_tok,
                                    int64_t q_head, int q_heads, const int32_t* table,
                                    int64_t table_stride, int row_pages, const int32_t* lengths,
                                    const int32_t* cu_seqlens, int rows, int64_t tokens,
                                    int max_new, int64_t max_length, float scale, int64_t window,
                                    int64_t sinks, void* o, int64_t o_tok, int64_t o_head,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  using namespace ss;
  const char* who = "ss_cached_attention4";
  if (const int rc = check_cache(who, cache)) return rc;
  if (const int rc = check_table(who, cache, table, table_stride, row_pages, lengths, rows))
    return rc;
  SS_CHECK_ARG(tokens >= 0 && max_new >= 0 && max_length >= 0, "%s: negative size", who);
  SS_CHECK_ARG(window >= 0 && sinks >= 0, "%s: negative window or sinks", who);
  SS_CHECK_ARG(q_heads > 0 && q_heads % cache->kv_heads == 0,
               "%s: %d q heads are no multiple of %d kv heads", who, q_heads, cache->kv_heads);
  if (tokens == 0) return SS_OK;
  SS_CHECK_ARG((rows == 0 || cu_seqlens) && q && o, "%s: null pointer", who);
  SS_CHECK_ARG(aligned16(q) && aligned16(o) && ((q_tok | q_head | o_tok | o_head) & 7) == 0,
               "%s: needs 16-byte aligned bases and strides that are multiples of 8", who);
  SS_CHECK_ARG(max_new > 0, "%s: tokens, but max_new is 0", who);
  const Layout p = layout4(rows, tokens, q_heads, cache->kv_heads, max_new, max_length);
  SS_CHECK_ARG(tokens <= (int64_t)INT32_MAX / q_heads && p.units <= kMaxGrid / 4 &&
                   (rows > 0 || fits_grid(tokens * q_heads, kZeroRows, 256)),
               "%s: too many tokens in one call", who);
  const size_t need = ss_cached_attention4_workspace_size(rows, tokens, q_heads, cache->kv_heads,
                                                          max_new, max_length);
  SS_CHECK_ARG(need <= workspace_bytes && (need == 0 || (workspace && aligned16(workspace))),
               "%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, need);
  char* ws = (char*)workspace;
  CachedAttnArgs a{cache_view(cache), TableView{table, table_stride, row_pages, lengths},
                   cu_seqlens, rows, tokens, max_length, (const char*)q, q_tok * 2, q_head * 2,
                   (char*)o, o_tok * 2, o_head * 2, q_heads, q_heads / cache->kv_heads,
                   scale == 0.f ? 1.f : fabsf(scale) * kLog2e,
                   scale < 0.f ? -1.f : scale == 0.f ? 0.f : 1.f, window, sinks, nullptr, nullptr,
                   nullptr, p.max_new, p.blocks, p.workers, (int4*)(ws + p.list),
                   (float*)(ws + p.ml), (float*)(ws + p.o), nullptr, 0, p.score_keys};
  const hipStream_t st = (hipStream_t)stream;
  return cache->dtype == SS_F16 ? launch4<half_t>(a, p, st) : launch4<bhalf_t>(a, p, st);
}
