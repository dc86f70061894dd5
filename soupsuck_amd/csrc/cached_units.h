// What attention over a paged cache shares whatever the cache holds its rows in: the calls'
// arguments, sequences and what their tokens see, units of work and their split over the
// workgroups, the join of partial results and the workspace's layout.
//
// A unit of work is one kv head over one block of a sequence's query rows (token-major, the
// q heads of the group side by side: all of them share the cache's rows).  Its keys go in
// tiles of 32, dealt to the waves of a workgroup in turn; each wave keeps its own (m, l, o)
// in registers and meets the others only at the end (finish_unit).
//
// Split over the keys: the tiles of all units form one line that is cut into equal ranges, one
// a workgroup, from the lengths on the device (for_ranges), so that one long sequence and a
// batch of ragged ones load every CU alike whatever the bounds that the host knows.  A unit
// inside a range is finished there; of one that crosses ranges each part leaves (o, m, l), and
// cached_join_kernel adds them up.
#pragma once

#include <algorithm>
#include <type_traits>

#include "paged.h"
#include "elementwise.h"

namespace ss {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeys = 32;       // of a tile
constexpr int kPadDim = kCacheDim + 4;  // fp32 row of the waves' results in LDS
// Query rows of a kv head up to which their scores are kept (those of one 16-row block): kept
// and with the keys again, 64 sequences of 7000 keys with 7 rows 196 and 249 us, 14 rows 215 and
// 252, 16 rows (two kv heads) 117 and 135; 4 of them 27.9 / 32.4, 32.7 / 33.6, 25.2 / 26.8; 4 of
// 1000 18.1 / 17.4, 22.0 / 18.3, 18.0 / 18.1.  4 sequences with 28 rows took 60 and 34.
constexpr int kScoreRows = 16;
constexpr size_t kScoreBytes = (size_t)512 << 20;
// Tiles that a unit's start and join take the time of: 16 ragged sequences 47 us with 0, 32
// with 4, 26.7 with 8, 26.5 with 12; 33 new tokens of 4 sequences 34, 36 and 42 us.
constexpr int kStart = 8;
// Tiles of a range at least.  With one for each wave and a start (16) many ranges of a small
// call held the end of one unit and the start of another, one after the other: 8 sequences
// x 5 tokens 24.0 us against 18.2; with 3 18.9, 131071 keys the same with each.
constexpr int kMinRange = kStart + 1;
constexpr int64_t kMaxGrid = (int64_t)1 << 23;  // workgroups of a launch

struct CachedAttnArgs {
  CacheView cache;
  TableView rows;
  const int32_t* cu;
  int sequences;
  int64_t tokens, max_length;
  const char* q; int64_t q_tok, q_head;  // bytes
  char* o; int64_t o_tok, o_head;
  int hq, group;
  float scale_log2;  // |scale| log2(e), 1 for a scale of zero
  float q_sign;      // of the scale
  int64_t window, sinks;
  const float* w_in;
  float* w_out;
  float2v* stats;  // [tokens][hq]: greatest q . k and 1 / sum; +inf and 0 where a row sees nothing
  int max_new, blocks;      // new tokens of a sequence at most; row blocks of as many
  int workers;              // ranges
  int4* units;              // [sequences][blocks][kv heads]: first, last worker, slot of the first
  float* part_ml;           // [workers][2][block rows][2]
  float* part_o;            // [workers][2][block rows][128]
  float* scores;            // [sequences][kv heads][score_rows][score_keys]
  int score_rows;
  int64_t score_keys;
};

template <class T>
using Vec8 = T __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float4v mfma(Vec8<half_t> a, Vec8<half_t> b, float4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float4v mfma(Vec8<bhalf_t> a, Vec8<bhalf_t> b, float4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Powers of two that P is raised by: fp16 holds 2^-14 .. 2^15 in full, and the many small
// weights beside a large one count together.
template <class T>
constexpr float kLift = std::is_same<T, half_t>::value ? 15.f : 0.f;

// What the weights need of a row, from its maximum and its (lifted) sum.
template <class T>
__device__ __forceinline__ float2v row_stats(float top, float sum, float inverse) {
  return sum == 0.f ? float2v{INFINITY, 0.f} : float2v{top, inverse * __builtin_exp2f(kLift<T>)};
}

// Over the four lane groups: each swap leaves a pair of rows (halves) of lanes side by side.
template <class F>
__device__ __forceinline__ float over_groups(float v, F f) {
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto rows = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  u = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, (uint32_t)rows[0]),
                                     __builtin_bit_cast(float, (uint32_t)rows[1])));
  const auto halves = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return f(__builtin_bit_cast(float, (uint32_t)halves[0]),
           __builtin_bit_cast(float, (uint32_t)halves[1]));
}
__device__ __forceinline__ float group_max(float v) {
  return over_groups(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float group_sum(float v) {
  return over_groups(v, [](float a, float b) { return a + b; });
}
// Sums over the lanes up to and with each.
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t add_moved(int64_t v) {
  const uint32_t low = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
  const uint32_t high = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false);
  return v + (int64_t)((uint64_t)high << 32 | low);
}
__device__ __forceinline__ int64_t lanes_upto(int64_t v) {
  v = add_moved<0x111, 0xf>(v);  // lanes 1, 2, 4, 8 below in the row
  v = add_moved<0x112, 0xf>(v);
  v = add_moved<0x114, 0xf>(v);
  v = add_moved<0x118, 0xf>(v);
  v = add_moved<0x142, 0xa>(v);  // the last lane of rows 0 and 2 to rows 1 and 3
  return add_moved<0x143, 0xc>(v);  // and of row 1 to rows 2 and 3
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t add_moved(uint32_t v) {
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t lanes_upto(uint32_t v) {
  v = add_moved<0x111, 0xf>(v);
  v = add_moved<0x112, 0xf>(v);
  v = add_moved<0x114, 0xf>(v);
  v = add_moved<0x118, 0xf>(v);
  v = add_moved<0x142, 0xa>(v);
  return add_moved<0x143, 0xc>(v);
}
// a / b of numbers from 0 and 1 up: seldom more than 32 bits.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)v) |
                   (uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32);
}

__device__ __forceinline__ int clamp_to(int64_t v, int64_t lo, int64_t hi) {
  return (int)(v < lo ? lo : v > hi ? hi : v);
}

// The new tokens of sequence b, and the cache rows they see.
struct Sequence {
  int start, n, len;  // first packed token, tokens, cache rows
  int64_t at;         // cache row of the first token
  Sequence() = default;
  __device__ __forceinline__ Sequence(const CachedAttnArgs& a, int b) {
    const int64_t c0 = clamp_to(a.cu[b], 0, a.tokens), c1 = clamp_to(a.cu[b + 1], 0, a.tokens);
    start = (int)c0;
    n = (int)(c1 > c0 ? c1 - c0 : 0);
    len = (int)a.rows.length(b, a.cache.page_size, a.max_length);
    at = (int64_t)a.rows.lengths[b] - a.cu[b + 1] + c0;
  }
  __device__ __forceinline__ void settle() {  // into scalar registers
    start = uniform(start);
    n = uniform(n);
    len = uniform(len);
    at = uniform(at);
  }
  // Token i sees [low(i), last(i)] and below last(i) the sinks.
  __device__ __forceinline__ int last(int i) const { return clamp_to(at + i, -1, len - 1); }
  __device__ __forceinline__ int low(const CachedAttnArgs& a, int i) const {
    return a.window ? clamp_to(at + i - a.window + 1, 0, len) : 0;
  }
};

// The tiles that a block of query rows has to visit: those of the sinks, then from the
// first token's window to the last token's row.
struct Span {
  int i0, i1;     // tokens of the block
  int low, high;  // rows [low, high) and the sinks below low
  int sink_tiles, first, tiles;
  int clear_low, clear_end, sinks;  // what every row of the block sees: [clear_low, clear_end), sinks
  __device__ __forceinline__ Span(const CachedAttnArgs& a, const Sequence& s, int block,
                                  int block_rows) {
    const int rows = min(s.n, a.max_new) * a.group;
    const int r0 = block * block_rows;
    i0 = r0 / a.group;
    i1 = (min(rows, r0 + block_rows) - 1) / a.group;
    tiles = low = high = sink_tiles = first = clear_low = clear_end = 0;
    sinks = clamp_to(a.sinks, 0, s.len);
    if (r0 >= rows) return;
    high = s.last(i1) + 1;
    clear_end = s.last(i0) + 1;
    clear_low = s.low(a, i1);
    low = min(s.low(a, i0), high);
    sink_tiles = (clamp_to(a.sinks, 0, low) + kKeys - 1) / kKeys;
    first = max(low / kKeys, sink_tiles);
    tiles = sink_tiles + max((high + kKeys - 1) / kKeys - first, 0);
    // A block that sees nothing still has its zeros to write, and does so over tile 0: the one
    // behind the last row would put its scores behind the score row's end.
    if (!tiles) first = 0, tiles = 1;
  }
  // Whether every row sees the whole tile from row j on.
  __device__ __forceinline__ bool clear(int j) const {
    return j + kKeys <= clear_end && (j >= clear_low || j + kKeys <= sinks);
  }
  __device__ __forceinline__ int tile(int x) const {
    return x < sink_tiles ? x : x - sink_tiles + first;
  }
};

// The kernel's arguments, loaded where they are used and not kept in registers until then.
typedef const __attribute__((address_space(4))) CachedAttnArgs LateArgs;
__device__ __forceinline__ LateArgs* late_args() {
  auto p = (LateArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// A workgroup's tiles [x0, x1) of a unit.
struct Segment {
  int line, kv, x0, x1, slot;
  bool whole;
  Sequence seq;
};

// What the workgroup's waves leave for each other, and 64 lines (sequence, block) of the split.
template <int QT, int W>
struct Results {
  float m[W][16 * QT], l[W][16 * QT];
  int64_t upto[64];
  int tiles[64];
  Sequence seq[64];
  Segment mine;
  bool equal;
};

typedef __amdgpu_buffer_rsrc_t Rsrc;

// The 16 cache rows of half tile h of a wave, whose first one's address lane h holds (with
// the top bit set where no page holds them: addresses have 48).
struct Halves {
  uint32_t low, high;
  __device__ __forceinline__ void set(const char* at, bool held) {
    low = (uint32_t)(uintptr_t)at;
    high = (uint32_t)((uintptr_t)at >> 32) | (held ? 0u : 0x80000000u);
  }
  __device__ __forceinline__ bool held(int h) const {
    return (int)__builtin_amdgcn_readlane(high, h) >= 0;
  }
  __device__ __forceinline__ Rsrc rows(int h) const {
    const uint32_t lo = __builtin_amdgcn_readlane(low, h), hi = __builtin_amdgcn_readlane(high, h);
    return __builtin_amdgcn_make_buffer_rsrc((void*)((uint64_t)hi << 32 | lo), 0, ~((int)hi >> 31),
                                             0x00027000);
  }
};
template <bool ONCE>
__device__ __forceinline__ u32x4 load16(Rsrc r, uint32_t lane, uint32_t all) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, lane, all, ONCE * 2));
}
// The operand of columns 8 c + e from eight keys' rows, two keys a register.
__device__ __forceinline__ u32x4 turned(const u32x4 (&v)[8], int e) {
  u32x4 out;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    out[i] = __builtin_amdgcn_perm(v[2 * i + 1][e >> 1], v[2 * i][e >> 1],
                                   e & 1 ? 0x07060302u : 0x05040100u);
  return out;
}

// The join of a unit's waves, whose (m, l) are in lds and o in waves[w].o: the result where the
// range is the whole unit, a partial one in the workspace elsewhere.
template <class T, int QT, int W, int RW, class Wave>
__device__ __forceinline__ void finish_unit(const Results<QT, W>& lds, const Wave (&waves)[W],
                                            int thread, int block, int block_row, int rows, int kv,
                                            const Sequence& seq, const Span& span, int x1,
                                            bool whole, int slot) {
  __syncthreads();

  LateArgs* late = late_args();
  const int group = late->group;
  // Columns of a thread and row: fewer where threads would have none.
  constexpr int kCols = 16 * QT * RW * 16 <= 32 * W ? 4 : 8;
  constexpr int kPieces = kCacheDim / kCols;
  typedef T Out __attribute__((ext_vector_type(kCols)));
  for (int item = thread; item < 16 * QT * RW * kPieces; item += 64 * W) {
    const int line = item / kPieces, c = item % kPieces * kCols;
    if (block_row + line >= rows) continue;
    const int half = line / (16 * QT), r = line % (16 * QT);
    float top = -INFINITY;
#pragma unroll
    for (int w = half; w < W; w += RW) top = fmaxf(top, lds.m[w][r]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, o[kCols] = {};
#pragma unroll
    for (int w = half; w < W; w += RW) {
      const float f = __builtin_amdgcn_exp2f((lds.m[w][r] - base) * late->scale_log2);
      sum += f * lds.l[w][r];
#pragma unroll
      for (int q = 0; q < kCols; q += 4) {
        const float4v x = *reinterpret_cast<const float4v*>(&waves[w].o[r][c + q]);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[q + i] += f * x[i];
      }
    }
    if (whole) {
      const int i = (block_row + line) / group;
      const int head = kv * group + block_row + line - i * group;
      const float inverse = sum == 0.f ? 0.f : 1.f / sum;
      Out out;
#pragma unroll
      for (int e = 0; e < kCols; ++e) out[e] = (T)(sum == 0.f ? 0.f : o[e] * inverse);
      *reinterpret_cast<Out*>(late->o + (int64_t)(seq.start + i) * late->o_tok + head * late->o_head +
                              c * 2) = out;
      if (late->stats && c == 0)
        late->stats[(int64_t)(seq.start + i) * late->hq + head] = row_stats<T>(base, sum, inverse);
    } else {
      const int64_t part = (int64_t)slot * 16 * QT * RW + line;
      float* out = late->part_o + part * kCacheDim + c;
#pragma unroll
      for (int q = 0; q < kCols; q += 4)
        *reinterpret_cast<float4v*>(out + q) = float4v{o[q], o[q + 1], o[q + 2], o[q + 3]};
      if (c == 0) *reinterpret_cast<float2v*>(late->part_ml + part * 2) = float2v{top, sum};
    }
  }
  // Tokens behind the bound on a sequence's new ones have no part in the call.
  if (whole || x1 == span.tiles)
    if (seq.n > late->max_new && block == late->blocks - 1)
      for (int64_t i = thread; i < (int64_t)(seq.n - late->max_new) * group * 16; i += 64 * W) {
        const int64_t r = i / 16 + (int64_t)late->max_new * group;
        const int64_t t = r / group;
        const int64_t at = (seq.start + t) * late->o_tok + (kv * group + r - t * group) * late->o_head;
        *reinterpret_cast<u32x4*>(late->o + at + (i & 15) * 16) = u32x4{0, 0, 0, 0};
      }
}

// Zeros for packed tokens that no sequence has.
template <int W>
__device__ __forceinline__ void clear_outside(const CachedAttnArgs& a) {
  const int64_t head = clamp_to(a.cu[0], 0, a.tokens);
  const int64_t tail = clamp_to(a.cu[a.sequences], 0, a.tokens);
  const int64_t per = (int64_t)a.hq * 16;
  for (int64_t i = threadIdx.x; i < (head + a.tokens - tail) * per; i += 64 * W) {
    int64_t t = i / per;
    const int64_t c = i - t * per;
    if (t >= head) t += tail - head;
    *reinterpret_cast<u32x4*>(a.o + t * a.o_tok + c / 16 * a.o_head + (c & 15) * 16) =
        u32x4{0, 0, 0, 0};
  }
}

// Zeros for every token of a call without sequences.
constexpr int kZeroRows = 16;  // of a workgroup
__global__ __launch_bounds__(256) void cached_zeros_kernel(CachedAttnArgs a) {
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x, row = item / (256 / kZeroRows);
  if (row >= a.tokens * a.hq) return;
  const int64_t t = row / a.hq;
  *reinterpret_cast<u32x4*>(a.o + t * a.o_tok + (row - t * a.hq) * a.o_head + (item & 15) * 16) =
      u32x4{0, 0, 0, 0};
}

// Units cut into equal parts, each a workgroup's (`mine`, with x1 0 where there is none left):
// true where that is done.  A range that holds the end of one unit and the start of another goes through
// both one after the other, 5 us more than the others take.  Parts of up to as many tiles as
// a range has places (its units' starts counted) are therefore better, if there are workgroups
// for all of them; with few units there are.  For one wave.
template <int QT, int RW>
__device__ __forceinline__ bool equal_parts(const CachedAttnArgs& a, Segment& mine) {
  constexpr int kMostTiles = 1 << 22;  // of a unit: sums over 128 units are 32-bit numbers
  const int hk = a.cache.kv_heads, lane = threadIdx.x & 63;
  const int lines = a.sequences * a.blocks;
  Sequence seq{};
  uint32_t tiles = 0;
  if (lane < lines) {
    const int b = lane / a.blocks;
    seq = Sequence(a, b);
    tiles = Span(a, seq, lane - b * a.blocks, 16 * QT * RW).tiles;
  }
  if (__any(tiles > kMostTiles)) return false;
  auto all = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); };
  const uint32_t workers = a.workers, total = all(lanes_upto(tiles)) * hk;
  const uint32_t starts = (uint32_t)__popcll(__ballot(tiles > 0)) * hk * kStart;
  const uint32_t least = (total + workers - 1) / workers;
  const uint32_t most = max((total + starts + workers - 1) / workers, (uint32_t)kMinRange);
  // The largest parts first, which fit if any do, then the smallest that do.
  uint32_t parts = 0, upto = 0;
  auto fit = [&](uint32_t size) {
    parts = (tiles + size - 1) / size;
    upto = lanes_upto(parts) * hk;
    return all(upto) <= workers;
  };
  if (!fit(most)) return false;
#pragma unroll 1
  for (uint32_t i = 0; i < 4; ++i)
    if (fit(max(least + (most - least) * i / 3, 1u))) break;
  mine.x1 = 0;
  if (blockIdx.x >= all(upto)) return true;
  const int at = uniform(__ffsll((long long)__ballot(upto > blockIdx.x)) - 1);
  auto of_line = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, at); };
  parts = of_line(parts);
  tiles = of_line(tiles);
  const uint32_t within = blockIdx.x - of_line(upto) + parts * hk;
  const uint32_t kv = within / parts, part = within - kv * parts;
  mine.line = at;
  mine.kv = kv;
  mine.x0 = (int)((uint64_t)tiles * part / parts);
  mine.x1 = (int)((uint64_t)tiles * (part + 1) / parts);
  mine.whole = parts == 1;
  mine.slot = 2 * (int)blockIdx.x;
  mine.seq.start = of_line(seq.start);
  mine.seq.n = of_line(seq.n);
  mine.seq.len = of_line(seq.len);
  mine.seq.at = (int64_t)((uint64_t)of_line((uint32_t)seq.at) |
                          (uint64_t)of_line((uint32_t)(seq.at >> 32)) << 32);
  if (part == 0 && lane == 0)
    a.units[(int64_t)at * hk + kv] = int4{(int)blockIdx.x, (int)(blockIdx.x + parts) - 1, 0, 0};
  return true;
}

// The workgroup's range of the line of all units' tiles (PARTS: or its equal part), as calls of
// unit_of.
template <int QT, int W, int RW, bool PARTS, class F>
__device__ __forceinline__ void for_ranges(const CachedAttnArgs& a, Results<QT, W>& lds, F unit_of) {
  const int hk = a.cache.kv_heads;
  Segment mine;
  bool equal = false;
  if constexpr (PARTS) {
    // (Where there are at most half as many units as workgroups.)
    if (a.sequences * a.blocks <= 64 && 2 * a.sequences * a.blocks * hk <= a.workers) {
      if (threadIdx.x < 64) {
        equal = equal_parts<QT, RW>(a, mine);
        if (threadIdx.x == 0) lds.equal = equal, lds.mine = mine;
      }
      __syncthreads();
      equal = uniform((int)lds.equal);
      if (equal) {
        mine = lds.mine;
        mine.line = uniform(mine.line);
        mine.kv = uniform(mine.kv);
        mine.x0 = uniform(mine.x0);
        mine.x1 = uniform(mine.x1);
        mine.slot = uniform(mine.slot);
        mine.whole = uniform((int)mine.whole);
        mine.seq.settle();
      }
    }
  }
  // Lines (sequence, block), 64 at a time: the places of each, and up to and with it.
  const int lane = threadIdx.x & 63;
  const int lines = a.sequences * a.blocks;
  auto scan = [&](int first) {
    __syncthreads();
    if (threadIdx.x < 64) {
      uint32_t places = 0;
      if (first + lane < lines) {
        const int b = (first + lane) / a.blocks;
        const Sequence seq(a, b);
        places = Span(a, seq, first + lane - b * a.blocks, 16 * QT * RW).tiles;
        lds.seq[lane] = seq;
        lds.tiles[lane] = places;
        if (places) places += kStart;
      }
      lds.upto[lane] = lanes_upto((int64_t)places);
    }
    __syncthreads();
  };
  int64_t total = 0;
  if (!equal) {
#pragma unroll 1
    for (int first = (lines - 1) / 64 * 64; first >= 0; first -= 64) {
      scan(first);
      total += lds.upto[63];
    }
  }
  total = uniform(total) * hk;
  const int64_t range = max(uniform(quotient(total + a.workers - 1, a.workers)),
                            (int64_t)kMinRange);
  const int64_t begin = uniform((int64_t)(blockIdx.x * range));
  const int64_t end = min(begin + range, total);
  int base = 0;
  int64_t before = 0;  // places (of one kv head) of the lines before these 64
  for (int64_t pos = begin; equal || pos < end;) {
    if (equal) {
      if (!mine.x1) break;
    } else {
      while (pos >= (before + uniform(lds.upto[63])) * hk) {
        before += uniform(lds.upto[63]);
        base += 64;
        scan(base);
      }
      const int at =
          uniform(__ffsll((long long)__ballot((before + lds.upto[lane]) * hk > pos)) - 1);
      const int tiles = uniform(lds.tiles[at]);
      const int64_t line_start = (before + uniform(lds.upto[at]) - tiles - kStart) * hk;
      mine.kv = uniform((int)quotient(pos - line_start, tiles + kStart));
      const int64_t unit = line_start + (int64_t)mine.kv * (tiles + kStart);
      mine.x0 = max((int)(pos - unit) - kStart, 0);
      mine.x1 = (int)min((int64_t)tiles, end - unit - kStart);
      mine.line = base + at;
      pos = unit + kStart + mine.x1;
      if (mine.x1 <= mine.x0) break;  // the range ends before the unit's first tile
      mine.whole = mine.x0 == 0 && mine.x1 == tiles;
      mine.slot = (int)(2 * blockIdx.x + (unit > begin));
      if (mine.x0 == 0 && threadIdx.x == 0)
        a.units[(int64_t)mine.line * hk + mine.kv] =
            int4{(int)blockIdx.x, (int)quotient(unit + kStart + tiles - 1, range), unit > begin, 0};
      mine.seq = lds.seq[at];
      mine.seq.settle();
    }
    const int b = uniform(mine.line / a.blocks), block = mine.line - b * a.blocks;
    const Span span(a, mine.seq, block, 16 * QT * RW);
    unit_of(b, block, mine.kv, mine.seq, span, mine.x0, mine.x1, mine.whole, mine.slot);
    if (equal) break;
    if (pos < end) __syncthreads();  // the waves' results are read before the next ones come
  }
}

// The unit of a workgroup that has one for itself.
template <int QT, int RW, class F>
__device__ __forceinline__ void for_unit(const CachedAttnArgs& a, F unit_of) {
  const int hk = a.cache.kv_heads;
  const int line = uniform((int)(blockIdx.x / hk)), kv = (int)(blockIdx.x - line * hk);
  const int b = uniform(line / a.blocks), block = line - b * a.blocks;
  Sequence seq(a, b);
  seq.settle();
  const Span span(a, seq, block, 16 * QT * RW);
  if (span.tiles)
    unit_of(b, block, kv, seq, span, 0, span.tiles, true, 0);
}

// Four columns of a query row, from its parts' sums under the maximum `base`.
template <class T>
__device__ __forceinline__ void store_joined(const CachedAttnArgs& a, const Sequence& seq, int kv,
                                             int row, int c, float4v o, float sum, float base) {
  const int i = row / a.group;
  const int head = kv * a.group + row - i * a.group;
  T* out = reinterpret_cast<T*>(a.o + (int64_t)(seq.start + i) * a.o_tok + head * a.o_head) + 4 * c;
  const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(sum == 0.f ? 0.f : o[e] * inverse);
  if (a.stats && c == 0)
    a.stats[(int64_t)(seq.start + i) * a.hq + head] = row_stats<T>(base, sum, inverse);
}

struct JoinShared {
  float4v sums[8][32];
  float ml[8][2];
};

// Parts of a unit that crosses ranges, row `at` of its block: 32 lanes of 4 columns for every
// eighth part, joined in the order of the ranges.
template <class T, int ROWS>
__device__ __forceinline__ void join_row(const CachedAttnArgs& a, JoinShared& lds,
                                         const Sequence& seq, int4 unit, int block, int kv,
                                         int at) {
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  float4v o{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
#pragma unroll 4
  for (int w = unit.x + g; w <= unit.y; w += 8) {
    const int64_t p = (int64_t)(2 * w + (w == unit.x ? unit.z : 0)) * ROWS + at;
    const float2v s = *reinterpret_cast<const float2v*>(a.part_ml + p * 2);
    const float4v x = *reinterpret_cast<const float4v*>(a.part_o + p * kCacheDim + 4 * c);
    const float top = fmaxf(m, s[0]), base = top == -INFINITY ? 0.f : top;
    const float f = __builtin_amdgcn_exp2f((m - base) * a.scale_log2);
    const float h = __builtin_amdgcn_exp2f((s[0] - base) * a.scale_log2);
    o = o * f + x * h;
    l = l * f + s[1] * h;
    m = top;
  }
  lds.sums[g][c] = o;
  if (c == 0) lds.ml[g][0] = m, lds.ml[g][1] = l;
  __syncthreads();
  if (g) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, lds.ml[i][0]);
  const float base = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
  o = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = __builtin_amdgcn_exp2f((lds.ml[i][0] - base) * a.scale_log2);
    sum += f * lds.ml[i][1];
    o += f * lds.sums[i][c];
  }
  store_joined<T>(a, seq, kv, block * ROWS + at, c, o, sum, base);
}

template <class T, int ROWS>
__global__ __launch_bounds__(256) void cached_join_kernel(CachedAttnArgs a) {
  __shared__ JoinShared lds;
  const int hk = a.cache.kv_heads;
  const int line = (int)(blockIdx.x / hk), kv = (int)(blockIdx.x - line * hk);
  const int b = line / a.blocks, block = line - b * a.blocks;
  const int4 unit = a.units[blockIdx.x];
  const Sequence seq(a, b);
  if (block * ROWS + (int)blockIdx.y >= min(seq.n, a.max_new) * a.group || unit.x == unit.y) return;
  join_row<T, ROWS>(a, lds, seq, unit, block, kv, blockIdx.y);
}

// Waves of a workgroup side by side on the query rows of a block: one as long as a sequence
// has at most 32.
constexpr int kWaves = 8;
static_assert(kScoreRows == 16, "scores are kept by blocks of 16 rows only");

// How a call is laid out, from what the host knows.
struct Layout {
  int max_new, block_rows, blocks, workers;  // query rows of a block; workers 0: one workgroup a unit
  int64_t units;
  int score_rows;           // 0: no scores kept
  int64_t score_keys;
  size_t stats, list, ml, o, scores, bytes;  // workspace offsets
  // whole: whether the units are a workgroup's each, from the query rows of a unit, the units, the
  // CUs and the tiles that a wave then has.
  template <class Whole>
  Layout(int rows, int64_t tokens, int q_heads, int kv_heads, int new_bound, int64_t max_length,
         bool weights, Whole whole, int widest = 128) {
    max_new = (int)(new_bound < tokens ? new_bound : tokens);
    const int64_t of_sequence = (int64_t)(max_new > 0 ? max_new : 1) * (q_heads / kv_heads);
    // A wave takes 16 rows, or 32, and up to four waves of 32 share a tile: 33 new tokens of 4
    // sequences (231 rows) 36 us in blocks of 128, 39 in blocks of 64.
    block_rows = of_sequence <= 16 ? 16 : of_sequence <= 32 ? 32 : of_sequence <= 64 ? 64 : widest;
    blocks = (int)cdiv(of_sequence, block_rows);
    units = (int64_t)rows * blocks * kv_heads;
    const int stripes = kWaves / (block_rows <= 32 ? 1 : block_rows / 32);
    const int unit_rows = (int)(of_sequence < block_rows ? of_sequence : block_rows);
    workers = whole(unit_rows, units, device_cu_count(), cdiv(max_length, kKeys * stripes))
                  ? 0 : device_cu_count();
    score_keys = cdiv(max_length > 0 ? max_length : 1, kKeys) * kKeys;
    score_rows = 0;
    if (weights && of_sequence <= kScoreRows &&
        (size_t)rows * kv_heads * of_sequence * score_keys * 4 <= kScoreBytes)
      score_rows = (int)of_sequence;
    bytes = 0;
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) / 256 * 256;
      return at;
    };
    stats = take(weights ? (size_t)tokens * q_heads * sizeof(float2v) : 0);
    list = take(workers ? (size_t)units * sizeof(int4) : 0);
    ml = take((size_t)workers * 2 * block_rows * 2 * 4);
    o = take((size_t)workers * 2 * block_rows * kCacheDim * 4);
    scores = take((size_t)rows * kv_heads * score_rows * score_keys * 4);
  }
};

}  // namespace
}  // namespace ss
