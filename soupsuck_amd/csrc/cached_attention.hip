// Attention of new tokens over a paged key-value cache.
//
// o = sum_j softmax_j(scale q . k_j) v_j over the rows j that the token at row p sees
// (j <= p, and inside the window or among the sinks), with a running maximum and sum in
// fp32: m' = max(m, s), l' = l 2^(c (m - m')) + 2^(c (s - m')), o' likewise, s = q . k and
// c = |scale| log2(e).  The maximum is taken off before the scale, here, in the joins and for
// the weights: c s would be rounded to steps of whole powers of two at |c s| = 2^24, and two
// such roundings against each other take a weight past what fp16 holds; s - m' is exact at
// the top and next to it.
//
// A unit of work is one kv head over one block of a sequence's query rows (token-major, the
// q heads of the group side by side: all of them share the cache's rows, which are read
// once for the block).  Its keys go in tiles of 32, dealt to the waves of a workgroup in
// turn; each wave keeps its own (m, l, o) in registers and meets the others only at the
// end, so no barrier stands between two loads.
//
// Products (v_mfma_f32_16x16x32): S^T = K Q^T, keys down, one query row per lane and
// column; the accumulator of two 16-key halves is the operand P^T of O^T += V^T P^T as it
// stands, slots 8 h .. + 7 of lane group h being keys 4 h + i and 16 + 4 h + i.  V is read
// as whole rows (lane c of a group takes columns 8 c .. + 7 of a key) and turned in
// registers: tile e of O^T holds the columns 8 c + e.  K goes by DMA to a place in LDS that the
// wave has for itself and is the operand from there.
//
// What bounds it: HBM, at which rate a CU gets 10 to 13 bytes a clock; against that the 32 permutes
// and 16 MFMAs of a 16 KiB tile are small (from L2 the same loop runs at 21 TB/s), and what
// counts is the loads in flight: 16 KiB a wave, the next tile's keys issued before this
// one's softmax and its values before the next scores.  131071 keys, 28 / 4 heads (268 MB):
// 48 us and 5 us for the join, 5.1 TB/s in all and 6.2 in the loop; 64 sequences of 7800
// (1.02 GB) 164 us, 6.2 TB/s.  Short ones are latency: 518 keys 8.9 us.
//
// Split over the keys (cached_attention_kernel<.., true>): the tiles of all units form one
// line that is cut into equal ranges, one a workgroup, from the lengths on the device, so
// that one long sequence and a batch of ragged ones load every CU alike whatever the
// bounds that the host knows.  A unit inside a range is finished there; of one that
// crosses ranges each part leaves (o, m, l), and cached_join_kernel adds them up.
// Bounds on the length that give a wave at most four tiles take one workgroup a unit and no
// second launch.
//
// Masked rows: a tile that every query row sees whole takes no mask.  In the others scores
// are replaced (never multiplied) by -inf and the values of rows that no query row sees by
// 0, so that nothing stored there counts.  In a row that some tokens of a wave see and others
// do not an infinity or NaN would reach the others as 0 times it: such values are taken as 0
// there, and added at the end to the rows that see them.
//
// Weights: the scores (fp32, base 2) are left in the workspace, 4 bytes a query row and
// key against 256 for the key again, and added up once the statistics are known.  The
// stores cost more than their bytes (148 us without, 183 with 50 MB of them in 918).  Where
// the scores would be many (more than kScoreRows query rows a kv head, or more than
// kScoreBytes in all) the keys are multiplied again.
#include <algorithm>
#include <type_traits>

#include "paged.h"
#include "elementwise.h"

namespace ss {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeys = 32;       // of a tile
constexpr int kRowBytes = kCacheDim * 2;
constexpr int kPadDim = kCacheDim + 4;  // fp32 row of the waves' results in LDS
// Tiles of a wave up to which a unit is one workgroup's.  So and cut, one sequence and eight, us:
// 6 query rows a kv head (4 tiles are 1024 keys) 1000 keys 11.9 / 12.5 and 12.4 / 14.7, 2000 keys
// 16.5 / 13.9 and 20.8 / 15.0; 30 rows, 500 keys 13.0 / 15.4 and 13.4 / 17.1, 1100 keys 16.2 / 15.8
// and 16.4 / 17.3; 54 rows (512 keys) 500 keys 16.0 / 16.3 and 16.3 / 18.7, 700 keys 17.5 / 16.4 and
// 17.8 / 18.7; 198 rows (256 keys) 250 keys 16.6 / 20.0 and 17.4 / 25.3.
constexpr int kWholeTiles = 4;
// Query rows of a kv head up to which their scores are kept (those of one 16-row block): kept
// and with the keys again, 64 sequences of 7000 keys with 7 rows 196 and 249 us, 14 rows 215 and
// 252, 16 rows (two kv heads) 117 and 135; 4 of them 27.9 / 32.4, 32.7 / 33.6, 25.2 / 26.8; 4 of
// 1000 18.1 / 17.4, 22.0 / 18.3, 18.0 / 18.1.  4 sequences with 28 rows took 60 and 34.
constexpr int kScoreRows = 16;
constexpr size_t kScoreBytes = (size_t)512 << 20;
constexpr int kSteps = 31;      // tiles of a wave whose pages are looked up at once
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

template <class T, int QT, int W, int RW>
struct Shared {
  // A wave's keys while it goes through its tiles, then its results.
  union {
    float o[16 * QT][kPadDim];
    char keys[kKeys * kRowBytes];
  } wave[W];
  float m[W][16 * QT], l[W][16 * QT];
  int64_t upto[64];
  int tiles[64];
  Sequence seq[64];
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
// The lanes' 16 bytes to lds, side by side.
template <bool ONCE>
__device__ __forceinline__ void load16_to(char* lds, Rsrc r, uint32_t lane, uint32_t all) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      r, (__attribute__((address_space(3))) void*)lds, 16, lane, all, 0, ONCE * 2);
}

// Whether two 16-bit values hold an infinity or NaN (in the upper bits of each).
template <class T>
__device__ __forceinline__ uint32_t not_finite(uint32_t v) {
  constexpr uint32_t least = std::is_same<T, half_t>::value ? 0x04000400u : 0x00800080u;
  return ((v & 0x7fff7fffu) + least) & 0x80008000u;
}

template <class T>
__device__ __forceinline__ float value(uint32_t v) {
  return (float)__builtin_bit_cast(T, (uint16_t)v);
}

// The infinities and NaN that a wave's products left out, to the rows that see them (two
// columns a lane): its tiles again, rarely.
template <class T, int QT>
__device__ __noinline__ void add_left_out(LateArgs* late, float (*o)[kPadDim], int b, Sequence seq,
                                          Span span, int kv, int r0, int x, int x_end, int stripes) {
  CachedAttnArgs a;
  __builtin_memcpy(&a, (const void*)late, sizeof a);
  const int lane = threadIdx.x & 63, size = a.cache.page_size;
  const int rows = min(16 * QT, min(seq.n, a.max_new) * a.group - r0);
  const char* v_base = a.cache.v + (int64_t)kv * a.cache.v_head + lane * 4;
  for (; x < x_end; x += stripes) {
    const int j0 = span.tile(x) * kKeys;
    const bool clear = span.clear(j0) && a.rows.page(b, j0 / size, a.cache.pages) >= 0 &&
                       a.rows.page(b, (j0 + 16) / size, a.cache.pages) >= 0;
    for (int j = j0; j < min(j0 + kKeys, seq.len) && !clear; ++j) {
      const int entry = j / size;
      const int page = a.rows.page(b, entry, a.cache.pages);
      if (page < 0) continue;
      const uint32_t v = *reinterpret_cast<const uint32_t*>(
          v_base + (int64_t)page * a.cache.v_page + (int64_t)(j - entry * size) * a.cache.v_row);
      const uint32_t odd = not_finite<T>(v);
      if (!odd) continue;
      for (int r = 0; r < rows; ++r) {
        const int i = (r0 + r) / a.group;
        if (j > seq.last(i) || (j < seq.low(a, i) && j >= a.sinks)) continue;
        if (odd & 0x8000u) o[r][2 * lane] += value<T>(v);
        if (odd >> 31) o[r][2 * lane + 1] += value<T>(v >> 16);
      }
    }
  }
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

// The tiles [x0, x1) of a unit by the waves of the workgroup, and their join: the result
// where the range is the whole unit, a partial one in the workspace elsewhere.
template <class T, int QT, int W, int RW, bool SCORES, bool ONCE>
__device__ __forceinline__ void attend(const CachedAttnArgs& a, Shared<T, QT, W, RW>& lds, int b,
                                       int block, int kv, const Sequence& seq, const Span& span,
                                       int x0, int x1, bool whole, int slot) {
  // Opaque, or all that follows from them is computed ahead of the segments' loop and kept
  // in registers through it (45 more).
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

  Vec8<T> q[QT][4];  // Q[row][32 ks + 8 grp ..]
  int last[QT], low[QT], token[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = min(r0 + 16 * t + col, rows - 1);
    token[t] = r / a.group;
    const char* p = a.q + (int64_t)(seq.start + token[t]) * a.q_tok +
                    (int64_t)(kv * a.group + r - token[t] * a.group) * a.q_head + grp * 16;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) q[t][ks] = *reinterpret_cast<const Vec8<T>*>(p + ks * 64);
    last[t] = seq.last(token[t]);
    low[t] = seq.low(a, token[t]);
  }
  // The maximum and the masks want a positive scale: a negative one changes the queries' sign
  // (exact), a zero one makes them zeros.
  const float scale = a.scale_log2;
  if (a.q_sign != 1.f) {
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) q[t][ks] *= (T)a.q_sign;
  }
  const int sinks = span.sinks;
  // Keys go through LDS: four whole rows an instruction (as the operand's 16 rows of 64 bytes
  // the same bytes took the texture unit four times as long).  Chunk c of row r lies at c ^ r,
  // so that the 16 rows of an operand's read take different banks.
  char* keys = lds.wave[wave].keys;
  uint32_t k_lane[4];
  int k_read[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    k_lane[i] = (uint32_t)grp * (uint32_t)a.cache.k_row + (col ^ (4 * i + grp)) * 16;
    k_read[i] = col * kRowBytes + ((4 * i + grp) ^ col) * 16;
  }
  const uint32_t v_lane = (uint32_t)(4 * grp) * (uint32_t)a.cache.v_row + col * 16;
  const char* k_base = a.cache.k + (int64_t)kv * a.cache.k_head;
  const char* v_base = a.cache.v + (int64_t)kv * a.cache.v_head;
  float* scores = SCORES ? a.scores + ((int64_t)b * a.cache.kv_heads + kv) * a.score_rows *
                                          a.score_keys
                         : nullptr;

  // Tokens of this wave's rows.
  const int t0 = uniform(min(r0, rows - 1) / a.group);
  const int t1 = uniform(min(r0 + 16 * QT - 1, rows - 1) / a.group);
  const int see_low = seq.low(a, t0), see_high = seq.last(t1) + 1;
  const bool several = t0 != t1;
  uint32_t left_out = 0;
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
    // Some of this wave's tiles at a time: their halves' pages in one load, the last two
    // lanes' none.
#pragma unroll 1
    for (int x = x0 + stripe; x < x_end; x += kSteps * kStripes) {
      const int steps = uniform(min((x_end - x + kStripes - 1) / kStripes, kSteps));
      Halves k_at, v_at;
      {
        int page = -1, row = 0;
        const int j = span.tile(x + (lane >> 1) * kStripes) * kKeys + (lane & 1) * 16;
        if ((lane >> 1) < steps && j < seq.len) {
          const int entry = j / size;
          page = a.rows.page(b, entry, a.cache.pages);
          row = j - entry * size;
        }
        k_at.set(k_base + (int64_t)max(page, 0) * a.cache.k_page + (int64_t)row * a.cache.k_row,
                 page >= 0);
        v_at.set(v_base + (int64_t)max(page, 0) * a.cache.v_page + (int64_t)row * a.cache.v_row,
                 page >= 0);
      }
      u32x4 vf[8];
      // Of a half that no page holds, or behind the last tile, nothing is fetched (or, where
      // the bounds of a load to LDS are not looked at, rows of page 0 that are masked).
      auto load_k = [&](int s) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const Rsrc half = k_at.rows(2 * s + u);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            load16_to<ONCE>(keys + (4 * u + i) * 4 * kRowBytes, half, k_lane[i],
                      4 * i * (uint32_t)a.cache.k_row);
        }
      };
      auto load_v = [&](int s) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const Rsrc half = v_at.rows(2 * s + u);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            vf[4 * u + i] = load16<ONCE>(half, v_lane, i * (uint32_t)a.cache.v_row);
        }
      };
      load_k(0);
      __builtin_amdgcn_sched_barrier(0);  // in the order of the loop's, for its waits
      load_v(0);
#pragma unroll 1
      for (int s = 0; s < steps; ++s) {
        const int j0 = span.tile(x + s * kStripes) * kKeys;
        // This tile's keys have landed: only its values' eight loads may be on their way.
        asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        const bool held0 = k_at.held(2 * s);
        const bool held1 = k_at.held(2 * s + 1);
        float sc[QT][8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float4v c[QT] = {};
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const Vec8<T> k = *reinterpret_cast<const Vec8<T>*>(keys + u * 16 * kRowBytes +
                                                                k_read[ks]);
#pragma unroll
            for (int t = 0; t < QT; ++t) c[t] = mfma(k, q[t][ks], c[t]);
          }
#pragma unroll
          for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[t][4 * u + i] = c[t][i];
        }
        // Not before the products: the next keys take their operands' place.
        __builtin_amdgcn_sched_barrier(0);
        load_k(s + 1);
        if (!(held0 && held1 && span.clear(j0))) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int j = j0 + 4 * grp + (i & 3) + 16 * (i >> 2);
            const bool held = i < 4 ? held0 : held1;
#pragma unroll
            for (int t = 0; t < QT; ++t)
              sc[t][i] = held & (j <= last[t]) & ((j >= low[t]) | (j < sinks)) ? sc[t][i] : -INFINITY;
            const bool seen = held & (j < see_high) & ((j >= see_low) | (j < sinks));
#pragma unroll
            for (int w = 0; w < 4; ++w) vf[i][w] = seen ? vf[i][w] : 0u;
          }
          if (several) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const uint32_t odd = not_finite<T>(vf[i][w]);
                vf[i][w] &= ~((odd >> 15) * 0xffffu);
                left_out |= odd;
              }
          }
        }
        if constexpr (SCORES) {
#pragma unroll
          for (int t = 0; t < QT; ++t)
            if (16 * t + col < rows) {
              float* out = scores + (int64_t)(16 * t + col) * a.score_keys + j0 + 4 * grp;
#pragma unroll
              for (int u = 0; u < 2; ++u)
                *reinterpret_cast<float4v*>(out + 16 * u) = float4v{
                    sc[t][4 * u], sc[t][4 * u + 1], sc[t][4 * u + 2], sc[t][4 * u + 3]};
            }
        }
        Vec8<T> p[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          float top = sc[t][0];
#pragma unroll
          for (int i = 1; i < 8; ++i) top = fmaxf(top, sc[t][i]);
          top = fmaxf(m[t], group_max(top));
          const float base = top == -INFINITY ? 0.f : top;
          if (__any(top > m[t])) {
            const float keep = __builtin_amdgcn_exp2f((m[t] - base) * scale);
            l[t] *= keep;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[t][e] *= keep;
            m[t] = top;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float w =
                __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i] - base, scale, kLift<T>));
            l[t] += w;
            p[t][i] = (T)w;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const Vec8<T> v = __builtin_bit_cast(Vec8<T>, turned(vf, e));
#pragma unroll
          for (int t = 0; t < QT; ++t) acc[t][e] = mfma(v, p[t], acc[t][e]);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_v(s + 1);
      }
      // The loads behind the last tile may still write to the keys' place.
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
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
    add_left_out<T, QT>(late_args(), lds.wave[wave].o, b, seq, span, kv, r0, x0 + stripe, x_end,
                        kStripes);
  __syncthreads();

  LateArgs* late = late_args();
  const int group = late->group;
  for (int item = thread; item < 16 * QT * RW * 16; item += 64 * W) {
    const int line = item >> 4, c = (item & 15) * 8;
    if (block_row + line >= rows) continue;
    const int half = line / (16 * QT), r = line % (16 * QT);
    float top = -INFINITY;
#pragma unroll
    for (int w = half; w < W; w += RW) top = fmaxf(top, lds.m[w][r]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, o[8] = {};
#pragma unroll
    for (int w = half; w < W; w += RW) {
      const float f = __builtin_amdgcn_exp2f((lds.m[w][r] - base) * late->scale_log2);
      sum += f * lds.l[w][r];
      const float4v x = *reinterpret_cast<const float4v*>(&lds.wave[w].o[r][c]);
      const float4v y = *reinterpret_cast<const float4v*>(&lds.wave[w].o[r][c + 4]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i] += f * x[i];
        o[4 + i] += f * y[i];
      }
    }
    if (whole) {
      const int i = (block_row + line) / group;
      const int head = kv * group + block_row + line - i * group;
      const float inverse = sum == 0.f ? 0.f : 1.f / sum;
      Vec8<T> out;
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = (T)(sum == 0.f ? 0.f : o[e] * inverse);
      *reinterpret_cast<Vec8<T>*>(late->o + (int64_t)(seq.start + i) * late->o_tok + head * late->o_head +
                                  c * 2) = out;
      if (late->stats && c == 0)
        late->stats[(int64_t)(seq.start + i) * late->hq + head] = row_stats<T>(base, sum, inverse);
    } else {
      const int64_t part = (int64_t)slot * 16 * QT * RW + line;
      float* out = late->part_o + part * kCacheDim + c;
      *reinterpret_cast<float4v*>(out) = float4v{o[0], o[1], o[2], o[3]};
      *reinterpret_cast<float4v*>(out + 4) = float4v{o[4], o[5], o[6], o[7]};
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
__global__ __launch_bounds__(256) void cached_zeros_kernel(CachedAttnArgs a) {
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x, row = item / 16;
  if (row >= a.tokens * a.hq) return;
  const int64_t t = row / a.hq;
  *reinterpret_cast<u32x4*>(a.o + t * a.o_tok + (row - t * a.hq) * a.o_head + (item & 15) * 16) =
      u32x4{0, 0, 0, 0};
}

template <class T, int QT, int W, int RW, bool SPLIT, bool SCORES, bool ONCE>
__global__ __launch_bounds__(64 * W) void cached_attention_kernel(CachedAttnArgs a) {
  __shared__ Shared<T, QT, W, RW> lds;
  const int hk = a.cache.kv_heads;
  if constexpr (!SPLIT) {
    const int line = uniform((int)(blockIdx.x / hk)), kv = (int)(blockIdx.x - line * hk);
    const int b = uniform(line / a.blocks), block = line - b * a.blocks;
    Sequence seq(a, b);
    seq.settle();
    const Span span(a, seq, block, 16 * QT * RW);
    if (span.tiles)
      attend<T, QT, W, RW, SCORES, ONCE>(a, lds, b, block, kv, seq, span, 0, span.tiles, true, 0);
  } else {
    // Lines (sequence, block), 64 at a time: the places of each, and up to and with it.
    const int lane = threadIdx.x & 63;
    const int lines = a.sequences * a.blocks;
    auto scan = [&](int first) {
      __syncthreads();
      if (threadIdx.x < 64) {
        uint32_t mine = 0;
        if (first + lane < lines) {
          const int b = (first + lane) / a.blocks;
          const Sequence seq(a, b);
          mine = Span(a, seq, first + lane - b * a.blocks, 16 * QT * RW).tiles;
          lds.seq[lane] = seq;
          lds.tiles[lane] = mine;
          if (mine) mine += kStart;
        }
        lds.upto[lane] = lanes_upto(mine);
      }
      __syncthreads();
    };
    int64_t total = 0;
#pragma unroll 1
    for (int first = (lines - 1) / 64 * 64; first >= 0; first -= 64) {
      scan(first);
      total += lds.upto[63];
    }
    total = uniform(total) * hk;
    const int64_t range = max(uniform(quotient(total + a.workers - 1, a.workers)),
                              (int64_t)kMinRange);
    const int64_t begin = uniform((int64_t)(blockIdx.x * range));
    const int64_t end = min(begin + range, total);
    int base = 0;
    int64_t before = 0;  // places (of one kv head) of the lines before these 64
    for (int64_t pos = begin; pos < end;) {
      while (pos >= (before + uniform(lds.upto[63])) * hk) {
        before += uniform(lds.upto[63]);
        base += 64;
        scan(base);
      }
      const int at = uniform(__ffsll((long long)__ballot((before + lds.upto[lane]) * hk > pos)) - 1);
      const int tiles = uniform(lds.tiles[at]);
      const int64_t line_start = (before + uniform(lds.upto[at]) - tiles - kStart) * hk;
      const int kv = uniform((int)quotient(pos - line_start, tiles + kStart));
      const int64_t unit = line_start + (int64_t)kv * (tiles + kStart);
      const int x0 = max((int)(pos - unit) - kStart, 0);
      const int x1 = (int)min((int64_t)tiles, end - unit - kStart);
      const int line = base + at;
      const int b = uniform(line / a.blocks), block = line - b * a.blocks;
      pos = unit + kStart + x1;
      if (x1 <= x0) break;  // the range ends before the unit's first tile
      const bool whole = x0 == 0 && x1 == tiles;
      if (x0 == 0 && threadIdx.x == 0)
        a.units[(int64_t)line * hk + kv] =
            int4{(int)blockIdx.x, (int)quotient(unit + kStart + tiles - 1, range), unit > begin, 0};
      Sequence seq = lds.seq[at];
      seq.settle();
      Span span(a, seq, block, 16 * QT * RW);
      attend<T, QT, W, RW, SCORES, ONCE>(a, lds, b, block, kv, seq, span, x0, x1, whole,
                               2 * blockIdx.x + (unit > begin));
      if (pos < end) __syncthreads();  // the waves' results are read before the next ones come
    }
  }
  if (blockIdx.x == 0) clear_outside<W>(a);
}

// Parts of units that cross ranges: one workgroup a query row, 32 lanes of 4 columns for every
// eighth part, joined in the order of the ranges.
template <class T, int ROWS>
__global__ __launch_bounds__(256) void cached_join_kernel(CachedAttnArgs a) {
  __shared__ float4v sums[8][32];
  __shared__ float ml[8][2];
  const int hk = a.cache.kv_heads;
  const int line = (int)(blockIdx.x / hk), kv = (int)(blockIdx.x - line * hk);
  const int b = line / a.blocks, block = line - b * a.blocks;
  const int row = block * ROWS + blockIdx.y;
  const int4 unit = a.units[blockIdx.x];
  const Sequence seq(a, b);
  if (row >= min(seq.n, a.max_new) * a.group || unit.x == unit.y) return;
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  float4v o{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
#pragma unroll 4
  for (int w = unit.x + g; w <= unit.y; w += 8) {
    const int64_t p = (int64_t)(2 * w + (w == unit.x ? unit.z : 0)) * ROWS + blockIdx.y;
    const float2v s = *reinterpret_cast<const float2v*>(a.part_ml + p * 2);
    const float4v x = *reinterpret_cast<const float4v*>(a.part_o + p * kCacheDim + 4 * c);
    const float top = fmaxf(m, s[0]), base = top == -INFINITY ? 0.f : top;
    const float f = __builtin_amdgcn_exp2f((m - base) * a.scale_log2);
    const float h = __builtin_amdgcn_exp2f((s[0] - base) * a.scale_log2);
    o = o * f + x * h;
    l = l * f + s[1] * h;
    m = top;
  }
  sums[g][c] = o;
  if (c == 0) ml[g][0] = m, ml[g][1] = l;
  __syncthreads();
  if (g) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, ml[i][0]);
  const float base = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
  o = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = __builtin_amdgcn_exp2f((ml[i][0] - base) * a.scale_log2);
    sum += f * ml[i][1];
    o += f * sums[i][c];
  }
  const int i = row / a.group;
  const int head = kv * a.group + row - i * a.group;
  T* out = reinterpret_cast<T*>(a.o + (int64_t)(seq.start + i) * a.o_tok + head * a.o_head) + 4 * c;
  const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(sum == 0.f ? 0.f : o[e] * inverse);
  if (a.stats && c == 0)
    a.stats[(int64_t)(seq.start + i) * a.hq + head] = row_stats<T>(base, sum, inverse);
}

// Weights of 512 cache rows of one kv head from the scores, every 256th to a thread.  The loads
// take no branch, so that several rows' are in flight (with one: a third longer).  64
// sequences with 7 rows, the whole call: 206, 200 and 201 us with 1, 2 and 4 rows a thread.
constexpr int kWeightRows = 2;

__global__ __launch_bounds__(256) void cached_weights_kernel(CachedAttnArgs a) {
  const int64_t cap = (int64_t)a.rows.row_pages * a.cache.page_size;
  const int64_t pieces = cdiv(cap, 256 * kWeightRows), unit = blockIdx.x / pieces;
  const int64_t first = (blockIdx.x - unit * pieces) * 256 * kWeightRows;
  const int b = (int)(unit / a.cache.kv_heads), kv = (int)(unit - (int64_t)b * a.cache.kv_heads);
  const Sequence seq(a, b);
  const int n = first < seq.len ? min(seq.n, a.max_new) : 0;
  float sum[kWeightRows] = {};
  int64_t j[kWeightRows], held[kWeightRows];
#pragma unroll
  for (int e = 0; e < kWeightRows; ++e) {
    j[e] = first + threadIdx.x + 256 * e;
    held[e] = min(j[e], a.score_keys - 1);
    if (a.w_in && j[e] < cap) sum[e] = a.w_in[unit * cap + j[e]];
  }
  const float* scores = a.scores + unit * a.score_rows * a.score_keys;
  for (int i = 0; i < n; ++i) {
    const int last = seq.last(i), low = seq.low(a, i);
    const float2v* stats = a.stats + (int64_t)(seq.start + i) * a.hq + kv * a.group;
    const float* row = scores + (int64_t)i * a.group * a.score_keys;
#pragma unroll 8
    for (int g = 0; g < a.group; ++g)
#pragma unroll
      for (int e = 0; e < kWeightRows; ++e) {
        const float2v s = stats[g];
        const float w = __builtin_amdgcn_exp2f((row[g * a.score_keys + held[e]] - s[0]) *
                                               a.scale_log2) * s[1];
        sum[e] += (j[e] <= last) & ((j[e] >= low) | (j[e] < a.sinks)) ? w : 0.f;
      }
  }
#pragma unroll
  for (int e = 0; e < kWeightRows; ++e)
    if (j[e] < cap) a.w_out[unit * cap + j[e]] = sum[e];
}

// Weights by multiplying the keys again: one wave to 32 cache rows of one kv head, all the
// sequence's query rows in tiles of 16.
template <class T>
__global__ __launch_bounds__(256) void cached_weights_again_kernel(CachedAttnArgs a) {
  const int64_t cap = (int64_t)a.rows.row_pages * a.cache.page_size;
  const int64_t pieces = cdiv(cap, 4 * kKeys), unit = blockIdx.x / pieces;
  const int64_t piece = blockIdx.x - unit * pieces;
  const int b = (int)(unit / a.cache.kv_heads), kv = (int)(unit - (int64_t)b * a.cache.kv_heads);
  const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
  const int col = lane & 15, grp = lane >> 4;
  const int64_t first = (piece * 4 + wave) * kKeys;
  if (first >= cap) return;
  const Sequence seq(a, b);
  const int rows = min(seq.n, a.max_new) * a.group;
  float sum[8] = {};
  if (first < seq.len && rows > 0) {
    const int j0 = (int)first, size = a.cache.page_size;
    Vec8<T> kf[2][4];
    bool held[2];
    const int sinks = clamp_to(a.sinks, 0, seq.len);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = j0 + 16 * u, entry = j / size;
      const int page = j < seq.len ? a.rows.page(b, entry, a.cache.pages) : -1;
      held[u] = page >= 0;
      const char* base = a.cache.k + (int64_t)max(page, 0) * a.cache.k_page +
                         (int64_t)kv * a.cache.k_head + (int64_t)(j - entry * size) * a.cache.k_row +
                         (uint32_t)col * (uint32_t)a.cache.k_row + grp * 16;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        kf[u][ks] = *reinterpret_cast<const Vec8<T>*>(base + ks * 64);
    }
    // The next 16 query rows are on their way while these are multiplied.
    struct Rows {
      Vec8<T> q[4];
      float2v stats;
      int last, low;
    };
    auto rows_from = [&](int r0) {
      Rows x;
      const int r = min(r0 + col, rows - 1), i = r / a.group;
      const int head = kv * a.group + r - i * a.group;
      const char* p = a.q + (int64_t)(seq.start + i) * a.q_tok + head * a.q_head + grp * 16;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) x.q[ks] = *reinterpret_cast<const Vec8<T>*>(p + ks * 64);
      x.stats = a.stats[(int64_t)(seq.start + i) * a.hq + head];
      x.last = r0 + col < rows ? seq.last(i) : -1;
      x.low = seq.low(a, i);
      return x;
    };
    Rows next = rows_from(0);
    for (int r0 = 0; r0 < rows; r0 += 16) {
      Rows now = next;
      if (r0 + 16 < rows) next = rows_from(r0 + 16);
      if (a.q_sign != 1.f)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) now.q[ks] *= (T)a.q_sign;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float4v c{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) c = mfma(kf[u][ks], now.q[ks], c);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + 16 * u + 4 * grp + e;
          const float w = __builtin_amdgcn_exp2f((c[e] - now.stats[0]) * a.scale_log2) *
                          now.stats[1];
          sum[4 * u + e] += held[u] & (j <= now.last) & ((j >= now.low) | (j < sinks)) ? w : 0.f;
        }
      }
    }
  }
  // Over the 16 query rows of a lane group; lane col keeps key col / 8, col % 8 of it.
#pragma unroll
  for (int d = 1; d < 16; d <<= 1)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] += __shfl_xor(sum[e], d, kWave);
  if (col < 8) {
    float mine = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) mine = col == e ? sum[e] : mine;
    const int64_t j = first + 16 * (col >> 2) + 4 * grp + (col & 3);
    const int64_t at = ((int64_t)b * a.cache.kv_heads + kv) * cap + j;
    if (j < cap) a.w_out[at] = (a.w_in ? a.w_in[at] : 0.f) + mine;
  }
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
  Layout(int rows, int64_t tokens, int q_heads, int kv_heads, int new_bound, int64_t max_length,
         bool weights) {
    max_new = (int)(new_bound < tokens ? new_bound : tokens);
    const int64_t of_sequence = (int64_t)(max_new > 0 ? max_new : 1) * (q_heads / kv_heads);
    // A wave takes 16 rows, or 32, and up to four waves of 32 share a tile: 33 new tokens of 4
    // sequences (231 rows) 36 us in blocks of 128, 39 in blocks of 64.
    block_rows = of_sequence <= 16 ? 16 : of_sequence <= 32 ? 32 : of_sequence <= 64 ? 64 : 128;
    blocks = (int)cdiv(of_sequence, block_rows);
    units = (int64_t)rows * blocks * kv_heads;
    const int stripes = kWaves / (block_rows <= 32 ? 1 : block_rows / 32);
    workers = max_length <= kWholeTiles * kKeys * stripes ? 0 : device_cu_count();
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

template <class T, int QT, int RW, bool SCORES, bool ONCE>
int launch_attention(const CachedAttnArgs& a, const Layout& p, hipStream_t st) {
  const dim3 block(64 * kWaves);
  if (!p.workers) {
    hipLaunchKernelGGL((cached_attention_kernel<T, QT, kWaves, RW, false, SCORES, ONCE>),
                       dim3((unsigned)p.units), block, 0, st, a);
    SS_CHECK_LAUNCH("cached_attention_kernel");
    return SS_OK;
  }
  hipLaunchKernelGGL((cached_attention_kernel<T, QT, kWaves, RW, true, SCORES, ONCE>),
                     dim3((unsigned)p.workers), block, 0, st, a);
  SS_CHECK_LAUNCH("cached_attention_kernel");
  const int64_t rows = (int64_t)a.max_new * a.group;
  hipLaunchKernelGGL((cached_join_kernel<T, 16 * QT * RW>),
                     dim3((unsigned)p.units, (unsigned)(rows < p.block_rows ? rows : p.block_rows)),
                     dim3(256), 0, st, a);
  SS_CHECK_LAUNCH("cached_join_kernel");
  return SS_OK;
}

// Bytes of keys and values that the bounds allow from which on they are loaded past the caches
// (nt): 64 sequences of 7800 keys 186 -> 165 us, one of 131071 59 -> 53, 64 of 500 (66 MB)
// 19 -> 17; but one of 16384 (17 MB) 16 -> 17, and rows that four waves share 36 -> 45 us.
constexpr int64_t kOnceBytes = (int64_t)32 << 20;

template <class T, bool SCORES>
int launch_attention(const CachedAttnArgs& a, const Layout& p, hipStream_t st) {
  if (!SCORES && p.block_rows > 32)
    return p.block_rows == 64 ? launch_attention<T, 2, 2, false, false>(a, p, st)
                              : launch_attention<T, 2, 4, false, false>(a, p, st);
  int64_t keys = a.max_length;
  if (a.window && a.window < keys && a.sinks < keys)
    keys = std::min(keys, a.window + a.sinks + a.max_new);
  const bool once = keys >= kOnceBytes / 512 / ((int64_t)a.sequences * a.cache.kv_heads);
  if (SCORES || p.block_rows == 16)
    return once ? launch_attention<T, 1, 1, SCORES, true>(a, p, st)
                : launch_attention<T, 1, 1, SCORES, false>(a, p, st);
  return once ? launch_attention<T, 2, 1, false, true>(a, p, st)
              : launch_attention<T, 2, 1, false, false>(a, p, st);
}

template <class T>
int launch(const CachedAttnArgs& a, const Layout& p, hipStream_t st) {
  if (a.sequences == 0) {
    hipLaunchKernelGGL(cached_zeros_kernel, dim3((unsigned)cdiv(a.tokens * a.hq, 16)), dim3(256), 0,
                       st, a);
    SS_CHECK_LAUNCH("cached_zeros_kernel");
    return SS_OK;
  }
  if (a.tokens > 0) {
    const int rc = p.score_rows ? launch_attention<T, true>(a, p, st)
                                : launch_attention<T, false>(a, p, st);
    if (rc) return rc;
  }
  if (!a.w_out) return SS_OK;
  const int64_t cap = (int64_t)a.rows.row_pages * a.cache.page_size;
  const int64_t units = (int64_t)a.sequences * a.cache.kv_heads;
  if (p.score_rows || a.tokens == 0)
    hipLaunchKernelGGL(cached_weights_kernel, dim3((unsigned)(units * cdiv(cap, 256 * kWeightRows))),
                       dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(cached_weights_again_kernel<T>,
                       dim3((unsigned)(units * cdiv(cap, 4 * kKeys))), dim3(256), 0, st, a);
  SS_CHECK_LAUNCH("cached_weights_kernel");
  return SS_OK;
}

}  // namespace
}  // namespace ss

extern "C" size_t ss_cached_attention_workspace_size(int rows, int64_t tokens, int q_heads,
                                                     int kv_heads, int max_new,
                                                     int64_t max_length, int weights) {
  if (rows <= 0 || tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || max_new < 0 ||
      max_length < 0 || q_heads % kv_heads)
    return 0;
  return ss::Layout(rows, tokens, q_heads, kv_heads, max_new, max_length, weights != 0).bytes;
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
  if (tokens == 0 && (rows == 0 || !weights_out)) return SS_OK;
  SS_CHECK_ARG((rows == 0 || cu_seqlens) && (tokens == 0 || (q && o)), "%s: null pointer", who);
  SS_CHECK_ARG(aligned16(q) && aligned16(o) && ((q_tok | q_head | o_tok | o_head) & 7) == 0,
               "%s: needs 16-byte aligned bases and strides that are multiples of 8", who);
  SS_CHECK_ARG(max_new > 0 || tokens == 0, "%s: tokens, but max_new is 0", who);
  SS_CHECK_ARG(cache->k_row >= 0 && cache->k_row < (1 << 26) && cache->v_row >= 0 &&
                   cache->v_row < (1 << 26),
               "%s: cache rows must lie less than 2^26 elements apart", who);
  const Layout p(rows, tokens, q_heads, cache->kv_heads, max_new, max_length, weights_out != 0);
  const int64_t cap = (int64_t)row_pages * cache->page_size;
  SS_CHECK_ARG(tokens <= (int64_t)INT32_MAX / q_heads && p.units <= kMaxGrid / 4 &&
                   (!weights_out || rows * (int64_t)cache->kv_heads * cdiv(cap, 4 * kKeys) <= kMaxGrid),
               "%s: too many tokens in one call", who);
  const size_t need = ss_cached_attention_workspace_size(rows, tokens, q_heads, cache->kv_heads,
                                                         max_new, max_length, weights_out != 0);
  SS_CHECK_ARG(need <= workspace_bytes && (need == 0 || (workspace && aligned16(workspace))),
               "%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, need);
  char* ws = (char*)workspace;
  CachedAttnArgs a{cache_view(cache), TableView{table, table_stride, row_pages, lengths},
                   cu_seqlens, rows, tokens, max_length, (const char*)q, q_tok * 2, q_head * 2,
                   (char*)o, o_tok * 2, o_head * 2, q_heads, q_heads / cache->kv_heads,
                   scale == 0.f ? 1.f : fabsf(scale) * kLog2e,
                   scale < 0.f ? -1.f : scale == 0.f ? 0.f : 1.f, window, sinks, weights_in, weights_out,
                   weights_out ? (float2v*)(ws + p.stats) : nullptr, p.max_new, p.blocks, p.workers,
                   (int4*)(ws + p.list), (float*)(ws + p.ml), (float*)(ws + p.o),
                   (float*)(ws + p.scores), p.score_rows, p.score_keys};
  const hipStream_t st = (hipStream_t)stream;
  return cache->dtype == SS_F16 ? launch<half_t>(a, p, st) : launch<bhalf_t>(a, p, st);
}
