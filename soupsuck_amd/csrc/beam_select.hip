// The best continuations of each sequence's beams.
//
// A candidate is (beam b, token x) with v = (l_bx - log sum_y exp l_by) + score_b, in fp64 from
// the sum on; a v that is NaN counts as -inf.  The `count` first of beams x vocabulary are
// wanted, by v, then the lower beam, the greater logit, the lower token.  Within a beam the
// order of v is that of the logits, so no v is needed before the few that can win are
// known, and one pass over the logits does:
//
// beam_slice_kernel: a workgroup holds a slice of one beam's logits in registers (at most
// kVectors loads of 16 bytes a thread, all on their way at once), takes its maximum, the sum of
// exp(l - maximum) and its `count` first.  Exponentials are fp32 (a difference next to the
// maximum, where it counts, is exact or off by 2^-24), sums of them fp64: log-sums are good to
// some 1e-8.  The first: the count-th greatest of 64 maxima over disjoint parts is a bound that
// count candidates reach and few more do; those go to LDS and are ranked by counting.
// beam_join_kernel: a workgroup a sequence.  A wave joins a beam's sums and its slices' firsts in
// the same way, then every candidate finds its rank by a binary search in each beam's line.
//
// Keys are 64 bits and unique, the logit ordered as an integer over the complement of its
// token, so that results do not depend on the order in which LDS slots are handed out.
#include <type_traits>

#include "common.h"

namespace ss {
namespace {

typedef __bf16 bhalf_t;

constexpr int kThreads = 256;
constexpr int kMostCount = 64;
constexpr int kMostBeams = 64;
constexpr int kMostFirsts = 2048;  // beams * count: 32 KiB of LDS
constexpr int kVectors = 8;      // 16-byte loads of a thread at most
constexpr int kRoom = 1024;      // candidates ranked at once
constexpr int kJoinWaves = 8;
constexpr int kJoinRoom = 256;   // of a wave there

struct SelectArgs {
  const char* logits;
  int64_t seq, beam;  // bytes
  int beams, count;
  int64_t vocab;
  int slices;
  const float* scores;
  float* top;      // [sequences][beams][slices]
  double* sums;    // [sequences][beams][slices]
  uint64_t* best;  // [sequences][beams][slices][count]: keys, 0 for none
  float* out_scores;
  int32_t* parents;
  int64_t* tokens;
};

// Greater for a greater number (-0 is 0), from 0x007fffff up.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __builtin_bit_cast(float, u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

template <class T>
__device__ __forceinline__ float value(const u32x4& v, int e) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, (uint32_t)v[e]);
  else return (float)__builtin_bit_cast(T, (uint16_t)(v[e >> 1] >> 16 * (e & 1)));
}

// The n-th greatest (from 1) of the 64 lanes' numbers.
__device__ __forceinline__ uint32_t nth_of_lanes(uint32_t mine, int n) {
  const int lane = threadIdx.x & 63;
  int rank = 0;  // equal ones in the order of their lanes
#pragma unroll 16
  for (int i = 0; i < 64; ++i) {
    const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
    rank += (other > mine) | ((other == mine) & (i < lane));
  }
  const int at = __ffsll((long long)__ballot(rank == n - 1)) - 1;
  return (uint32_t)__builtin_amdgcn_readlane((int)mine, at);
}

// The least key of a logit's order, or of any key.
__device__ __forceinline__ uint64_t bound_from(uint32_t order) {
  return order ? (uint64_t)order << 32 : 1;
}

// Puts the keys that reach the bound into room[] and returns how many, at most ROOM.  each(bound, f)
// calls f(key) for the caller's keys from the bound up.  `count` of all keys reach the bound,
// or all keys do; where more do than there is room for, it is raised: keys are unique, so
// there is one that between count and ROOM of them reach.  sync() waits for all callers.
template <int ROOM, class Each, class Sync>
__device__ __forceinline__ int gather(uint64_t* room, int* used, uint64_t bound, int count,
                                      bool leader, Each each, Sync sync) {
  uint64_t low = bound, high = ~(uint64_t)0;
  for (;;) {
    if (leader) *used = 0;
    sync();
    each(bound, [&](uint64_t key) {
      const int at = atomicAdd(used, 1);
      if (at < ROOM) room[at] = key;
    });
    sync();
    const int n = *used;
    sync();
    if (n <= ROOM && (n >= count || bound == low)) return n;
    if (n > ROOM) low = bound;
    else high = bound;
    if (high - low < 2) return n < ROOM ? n : ROOM;  // not with unique keys
    bound = low + (high - low) / 2;
  }
}

template <class T, int V>
__global__ __launch_bounds__(kThreads) void beam_slice_kernel(SelectArgs a) {
  constexpr int kEach = 16 / sizeof(T);
  __shared__ uint64_t room[kRoom];
  __shared__ int used_slots;
  __shared__ float tops[4][64];
  __shared__ double sums[4];
  const int slice = blockIdx.x, beam = blockIdx.y, seq = blockIdx.z;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const char* line = a.logits + seq * a.seq + beam * a.beam;
  const int64_t first = (int64_t)slice * (kThreads * kEach * V) + threadIdx.x * kEach;
  // Rows of an odd vocabulary begin at any element.
  struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    u32x4 v;
  };
  u32x4 x[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int64_t i = first + (int64_t)v * kThreads * kEach;
    if (i + kEach <= a.vocab) {
      x[v] = reinterpret_cast<const Loose*>(line + i * sizeof(T))->v;
    } else {
      // -inf behind the last token, where key_of knows no candidate.
      constexpr uint32_t none = sizeof(T) == 4 ? 0xff800000u
                                : std::is_same<T, half_t>::value ? 0xfc00fc00u : 0xff80ff80u;
      x[v] = u32x4{none, none, none, none};
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (i + e < a.vocab) {
          if constexpr (sizeof(T) == 4) {
            x[v][e] = reinterpret_cast<const uint32_t*>(line)[i + e];
          } else {
            const uint32_t u = reinterpret_cast<const uint16_t*>(line)[i + e];
            const uint32_t keep = e & 1 ? 0x0000ffffu : 0xffff0000u;
            x[v][e >> 1] = (x[v][e >> 1] & keep) | u << 16 * (e & 1);
          }
        }
    }
  }
  float tops_of[V], top = -INFINITY;  // NaN is never greater
#pragma unroll
  for (int v = 0; v < V; ++v) {
    tops_of[v] = -INFINITY;
#pragma unroll
    for (int e = 0; e < kEach; ++e) tops_of[v] = fmaxf(tops_of[v], value<T>(x[v], e));
    top = fmaxf(top, tops_of[v]);
  }
  tops[wave][lane] = top;
  __syncthreads();
  const float lane_top = fmaxf(fmaxf(tops[0][lane], tops[1][lane]),
                               fmaxf(tops[2][lane], tops[3][lane]));
  // Lanes without a token of the slice have them behind its last one.
  const bool some = (int64_t)slice * (kThreads * kEach * V) + lane * kEach < a.vocab;
  const uint64_t bound = bound_from(nth_of_lanes(some ? ordered(lane_top) : 0u, a.count));
  top = lane_top;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, kWave));
  // A NaN logit makes the sum NaN, and so does one of +inf.
  const float base = top == -INFINITY ? 0.f : top;
  double sum = 0.0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float part = 0.f;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      part += __builtin_amdgcn_exp2f((value<T>(x[v], e) - base) * 1.4426950408889634f);
    sum += part;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, kWave);
  if (lane == 0) sums[wave] = sum;
  const int used = gather<kRoom>(
      room, &used_slots, bound, a.count, threadIdx.x == 0,
      [&](uint64_t from, auto f) {
        const float least = unordered(max((uint32_t)(from >> 32), 0x007fffffu));
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (tops_of[v] >= least) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
              const int64_t i = first + (int64_t)v * kThreads * kEach + e;
              const uint64_t key = (uint64_t)ordered(fmaxf(value<T>(x[v], e), -INFINITY)) << 32 |
                                   (uint32_t)~(uint32_t)i;
              if (i < a.vocab && key >= from) f(key);
            }
          }
      },
      [] { __syncthreads(); });
  const int64_t unit = ((int64_t)seq * a.beams + beam) * a.slices + slice;
  if (threadIdx.x == 0) {
    a.top[unit] = top;
    a.sums[unit] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
  uint64_t* out = a.best + unit * a.count;
  for (int c = threadIdx.x; c < used; c += kThreads) {
    const uint64_t key = room[c];
    int rank = 0;
    for (int o = 0; o < used; ++o) rank += room[o] > key;
    if (rank < a.count) out[rank] = key;
  }
  for (int c = used + threadIdx.x; c < a.count; c += kThreads) out[c] = 0;
}

// v ordered as an integer, 1 at least.
__device__ __forceinline__ uint64_t ordered(double v) {
  v = v == v ? v + 0.0 : -INFINITY;
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return u >> 63 ? ~u : u | (uint64_t)1 << 63;
}

__global__ __launch_bounds__(64 * kJoinWaves) void beam_join_kernel(SelectArgs a) {
  __shared__ uint64_t rooms[kJoinWaves][kJoinRoom];
  __shared__ int used_slots[kJoinWaves];
  // The beams' firsts in order: v (0 where there is none) and key.
  extern __shared__ uint64_t lines[];
  uint64_t* vs = lines;
  uint64_t* keys = lines + a.beams * a.count;
  const int seq = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // LDS is in order within a wave.
  auto wave_sync = [] {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  for (int b = wave; b < a.beams; b += kJoinWaves) {
    const int64_t unit = ((int64_t)seq * a.beams + b) * a.slices;
    float top = -INFINITY;
    for (int s = lane; s < a.slices; s += 64) top = fmaxf(top, a.top[unit + s]);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, kWave));
    double sum = 0.0;
    for (int s = lane; s < a.slices; s += 64) {
      const float t = a.top[unit + s];
      const double part = a.sums[unit + s];
      sum += t == -INFINITY ? part : part * exp((double)t - (double)top);  // 0 (or NaN) of -inf
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, kWave);
    const double whole = (double)top + log(sum);
    const double score = a.scores[(int64_t)seq * a.beams + b];
    const uint64_t* best = a.best + unit * a.count;
    const int n = a.slices * a.count;
    uint64_t most = 0;
    for (int c = lane; c < n; c += 64) most = max(most, best[c]);
    const uint64_t bound = bound_from(nth_of_lanes((uint32_t)(most >> 32), a.count));
    uint64_t* room = rooms[wave];
    const int used = gather<kJoinRoom>(
        room, &used_slots[wave], bound, a.count, lane == 0,
        [&](uint64_t from, auto f) {
          for (int c = lane; c < n; c += 64) {
            const uint64_t key = best[c];
            if (key >= from) f(key);
          }
        },
        wave_sync);
    for (int c = lane; c < used; c += 64) {
      const uint64_t key = room[c];
      int rank = 0;
      for (int o = 0; o < used; ++o) rank += room[o] > key;
      if (rank >= a.count) continue;
      const double l = unordered((uint32_t)(key >> 32));
      vs[b * a.count + rank] = ordered((l - whole) + score);
      keys[b * a.count + rank] = key;
    }
    for (int c = used + lane; c < a.count; c += 64) vs[b * a.count + c] = 0;
    wave_sync();
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.beams * a.count; c += 64 * kJoinWaves) {
    const uint64_t v = vs[c];
    if (!v) continue;
    const int b = c / a.count;
    int rank = c - b * a.count;
    for (int o = 0; o < a.beams && rank < a.count; ++o) {
      if (o == b) continue;
      // Those of line o that come before: v' > v, and the equal ones of a lower beam.
      const uint64_t least = v + (o > b);
      int lo = 0, hi = a.count;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (vs[o * a.count + mid] >= least) lo = mid + 1;
        else hi = mid;
      }
      rank += lo;
    }
    if (rank >= a.count) continue;
    const int64_t at = (int64_t)seq * a.count + rank;
    const uint64_t u = v >> 63 ? v & ~((uint64_t)1 << 63) : ~v;
    a.out_scores[at] = (float)__builtin_bit_cast(double, u);
    a.parents[at] = b;
    a.tokens[at] = (int64_t)(uint32_t)~(uint32_t)keys[c];
  }
}

struct SelectLayout {
  int vectors, slices;
  size_t top, sums, best, bytes;
  SelectLayout(int sequences, int beams, int64_t vocab, int count, int width) {
    const int64_t lines = (int64_t)sequences * beams;
    // As many loads a thread as leave every CU four workgroups.
    vectors = kVectors;
    auto cut = [&](int v) { return cdiv(vocab, (int64_t)kThreads * (16 / width) * v); };
    while (vectors > 1 && lines * cut(vectors) < 4 * (int64_t)device_cu_count()) vectors /= 2;
    slices = (int)cut(vectors);
    bytes = 0;
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) / 256 * 256;
      return at;
    };
    best = take((size_t)lines * slices * count * 8);
    sums = take((size_t)lines * slices * 8);
    top = take((size_t)lines * slices * 4);
  }
};

template <class T>
int launch(const SelectArgs& a, const SelectLayout& p, int sequences, hipStream_t st) {
  const dim3 grid((unsigned)p.slices, (unsigned)a.beams, (unsigned)sequences), block(kThreads);
  switch (p.vectors) {
    case 1: hipLaunchKernelGGL((beam_slice_kernel<T, 1>), grid, block, 0, st, a); break;
    case 2: hipLaunchKernelGGL((beam_slice_kernel<T, 2>), grid, block, 0, st, a); break;
    case 4: hipLaunchKernelGGL((beam_slice_kernel<T, 4>), grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL((beam_slice_kernel<T, 8>), grid, block, 0, st, a); break;
  }
  SS_CHECK_LAUNCH("beam_slice_kernel");
  hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)sequences), dim3(64 * kJoinWaves),
                     (unsigned)(a.beams * a.count * 16), st, a);
  SS_CHECK_LAUNCH("beam_join_kernel");
  return SS_OK;
}

bool select_sizes(int sequences, int beams, int64_t vocab, int count) {
  return sequences >= 0 && sequences <= 65535 && beams > 0 && beams <= kMostBeams && vocab > 0 &&
         vocab <= INT32_MAX - 65536 && count > 0 && count <= kMostCount && count <= beams * vocab &&
         beams * count <= kMostFirsts;
}

int width_of(int dtype) { return dtype == SS_F32 ? 4 : 2; }

}  // namespace
}  // namespace ss

extern "C" size_t ss_select_beams_workspace_size(int sequences, int beams, int64_t vocab, int count,
                                                 int dtype) {
  if (sequences <= 0 || !ss::select_sizes(sequences, beams, vocab, count)) return 0;
  return ss::SelectLayout(sequences, beams, vocab, count, ss::width_of(dtype)).bytes;
}

extern "C" int ss_select_beams(const void* logits, int64_t l_seq, int64_t l_beam, int dtype,
                               const float* scores, int sequences, int beams, int64_t vocab,
                               int count, float* out_scores, int32_t* parents, int64_t* tokens,
                               void* workspace, size_t workspace_bytes, void* stream) {
  using namespace ss;
  const char* who = "ss_select_beams";
  SS_CHECK_ARG(dtype == SS_F16 || dtype == SS_BF16 || dtype == SS_F32, "%s: bad dtype %d", who,
               dtype);
  SS_CHECK_ARG(select_sizes(sequences, beams, vocab, count),
               "%s: bad sizes (%d sequences, %d beams, vocabulary %lld, count %d)", who, sequences,
               beams, (long long)vocab, count);
  if (sequences == 0) return SS_OK;
  SS_CHECK_ARG(logits && scores && out_scores && parents && tokens, "%s: null pointer", who);
  const int width = width_of(dtype);
  SS_CHECK_ARG(((uintptr_t)logits & (width - 1)) == 0, "%s: logits are not aligned", who);
  const SelectLayout p(sequences, beams, vocab, count, width);
  SS_CHECK_ARG(p.bytes <= workspace_bytes && workspace && ((uintptr_t)workspace & 15) == 0,
               "%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, p.bytes);
  char* ws = (char*)workspace;
  SelectArgs a{(const char*)logits, l_seq * width, l_beam * width, beams, count, vocab, p.slices,
               scores, (float*)(ws + p.top), (double*)(ws + p.sums), (uint64_t*)(ws + p.best),
               out_scores, parents, tokens};
  const hipStream_t st = (hipStream_t)stream;
  return dtype == SS_F32   ? launch<float>(a, p, sequences, st)
         : dtype == SS_F16 ? launch<half_t>(a, p, sequences, st)
                           : launch<bhalf_t>(a, p, sequences, st);
}
