// The best continuations of each sequence's beams.
//
// A candidate is (beam b, token x) with v = (l_bx - log sum_y exp l_by) + score_b, in fp64 from
// the sum on; a v that is NaN counts as -inf.  The `count` first of beams x vocabulary are
// wanted, by v, then the lower beam, the greater logit, the lower token.  Within a beam the
// order of v is that of the logits, so no v is needed before the few that can win are
// known, and one pass over the logits does:
//
// beam_slice_kernel: a workgroup goes through a slice of one beam's logits, sums exp(l) and
// takes its `count` first.  Exponentials are fp32 (arguments off by 2^-22 at most at the top,
// where they count), sums of 16 of them fp32 and of those fp64: log-sums are good to some 1e-8,
// and to 1e-6 in any case.  The first: the count-th greatest of 64 maxima over disjoint parts is
// a bound that count candidates reach and few more do; the rounds that hold one are loaded
// again (each round's maximum is kept), and what reaches the bound goes to LDS and is ranked
// by counting.  Keys in registers for all of it, with the code for each, left room for two waves
// a SIMD: 104 us instead of 51 for 155 MB.
// beam_join_kernel: a workgroup a sequence.  A wave joins a beam's sums and its slices' firsts in
// the same way, then the beams' firsts are ranked by counting, those that reach a bound where they
// are many.
//
// 64 sequences x 8 beams x 151936 bf16 logits (155 MB): 36 us and 7 for the join.  It loads at 4.3
// TB/s with the VALUs busy 55 of 100 cycles (an exponential is a quarter as fast as an addition);
// the start and the ranking, when nothing is loaded, are the rest.  All workgroups are there at
// once, eight a CU: 12, 16 and 24 a CU took 37.3, 38.0 and 38.3 us, slices held in registers with
// a barrier between maxima and sums 36.4 to 42.7.  One sequence is two latencies, 5.9 and 5.6 us.
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
constexpr int kRounds = 16;      // of a slice at most: their maxima are kept, 1 KiB each
constexpr int kRoom = 512;       // candidates ranked at once
constexpr int kJoinRoom = 256;   // of a wave there
constexpr int kJoinLoads = 10;   // of a lane on their way
constexpr int kJoinCounted = 128;  // candidates up to which ranks are counted

struct SelectArgs {
  const char* logits;
  int64_t seq, beam;  // bytes
  int beams, count;
  int64_t vocab;
  int slices;
  const float* scores;
  int rounds;      // of a slice at most
  double* base;    // [sequences][beams][slices]: the slice's sum of exp(l) is sums e^base
  double* sums;
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

// Lane exchanges without LDS: rotations within rows of 16, then rows and halves side by side.
template <int CTRL>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
template <int CTRL>
__device__ __forceinline__ float moved(float v) {
  return __builtin_bit_cast(float, moved<CTRL>(__builtin_bit_cast(uint32_t, v)));
}
template <int CTRL, class V>
__device__ __forceinline__ V moved_pair(V v) {
  const u32x2 u = __builtin_bit_cast(u32x2, v);
  return __builtin_bit_cast(V, u32x2{moved<CTRL>((uint32_t)u[0]), moved<CTRL>((uint32_t)u[1])});
}
template <int CTRL>
__device__ __forceinline__ double moved(double v) {
  return moved_pair<CTRL>(v);
}
template <int CTRL>
__device__ __forceinline__ uint64_t moved(uint64_t v) {
  return moved_pair<CTRL>(v);
}
template <class V>
__device__ __forceinline__ V lane_of(V v, int lane) {
  if constexpr (sizeof(V) == 8) {
    const u32x2 u = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(V, u32x2{(uint32_t)__builtin_amdgcn_readlane((int)u[0], lane),
                                       (uint32_t)__builtin_amdgcn_readlane((int)u[1], lane)});
  } else {
    return __builtin_bit_cast(
        V, (uint32_t)__builtin_amdgcn_readlane((int)__builtin_bit_cast(uint32_t, v), lane));
  }
}
// f over the wave's lanes, the same in all of them (f commutes; the order is fixed).
template <class V, class F>
__device__ __forceinline__ V over_lanes(V v, F f) {
  v = f(v, moved<0x121>(v));  // row_ror 1, 2, 4, 8
  v = f(v, moved<0x122>(v));
  v = f(v, moved<0x124>(v));
  v = f(v, moved<0x128>(v));
  return f(f(lane_of(v, 0), lane_of(v, 16)), f(lane_of(v, 32), lane_of(v, 48)));
}
__device__ __forceinline__ float greatest(float v) {
  return over_lanes(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ double total(double v) {
  return over_lanes(v, [](double a, double b) { return a + b; });
}

// The n-th greatest (from 1) of the 64 lanes' numbers: the least of those that fewer than n are
// greater than.
__device__ __forceinline__ uint32_t nth_of_lanes(uint32_t mine, int n) {
  int rank = 0;
#pragma unroll 16
  for (int i = 0; i < 64; ++i) rank += (uint32_t)__builtin_amdgcn_readlane((int)mine, i) > mine;
  return over_lanes(rank < n ? mine : ~0u, [](uint32_t a, uint32_t b) { return min(a, b); });
}

// The n-th greatest of the lanes' 128 numbers, two each.  Of 64 maxima over disjoint parts the
// least is a poor bound: some 300 keys reach it.
__device__ __forceinline__ uint32_t nth_of_pairs(uint32_t a, uint32_t b, int n) {
  int rank_a = 0, rank_b = 0;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) {
    const uint32_t x = (uint32_t)__builtin_amdgcn_readlane((int)a, i);
    const uint32_t y = (uint32_t)__builtin_amdgcn_readlane((int)b, i);
    rank_a += (x > a) + (y > a);
    rank_b += (x > b) + (y > b);
  }
  const uint32_t least = min(rank_a < n ? a : ~0u, rank_b < n ? b : ~0u);
  return over_lanes(least, [](uint32_t u, uint32_t w) { return min(u, w); });
}
constexpr int kLanesBound = 32;  // counts up to which 64 maxima give the bound

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

// 16 bytes of a line from token `at` on; at the line's end those before it, with -inf for the
// tokens that are another thread's.  Lines of an odd vocabulary begin at any element.
template <class T>
struct Piece {
  static constexpr int kEach = 16 / sizeof(T);
  u32x4 x;
  __device__ __forceinline__ static int from(int at, int vocab) { return min(at, vocab - kEach); }
  __device__ __forceinline__ void load(const char* line, int at, int vocab) {
    struct __attribute__((packed, aligned(sizeof(T)))) Loose {
      u32x4 v;
    };
    x = reinterpret_cast<const Loose*>(line + (int64_t)from(at, vocab) * sizeof(T))->v;
  }
  __device__ __forceinline__ void mask(int at, int vocab) {
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (from(at, vocab) + e < at) none(e);
  }
  // Of a line shorter than a piece.
  __device__ __forceinline__ void load_short(const char* line, int at, int vocab) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      none(e);
      if (at + e < vocab) {
        if constexpr (sizeof(T) == 4) put(e, reinterpret_cast<const uint32_t*>(line)[at + e]);
        else put(e, reinterpret_cast<const uint16_t*>(line)[at + e]);
      }
    }
  }
  __device__ __forceinline__ float operator[](int e) const { return value<T>(x, e); }

 private:
  __device__ __forceinline__ void put(int e, uint32_t u) {
    if constexpr (sizeof(T) == 4) x[e] = u;
    else x[e >> 1] = (x[e >> 1] & (e & 1 ? 0xffffu : 0xffff0000u)) | u << 16 * (e & 1);
  }
  __device__ __forceinline__ void none(int e) {
    put(e, sizeof(T) == 4 ? 0xff800000u : std::is_same<T, half_t>::value ? 0xfc00u : 0xff80u);
  }
};

// A wave's running sums of exp(l), each lane's own `sum` times 2^shift, which stands for
// e^(shift / c).  The shift is the wave's, a whole number next to the greatest logit so far (up to 4
// below: a term's argument is then off by 2^-22 at most), so that a greater one costs no
// rounding, and a term is 2^(l c - shift) by one fma.  Past 2^30 (`far`), where floats lie 64
// apart and more, the sum is how many are the top.
struct Terms {
  static constexpr float c = 1.4426950408889634f;
  double sum = 0.0;
  float top = -INFINITY, shift = 0.f, limit = -INFINITY;
  bool far = false;
  // For logits up to `to`, the same in all lanes.
  __device__ __forceinline__ void raise(float to) {
    if (to <= top) return;
    const bool was_far = far;
    far = fabsf(to) >= 0x1p30f;
    const float next = far ? 0.f : rintf(to * c);
    if (far || was_far) sum *= 0.0;  // a NaN stays one
    else if (top != -INFINITY) sum = __builtin_ldexp(sum, (int)fmaxf(shift - next, -4096.f));
    top = to;
    shift = next;
    limit = far ? to : (next + 4.f) / c;
  }
  __device__ __forceinline__ void see(float mine) {
    if (__any(mine > limit)) raise(greatest(mine));
  }
  template <class T, int P>
  __device__ __forceinline__ void add(const Piece<T> (&x)[P]) {
    constexpr int kEach = Piece<T>::kEach;
    float part[P * kEach];
    auto each = [&](auto term) {
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int e = 0; e < kEach; ++e) part[i * kEach + e] = term(x[i][e]);
    };
    if (far) each([&](float l) { return l == top ? 1.f : l == l ? 0.f : l; });
    else each([&](float l) { return __builtin_amdgcn_exp2f(__builtin_fmaf(l, c, -shift)); });
#pragma unroll
    for (int d = P * kEach / 2; d >= 1; d /= 2)
#pragma unroll
      for (int e = 0; e < d; ++e) part[e] += part[e + d];
    sum += part[0];
  }
  // What is factored out, as a natural logarithm.
  __device__ __forceinline__ double base() const {
    return top == -INFINITY ? -INFINITY : far ? (double)top : shift / (double)c;
  }
};

// P pieces a thread and round, the next round's on their way meanwhile (behind the last round
// the line's end once more).  SHORT: lines of fewer tokens than a piece has.
template <class T, int P, bool SHORT>
__global__ __launch_bounds__(kThreads) void beam_slice_kernel(SelectArgs a) {
  constexpr int kEach = Piece<T>::kEach, kPass = kThreads * kEach;
  __shared__ uint64_t room[kRoom];
  __shared__ int used_slots;
  __shared__ uint64_t shared_bound;
  __shared__ float tops[4][64];
  __shared__ double sums[4];
  extern __shared__ float round_tops[];  // [rounds][threads]
  const int slice = blockIdx.x, beam = blockIdx.y, seq = blockIdx.z;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const char* line = a.logits + seq * a.seq + beam * a.beam;
  const int vocab = (int)a.vocab, start = slice * a.rounds * (kPass * P);
  const int rounds = min(a.rounds, (vocab - start + kPass * P - 1) / (kPass * P));
  const int first = start + threadIdx.x * kEach;
  auto load = [&](Piece<T>& x, int at) {
    if constexpr (SHORT) x.load_short(line, at, vocab);
    else x.load(line, at, vocab);
  };
  Piece<T> next[P];
#pragma unroll
  for (int i = 0; i < P; ++i) load(next[i], first + i * kPass);
  Terms terms;
  float top = -INFINITY;
#pragma unroll 1
  for (int r = 0; r < rounds; ++r) {
    Piece<T> x[P];
#pragma unroll
    for (int i = 0; i < P; ++i) x[i] = next[i];
    const int at = first + r * (kPass * P);
#pragma unroll
    for (int i = 0; i < P; ++i) load(next[i], at + (P + i) * kPass);
    if (!SHORT && start + (r + 1) * (kPass * P) > vocab) {
#pragma unroll
      for (int i = 0; i < P; ++i) x[i].mask(at + i * kPass, vocab);
    }
    float here = -INFINITY;  // NaN is never greater
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
      for (int e = 0; e < kEach; ++e) here = fmaxf(here, x[i][e]);
    round_tops[r * kThreads + threadIdx.x] = here;
    top = fmaxf(top, here);
    terms.see(here);
    terms.add(x);
  }
  tops[wave][lane] = top;
  __syncthreads();
  const float lane_top = fmaxf(fmaxf(tops[0][lane], tops[1][lane]),
                               fmaxf(tops[2][lane], tops[3][lane]));
  if (wave == 0) {
    // Lanes without a token of the slice have theirs behind its last one.
    auto order_of = [&](float l, int thread) {
      return start + thread * kEach < vocab ? ordered(l) : 0u;
    };
    const uint32_t nth =
        a.count <= kLanesBound
            ? nth_of_lanes(order_of(lane_top, lane), a.count)
            : nth_of_pairs(order_of(fmaxf(tops[0][lane], tops[1][lane]), lane),
                           order_of(fmaxf(tops[2][lane], tops[3][lane]), 128 + lane), a.count);
    if (lane == 0) shared_bound = bound_from(nth);
  }
  terms.raise(greatest(lane_top));
  const double sum = total(terms.sum);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  // The few rounds that reach the bound are loaded again.
  const int used = gather<kRoom>(
      room, &used_slots, shared_bound, a.count, threadIdx.x == 0,
      [&](uint64_t from, auto f) {
        const float least = unordered(max((uint32_t)(from >> 32), 0x007fffffu));
        // Lanes go through their own rounds side by side, hardly ever more than one.
        uint32_t those = 0;
        for (int r = 0; r < rounds; ++r)
          those |= (uint32_t)(round_tops[r * kThreads + threadIdx.x] >= least) << r;
        while (those) {
          const int at = first + (__ffs((int)those) - 1) * (kPass * P);
          those &= those - 1;
          Piece<T> x[P];
#pragma unroll
          for (int i = 0; i < P; ++i) load(x[i], at + i * kPass);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const int from_here = at + i * kPass;
            const int token = SHORT ? from_here : Piece<T>::from(from_here, vocab);
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
              const float l = fmaxf(x[i][e], -INFINITY);
              if (l < least) continue;
              const int t = token + e;
              const uint64_t key = (uint64_t)ordered(l) << 32 | (uint32_t)~(uint32_t)t;
              if (t >= from_here && t < vocab && key >= from) f(key);
            }
          }
        }
      },
      [] { __syncthreads(); });
  const int64_t unit = ((int64_t)seq * a.beams + beam) * a.slices + slice;
  if (threadIdx.x == 0) {
    a.base[unit] = terms.base();
    a.sums[unit] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
  // Turned by slice, so that a lane of the join has some of each rank: the maxima of lanes that
  // held the slices' bests, and of others that held their lasts, gave a bound that most reached.
  uint64_t* out = a.best + unit * a.count;
  auto turned = [&](int c) { return (c + 11 * slice) % a.count; };
  for (int c = threadIdx.x; c < used; c += kThreads) {
    const uint64_t key = room[c];
    int rank = 0;
#pragma unroll 8
    for (int o = 0; o < used; ++o) rank += room[o] > key;
    if (rank < a.count) out[turned(rank)] = key;
  }
  for (int c = used + threadIdx.x; c < a.count; c += kThreads) out[turned(c)] = 0;
}

// v ordered as an integer, 1 at least.
__device__ __forceinline__ uint64_t ordered(double v) {
  v = v == v ? v + 0.0 : -INFINITY;
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return u >> 63 ? ~u : u | (uint64_t)1 << 63;
}

// W waves: as many as there are beams, 16 at most.
template <int W>
__global__ __launch_bounds__(64 * W) void beam_join_kernel(SelectArgs a) {
  __shared__ uint64_t rooms[W][kJoinRoom];
  __shared__ int used_slots[W];
  // The beams' firsts in order: v (0 where there is none) and key.
  extern __shared__ __attribute__((aligned(16))) uint64_t lines[];
  uint64_t* vs = lines;
  uint64_t* keys = lines + a.beams * a.count;
  const int seq = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // LDS is in order within a wave.
  auto wave_sync = [] {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  for (int b = wave; b < a.beams; b += W) {
    const int64_t unit = ((int64_t)seq * a.beams + b) * a.slices;
    const uint64_t* best = a.best + unit * a.count;
    const int n = a.slices * a.count;
    const double score = a.scores[(int64_t)seq * a.beams + b];
    // The first keys of a lane stay with it; the others are loaded as often as they are wanted.
    uint64_t mine[kJoinLoads];
#pragma unroll
    for (int i = 0; i < kJoinLoads; ++i) mine[i] = lane + 64 * i < n ? best[lane + 64 * i] : 0;
    auto each_key = [&](auto f) {
#pragma unroll
      for (int i = 0; i < kJoinLoads; ++i) f(mine[i]);
      for (int c = lane + 64 * kJoinLoads; c < n; c += 64 * kJoinLoads) {
        uint64_t key[kJoinLoads];
#pragma unroll
        for (int i = 0; i < kJoinLoads; ++i) key[i] = c + 64 * i < n ? best[c + 64 * i] : 0;
#pragma unroll
        for (int i = 0; i < kJoinLoads; ++i) f(key[i]);
      }
    };
    // The first 64 slices' sums at once with all the rest.
    const double my_base = lane < a.slices ? a.base[unit + lane] : -INFINITY;
    const double my_sum = lane < a.slices ? a.sums[unit + lane] : 0.0;
    uint64_t most = 0, second = 0;
    each_key([&](uint64_t key) {
      second = max(second, min(most, key));
      most = max(most, key);
    });
    double base = my_base;
    for (int s = 64 + lane; s < a.slices; s += 64) base = fmax(base, a.base[unit + s]);
    base = over_lanes(base, [](double u, double w) { return fmax(u, w); });
    // Bases are whole numbers over c, or (far) as good as 0 or nothing apart.
    auto scaled = [&](double of, double part) {  // 0 (or NaN) of a slice of -inf
      if (of == -INFINITY) return part;
      return __builtin_ldexp(part, (int)fmax(rint((of - base) * (double)Terms::c), -4096.0));
    };
    double sum = scaled(my_base, my_sum);
    for (int s = 64 + lane; s < a.slices; s += 64)
      sum += scaled(a.base[unit + s], a.sums[unit + s]);
    sum = total(sum);
    const double whole = base + log(sum);
    const uint32_t nth =
        a.count <= kLanesBound
            ? nth_of_lanes((uint32_t)(most >> 32), a.count)
            : nth_of_pairs((uint32_t)(most >> 32), (uint32_t)(second >> 32), a.count);
    const uint64_t bound = bound_from(nth);
    uint64_t* room = rooms[wave];
    const int used = gather<kJoinRoom>(
        room, &used_slots[wave], bound, a.count, lane == 0,
        [&](uint64_t from, auto f) {
          each_key([&](uint64_t key) {
            if (key >= from) f(key);
          });
        },
        wave_sync);
    for (int c = lane; c < used; c += 64) {
      const uint64_t key = room[c];
      int rank = 0;
#pragma unroll 8
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
  // Candidates in the order of beam and place there: equal ones stand in the order wanted.
  const int all = a.beams * a.count;
  auto place = [&](int c, uint64_t v, int rank) {
    if (rank >= a.count) return;
    const int64_t at = (int64_t)seq * a.count + rank;
    const uint64_t u = v >> 63 ? v & ~((uint64_t)1 << 63) : ~v;
    a.out_scores[at] = (float)__builtin_bit_cast(double, u);
    a.parents[at] = c / a.count;
    a.tokens[at] = (int64_t)(uint32_t)~(uint32_t)keys[c];
  };
  if (all <= kJoinCounted) {
    // Four threads count for one, two candidates at a time (the one behind the last is there: a
    // key, and not counted).
    const int part = threadIdx.x & 3;
    for (int c = threadIdx.x >> 2; c < all; c += 16 * W) {
      const uint64_t v = vs[c];
      uint32_t rank = 0;
#pragma unroll 8
      for (int o = 2 * part; o < all; o += 8) {
        const u32x4 two = *reinterpret_cast<const u32x4*>(vs + o);
        const uint64_t x = (uint64_t)two[1] << 32 | two[0], y = (uint64_t)two[3] << 32 | two[2];
        rank += (x > v) | ((x == v) & (o < c));
        rank += ((y > v) | ((y == v) & (o + 1 < c))) & (o + 1 < all);
      }
      rank += moved<0xb1>(rank);  // quad_perm: the neighbour, then the other two
      rank += moved<0x4e>(rank);
      if (part == 0 && v) place(c, v, rank);
    }
    return;
  }
  if (wave) return;
  // Many: 64 of them, the first of each line in equal numbers, give a bound again.
  const int each = 64 / a.beams, of_line = lane / each, in_line = lane - of_line * each;
  const uint64_t mine =
      of_line < a.beams && in_line < a.count ? vs[of_line * a.count + in_line] : 0;
  const uint64_t bound = bound_from(nth_of_lanes((uint32_t)(mine >> 32), a.count));
  uint32_t* those = reinterpret_cast<uint32_t*>(rooms);  // in order
  int n = 0;
  for (int c = lane; c - lane < all; c += 64) {
    const bool reaches = c < all && vs[c] >= bound;
    const uint64_t lanes = __ballot(reaches);
    const int at = n + __popcll(lanes & (((uint64_t)1 << lane) - 1));
    if (reaches && at < kJoinRoom) those[at] = c;
    n += __popcll(lanes);
  }
  wave_sync();
  if (n <= kJoinRoom) {
    for (int i = lane; i < n; i += 64) {
      const uint64_t v = vs[those[i]];
      int rank = 0;
#pragma unroll 8
      for (int o = 0; o < n; ++o) {
        const uint64_t x = vs[those[o]];
        rank += (x > v) | ((x == v) & (o < i));
      }
      place(those[i], v, rank);
    }
    return;
  }
  // Equal ones, -inf for instance: the lines are merged, of which a lane has one each.
  const int first = lane * a.count;
  uint64_t v = lane < a.beams ? vs[first] : 0;
  for (int i = 0, at = 0; i < a.count; ++i) {
    const uint64_t top = over_lanes(v, [](uint64_t x, uint64_t y) { return x > y ? x : y; });
    if (lane != __ffsll((long long)__ballot(v == top)) - 1) continue;
    place(first + at, v, i);
    ++at;
    v = at < a.count ? vs[first + at] : 0;
  }
}

struct SelectLayout {
  int pieces, rounds, slices;  // 16-byte loads of a thread and round
  size_t base, sums, best, bytes;
  SelectLayout(int sequences, int beams, int64_t vocab, int count, int width) {
    const int64_t lines = (int64_t)sequences * beams;
    const int64_t all = cdiv(vocab, (int64_t)kThreads * (16 / width));
    // Slices for eight workgroups a CU, of one round of one load as long as there are fewer; not
    // more than the join's lanes hold the firsts of at once (one sequence of 16 beams and 32
    // each 34 us without).
    int64_t wanted = cdiv(8 * (int64_t)device_cu_count(), lines);
    const int64_t most = 64 * kJoinLoads / count;
    wanted = wanted < most ? wanted : most;
    const int64_t each = cdiv(all, wanted < all ? wanted : all);
    pieces = each > 1 ? 2 : 1;
    rounds = (int)cdiv(each, pieces);
    if (rounds > kRounds) rounds = kRounds;
    slices = (int)cdiv(all, (int64_t)rounds * pieces);
    bytes = 0;
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) / 256 * 256;
      return at;
    };
    best = take((size_t)lines * slices * count * 8);
    sums = take((size_t)lines * slices * 8);
    base = take((size_t)lines * slices * 8);
  }
};

template <class T>
int launch(const SelectArgs& a, const SelectLayout& p, int sequences, hipStream_t st) {
  const dim3 grid((unsigned)p.slices, (unsigned)a.beams, (unsigned)sequences), block(kThreads);
  const unsigned lds = p.rounds * kThreads * 4;
  if (a.vocab < Piece<T>::kEach)
    hipLaunchKernelGGL((beam_slice_kernel<T, 1, true>), grid, block, lds, st, a);
  else if (p.pieces == 1)
    hipLaunchKernelGGL((beam_slice_kernel<T, 1, false>), grid, block, lds, st, a);
  else
    hipLaunchKernelGGL((beam_slice_kernel<T, 2, false>), grid, block, lds, st, a);
  SS_CHECK_LAUNCH("beam_slice_kernel");
  const dim3 sequence((unsigned)sequences);
  const unsigned firsts = (unsigned)(a.beams * a.count * 16);
  if (a.beams <= 8) hipLaunchKernelGGL(beam_join_kernel<8>, sequence, dim3(512), firsts, st, a);
  else hipLaunchKernelGGL(beam_join_kernel<16>, sequence, dim3(1024), firsts, st, a);
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
               scores, p.rounds, (double*)(ws + p.base), (double*)(ws + p.sums), (uint64_t*)(ws + p.best),
               out_scores, parents, tokens};
  const hipStream_t st = (hipStream_t)stream;
  return dtype == SS_F32   ? launch<float>(a, p, sequences, st)
         : dtype == SS_F16 ? launch<half_t>(a, p, sequences, st)
                           : launch<bhalf_t>(a, p, sequences, st);
}
