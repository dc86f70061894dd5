// Drafted tokens checked against the target's logits from given uniform numbers.
//
// p = softmax(target / T), q = softmax(draft / T); draft i is accepted while u_i q_i(x_i) <
// p_i(x_i).  At the first refusal the next token has the distribution max(p_i - q_i, 0), so
// that accepted and drawn tokens together are distributed as p; after no refusal it is drawn
// from p of the row behind the last draft.  Drawing inverts the running sum in token order.
//
// Probabilities and sums are fp64: a drawn token is the place of one number among up to
// 151936 running sums, and sums that are off by 1e-7 would name another token once in a
// hundred draws from a flat distribution.  The exponential is 2^t = 2^n 2^f, n = rint(t), with
// a polynomial of degree 8 for 2^f on [-1/2, 1/2] that interpolates at the Chebyshev nodes:
// off by 1.1e-12 at most, 18 fp64 operations (full rate here) for each logit.
//
// Three launches, each logit read once but for the chosen rows of refused drafts:
//   1. per (row, chunk of 8192 logits): maximum and sum of 2^((l - max) c), c = log2(e) / T (or
//      the place of the maximum at T = 0);
//   2. per (sequence, chunk): the decisions, then the chunk's part of the chosen row's mass;
//   3. per sequence: the chunk in which the drawn number lies, and the token in it.
#include <algorithm>

#include "paged.h"
#include "elementwise.h"

namespace ss {
namespace {

constexpr int kChunk = 8192;  // logits of a workgroup
// Threads of it, and groups of 8 logits that each takes: long parts where every row is
// summed (the reductions of a workgroup cost as much as 8 logits a thread), short ones where
// the chosen row is what a sequence waits for.
template <int THREADS>
struct Work {
  static constexpr int kThreads = THREADS, kWaves = THREADS / 64, kGroups = kChunk / 8 / THREADS;
};
using Sum = Work<256>;
using Pick = Work<512>;

struct Stat {  // of a chunk, or of a row
  double sum;  // of weight(l, max)
  float max;
  int at;      // first place of the maximum (T = 0)
};

struct Choice {  // of a sequence
  double p_inv, q_inv;    // 1 / sum, 0 where a row has no mass
  float p_max, q_max;
  int accepted, refused;  // refused: a draft was, and q applies
  int drafted;            // the refused token, or -1
};

struct VerifyArgs {
  const char* target; int64_t t_seq, t_row;  // bytes
  const char* draft; int64_t d_seq, d_row;
  const int64_t* tokens;
  const int32_t* counts;
  const float* uniform;
  int rows, drafts, chunks;
  int per;  // logit rows of a sequence: drafts + 1 of the target, then the draft's if given
  int64_t vocab;
  double c;  // log2(e) / T
  int32_t* accepted;
  int64_t* out;
  Stat* stats;      // target [rows][drafts + 1][chunks], then draft [rows][drafts][chunks]
  Choice* choices;  // [rows]
  double* parts;    // [rows][chunks]: mass to draw from

  __device__ __forceinline__ int count(int b) const {
    return counts ? min(max(counts[b], 0), drafts) : drafts;
  }
  __device__ __forceinline__ Stat* target_stats(int b, int i) const {
    return stats + ((int64_t)b * (drafts + 1) + i) * chunks;
  }
  __device__ __forceinline__ Stat* draft_stats(int b, int i) const {
    return stats + ((int64_t)rows * (drafts + 1) + (int64_t)b * drafts + i) * chunks;
  }
};

// 2^t, 0 for t below -1074 and NaN.
__device__ __forceinline__ double power(double t) {
  t = __builtin_fmax(t, -1100.0);
  const double n = __builtin_rint(t), f = t - n;
  double p = 0x1.63d1363930791p-20;
  p = __builtin_fma(p, f, 0x1.00dc4a53395d3p-16);
  p = __builtin_fma(p, f, 0x1.4308ac85a7718p-13);
  p = __builtin_fma(p, f, 0x1.5d8745a72831bp-10);
  p = __builtin_fma(p, f, 0x1.3b2ab7181b778p-7);
  p = __builtin_fma(p, f, 0x1.c6b08dd6fd236p-5);
  p = __builtin_fma(p, f, 0x1.ebfbdff823cedp-3);
  p = __builtin_fma(p, f, 0x1.62e42fef84cf0p-1);
  p = __builtin_fma(p, f, 0x1.0000000000000p+0);
  return __builtin_ldexp(p, (int)n);
}

// exp((l - top) / T): 1 at an infinite maximum and 0 below it, 0 where there is none.
__device__ __forceinline__ double weight(float l, float top, double c) {
  if (top == INFINITY) return l == top ? 1.0 : 0.0;
  return power(((double)l - (double)top) * c);
}
// The same of several logits; the branch on an infinite maximum is uniform.
template <int N>
__device__ __forceinline__ void weights(const float (&l)[N], float top, double c, double (&w)[N]) {
  const bool infinite = top == INFINITY;
  const double base = infinite ? 0.0 : (double)top;
#pragma unroll
  for (int e = 0; e < N; ++e) w[e] = power(((double)l[e] - base) * c);
  if (infinite) {
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = l[e] == top ? 1.0 : 0.0;
  }
}

template <class T>
using Vec8 = T __attribute__((ext_vector_type(8)));

// Logits j .. j + 7 of a row; what lies behind the row's end is -inf, and a NaN counts as that:
// it is no maximum, and its power is 0.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const char* row, int64_t j, int64_t vocab, float (&x)[8]) {
  const T* p = reinterpret_cast<const T*>(row) + j;
  if (VEC && j + 8 <= vocab) {
    const Vec8<T> v = *reinterpret_cast<const Vec8<T>*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = j + e < vocab ? (float)p[e] : -INFINITY;
  }
}

// f over the lanes up to and with each, in registers.
template <class V, int CTRL, int ROWS, class F>
__device__ __forceinline__ V moved(V v, V none, F f) {
  V other;
  if constexpr (sizeof(V) == 4) {
    other = __builtin_bit_cast(
        V, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v),
                                       CTRL, ROWS, 0xf, false));
  } else {
    const uint64_t n = __builtin_bit_cast(uint64_t, none), u = __builtin_bit_cast(uint64_t, v);
    const uint32_t low =
        __builtin_amdgcn_update_dpp((int)n, (int)u, CTRL, ROWS, 0xf, false);
    const uint32_t high =
        __builtin_amdgcn_update_dpp((int)(n >> 32), (int)(u >> 32), CTRL, ROWS, 0xf, false);
    other = __builtin_bit_cast(V, (uint64_t)high << 32 | low);
  }
  return f(v, other);
}
template <class V, class F>
__device__ __forceinline__ V upto(V v, V none, F f) {
  v = moved<V, 0x111, 0xf>(v, none, f);  // lanes 1, 2, 4, 8 below in the row
  v = moved<V, 0x112, 0xf>(v, none, f);
  v = moved<V, 0x114, 0xf>(v, none, f);
  v = moved<V, 0x118, 0xf>(v, none, f);
  v = moved<V, 0x142, 0xa>(v, none, f);  // the last lane of rows 0 and 2 to rows 1 and 3
  return moved<V, 0x143, 0xc>(v, none, f);  // and of row 1 to rows 2 and 3
}
template <class V>
__device__ __forceinline__ V lane_of(V v, int lane) {
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t low = __builtin_amdgcn_readlane((int)u, lane);
    const uint32_t high = __builtin_amdgcn_readlane((int)(u >> 32), lane);
    return __builtin_bit_cast(V, (uint64_t)high << 32 | low);
  }
}
__device__ __forceinline__ double wave_upto(double v) {
  return upto(v, 0.0, [](double x, double y) { return x + y; });
}
__device__ __forceinline__ double wave_sum_f64(double v) { return lane_of(wave_upto(v), 63); }
__device__ __forceinline__ float wave_top(float v) {
  return lane_of(upto(v, -INFINITY, [](float x, float y) { return fmaxf(x, y); }), 63);
}
__device__ __forceinline__ int wave_least(int v) {
  return lane_of(upto(v, INT32_MAX, [](int x, int y) { return min(x, y); }), 63);
}

// One statistic from the lanes' (those without a part: {0, -inf, INT32_MAX}).
__device__ __forceinline__ Stat join(Stat s, double c) {
  const float top = wave_top(s.max);
  return Stat{wave_sum_f64(s.sum * weight(s.max, top, c)), top,
              wave_least(s.max == top ? s.at : INT32_MAX)};
}

template <class T, bool VEC, bool GREEDY>
__global__ __launch_bounds__(Sum::kThreads) void verify_stats_kernel(VerifyArgs a) {
  __shared__ Stat waves[Sum::kWaves];
  const int chunk = blockIdx.x;
  const int b = blockIdx.y / a.per;
  const int i = blockIdx.y - b * a.per;
  const int n = a.count(b);
  const bool is_draft = i > a.drafts;
  if (is_draft ? i - a.drafts - 1 >= n : i > n) return;
  const char* row = is_draft ? a.draft + b * a.d_seq + (i - a.drafts - 1) * a.d_row
                             : a.target + b * a.t_seq + i * a.t_row;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t j0 = (int64_t)chunk * kChunk + threadIdx.x * 8;
  float x[Sum::kGroups][8];
#pragma unroll
  for (int g = 0; g < Sum::kGroups; ++g) load8<T, VEC>(row, j0 + g * Sum::kThreads * 8, a.vocab, x[g]);
  float top = -INFINITY;
#pragma unroll
  for (int g = 0; g < Sum::kGroups; ++g)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, x[g][e]);
  top = wave_top(top);
  Stat s{0.0, top, INT32_MAX};
  if (GREEDY) {
#pragma unroll
    for (int g = Sum::kGroups - 1; g >= 0; --g)
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (x[g][e] == top) s.at = (int)(j0 + g * Sum::kThreads * 8 + e);
    s.at = wave_least(s.at);
  } else {
#pragma unroll
    for (int g = 0; g < Sum::kGroups; ++g) {
      double w[8];
      weights(x[g], top, a.c, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) s.sum += w[e];
    }
    s.sum = wave_sum_f64(s.sum);
  }
  if (lane == 0) waves[wave] = s;
  __syncthreads();
  if (wave) return;
  s = join(lane < Sum::kWaves ? waves[lane] : Stat{0.0, -INFINITY, INT32_MAX}, a.c);
  if (lane == 0)
    (is_draft ? a.draft_stats(b, i - a.drafts - 1) : a.target_stats(b, i))[chunk] = s;
}

// Statistics of a whole row from its chunks', by one wave.
__device__ __forceinline__ Stat row_stat(const Stat* chunk, int chunks, double c) {
  const int lane = threadIdx.x & 63;
  Stat mine{0.0, -INFINITY, INT32_MAX};
  for (int i = lane; i < chunks; i += 64) {
    const Stat s = chunk[i];
    if (chunks <= 64) {
      mine = s;
    } else {
      const float top = fmaxf(mine.max, s.max);
      if (s.max > mine.max || (s.max == mine.max && s.at < mine.at)) mine.at = s.at;
      mine.sum = mine.sum * weight(mine.max, top, c) + s.sum * weight(s.max, top, c);
      mine.max = top;
    }
  }
  return join(mine, c);
}

template <class T>
__device__ __forceinline__ float logit(const char* row, int64_t j) {
  const float l = (float)reinterpret_cast<const T*>(row)[j];
  return l == l ? l : -INFINITY;
}

// Row i of sequence b as the one to draw from, and whether it is: a refused draft, or the
// row behind the last one.
template <class T>
__device__ __forceinline__ bool choose(const VerifyArgs& a, int b, int i, int n, Choice* c) {
  const int64_t x = i < n ? a.tokens[(int64_t)b * a.drafts + i] : -1;
  const bool known = x >= 0 && x < a.vocab;
  const bool drafted = i < n && a.draft;
  const float pl = known ? logit<T>(a.target + b * a.t_seq + i * a.t_row, x) : -INFINITY;
  const float ql = known && drafted ? logit<T>(a.draft + b * a.d_seq + i * a.d_row, x) : -INFINITY;
  const Stat p = row_stat(a.target_stats(b, i), a.chunks, a.c);
  c->p_inv = p.sum > 0.0 ? 1.0 / p.sum : 0.0;
  c->p_max = p.max;
  c->q_inv = 0.0;
  c->q_max = -INFINITY;
  c->accepted = i;
  c->refused = i < n;
  c->drafted = known ? (int)x : -1;
  if (drafted) {
    const Stat q = row_stat(a.draft_stats(b, i), a.chunks, a.c);
    c->q_inv = q.sum > 0.0 ? 1.0 / q.sum : 0.0;
    c->q_max = q.max;
  }
  if (i >= n || !known) return true;
  const double px = weight(pl, c->p_max, a.c) * c->p_inv;
  const double qx = drafted ? weight(ql, c->q_max, a.c) * c->q_inv : 1.0;
  return !(a.uniform[(int64_t)b * (a.drafts + 1) + i] * qx < px);
}

// The mass of eight logits of the chosen row: max(p - q, 0) of a refused draft, else (and
// where that is nothing) p.
template <class T, bool VEC>
__device__ __forceinline__ void masses(const VerifyArgs& a, const Choice& c, int b, int64_t j,
                                       bool plain, double (&m)[8]) {
  float x[8], y[8];
  const bool drafted = !plain && a.draft;
  load8<T, VEC>(a.target + b * a.t_seq + c.accepted * a.t_row, j, a.vocab, x);
  if (drafted) load8<T, VEC>(a.draft + b * a.d_seq + c.accepted * a.d_row, j, a.vocab, y);
  weights(x, c.p_max, a.c, m);
#pragma unroll
  for (int e = 0; e < 8; ++e) m[e] *= c.p_inv;
  if (drafted) {
    double q[8];
    weights(y, c.q_max, a.c, q);
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e] = fmax(m[e] - q[e] * c.q_inv, 0.0);
  } else if (!plain) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (j + e == c.drafted) m[e] = 0.0;
  }
}

// A chunk's part of p, from its statistics.
__device__ __forceinline__ double plain_part(const VerifyArgs& a, const Choice& c, int b,
                                             int chunk) {
  const Stat s = a.target_stats(b, c.accepted)[chunk];
  return s.sum * weight(s.max, c.p_max, a.c) * c.p_inv;
}

template <class T, bool VEC>
__global__ __launch_bounds__(Pick::kThreads) void verify_rest_kernel(VerifyArgs a) {
  __shared__ Choice choices[Pick::kWaves];
  __shared__ double sums[Pick::kWaves];
  const int chunk = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = a.count(b);
  // Every wave looks at its rows up to its first choice; the lowest of theirs is the one.
  Choice mine{};
  mine.accepted = INT32_MAX;
  for (int i = wave; i <= n; i += Pick::kWaves) {
    Choice c;
    if (choose<T>(a, b, i, n, &c)) {
      mine = c;
      break;
    }
  }
  if (lane == 0) choices[wave] = mine;
  __syncthreads();
  int first = 0;
#pragma unroll
  for (int w = 1; w < Pick::kWaves; ++w)
    if (choices[w].accepted < choices[first].accepted) first = w;
  const Choice c = choices[first];
  if (chunk == 0 && threadIdx.x == 0) a.choices[b] = c;
  double* part = a.parts + (int64_t)b * a.chunks + chunk;
  if (!c.refused) {
    if (threadIdx.x == 0) *part = plain_part(a, c, b, chunk);
    return;
  }
  double sum = 0.0;
  const int64_t j0 = (int64_t)chunk * kChunk + threadIdx.x * 8;
#pragma unroll
  for (int g = 0; g < Pick::kGroups; ++g) {
    double m[8];
    masses<T, VEC>(a, c, b, j0 + g * Pick::kThreads * 8, false, m);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += m[e];
  }
  sum = wave_sum_f64(sum);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  if (threadIdx.x) return;
  sum = 0.0;
#pragma unroll
  for (int w = 0; w < Pick::kWaves; ++w) sum += sums[w];
  *part = sum;
}

template <class T, bool VEC>
__global__ __launch_bounds__(Pick::kThreads) void verify_pick_kernel(VerifyArgs a) {
  __shared__ double sums[Pick::kWaves];
  __shared__ int hits[Pick::kWaves], lasts[Pick::kWaves];
  const int b = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Choice c = a.choices[b];
  const double* parts = a.parts + (int64_t)b * a.chunks;
  bool plain = !c.refused;
  auto part = [&](int i) {
    return i >= a.chunks ? 0.0 : plain && c.refused ? plain_part(a, c, b, i) : parts[i];
  };
  auto whole = [&] {
    double v = 0.0;
    for (int i = lane; i < a.chunks; i += 64) v += part(i);
    return wave_sum_f64(v);
  };
  double total = whole();
  if (!(total > 0.0) && c.refused) {
    plain = true;
    total = whole();
  }
  const double goal = (double)a.uniform[(int64_t)b * (a.drafts + 1) + a.drafts] * total;
  // The first chunk whose running sum exceeds the goal, or the last one that holds any.
  int chunk = -1;
  double ahead = 0.0, sum = 0.0;
  bool found = false;
  for (int i = 0; i < a.chunks && !found; i += 64) {
    const double v = part(i + lane);
    const double upto = sum + wave_upto(v);
    double below = __shfl_up(upto, 1, kWave);
    if (lane == 0) below = sum;
    const uint64_t over = __ballot(v > 0.0 && upto > goal), any = __ballot(v > 0.0);
    found = over != 0;
    if (any) {
      const int at = found ? __ffsll((long long)over) - 1 : 63 - __clzll((long long)any);
      chunk = i + at;
      ahead = lane_of(below, at);
    }
    sum = lane_of(upto, 63);
  }
  int64_t token = -1;
  if (chunk >= 0) {
    const int64_t j0 = (int64_t)chunk * kChunk + threadIdx.x * 8 * Pick::kGroups;
    double m[Pick::kGroups][8], mine = 0.0;
#pragma unroll
    for (int g = 0; g < Pick::kGroups; ++g) {
      masses<T, VEC>(a, c, b, j0 + g * 8, plain, m[g]);
#pragma unroll
      for (int e = 0; e < 8; ++e) mine += m[g][e];
    }
    double upto = wave_upto(mine);
    double start = __shfl_up(upto, 1, kWave);
    if (lane == 0) start = 0.0;
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) ahead += sums[w];
    start += ahead;
    // Place of the first running sum above the goal, and of the last logit with any mass
    // (taken where rounding leaves the chunk's own sum at or below the goal).
    int hit = INT32_MAX, any = -1;
#pragma unroll
    for (int g = 0; g < Pick::kGroups; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        start += m[g][e];
        if (m[g][e] > 0.0) {
          any = (int)(j0 + g * 8 + e);
          if (start > goal) hit = min(hit, any);
        }
      }
    hit = wave_least(hit);
    any = -wave_least(-any);
    if (lane == 0) hits[wave] = hit, lasts[wave] = any;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < Pick::kWaves; ++w) {
      hit = min(hit, hits[w]);
      any = max(any, lasts[w]);
    }
    token = hit != INT32_MAX ? hit : any;
  }
  int64_t* out = a.out + (int64_t)b * (a.drafts + 1);
  for (int i = threadIdx.x; i <= a.drafts; i += Pick::kThreads)
    out[i] = i < c.accepted ? a.tokens[(int64_t)b * a.drafts + i] : i == c.accepted ? token : -1;
  if (threadIdx.x == 0) a.accepted[b] = c.accepted;
}

__global__ __launch_bounds__(64) void verify_greedy_kernel(VerifyArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const int n = a.count(b);
  int i = 0;
  Stat s = row_stat(a.target_stats(b, 0), a.chunks, 1.0);
  while (i < n && s.max > -INFINITY && a.tokens[(int64_t)b * a.drafts + i] == s.at) {
    ++i;
    s = row_stat(a.target_stats(b, i), a.chunks, 1.0);
  }
  int64_t* out = a.out + (int64_t)b * (a.drafts + 1);
  for (int k = lane; k <= a.drafts; k += 64)
    out[k] = k < i ? a.tokens[(int64_t)b * a.drafts + k]
                   : k == i && s.max > -INFINITY ? (int64_t)s.at : -1;
  if (lane == 0) a.accepted[b] = i;
}

template <class T, bool VEC>
int launch(const VerifyArgs& a, bool greedy, hipStream_t st) {
  const dim3 block(Sum::kThreads), pick(Pick::kThreads);
  const dim3 grid((unsigned)a.chunks, (unsigned)a.rows * a.per);
  if (greedy) {
    hipLaunchKernelGGL((verify_stats_kernel<T, VEC, true>), grid, block, 0, st, a);
    SS_CHECK_LAUNCH("verify_stats_kernel");
    hipLaunchKernelGGL(verify_greedy_kernel, dim3((unsigned)a.rows), dim3(64), 0, st, a);
    SS_CHECK_LAUNCH("verify_greedy_kernel");
    return SS_OK;
  }
  hipLaunchKernelGGL((verify_stats_kernel<T, VEC, false>), grid, block, 0, st, a);
  SS_CHECK_LAUNCH("verify_stats_kernel");
  hipLaunchKernelGGL((verify_rest_kernel<T, VEC>), dim3((unsigned)a.chunks, (unsigned)a.rows),
                     pick, 0, st, a);
  SS_CHECK_LAUNCH("verify_rest_kernel");
  hipLaunchKernelGGL((verify_pick_kernel<T, VEC>), dim3((unsigned)a.rows), pick, 0, st, a);
  SS_CHECK_LAUNCH("verify_pick_kernel");
  return SS_OK;
}

template <class T>
int launch(const VerifyArgs& a, bool greedy, hipStream_t st) {
  const int64_t bytes = 8 * sizeof(T);  // of a vector load
  const int64_t all = (int64_t)(uintptr_t)a.target | (int64_t)(uintptr_t)a.draft | a.t_seq |
                      a.t_row | a.d_seq | a.d_row;
  return (all & (bytes - 1)) == 0 ? launch<T, true>(a, greedy, st) : launch<T, false>(a, greedy, st);
}

}  // namespace
}  // namespace ss

extern "C" size_t ss_verify_drafts_workspace_size(int rows, int drafts, int64_t vocab,
                                                  int drafted) {
  using namespace ss;
  if (rows <= 0 || drafts < 0 || vocab <= 0) return 0;
  const size_t chunks = (size_t)cdiv(vocab, kChunk);
  return (size_t)rows * ((2 * (size_t)drafts + 1) * chunks * sizeof(Stat) + sizeof(Choice) +
                         chunks * sizeof(double));
}

extern "C" int ss_verify_drafts(const void* target, int64_t t_seq, int64_t t_row,
                                const void* draft, int64_t d_seq, int64_t d_row, int dtype,
                                const int64_t* tokens, const int32_t* counts,
                                const float* uniform, int rows, int drafts, int64_t vocab,
                                double temperature, int32_t* accepted, int64_t* out,
                                void* workspace, size_t workspace_bytes, void* stream) {
  using namespace ss;
  const char* who = "ss_verify_drafts";
  SS_CHECK_ARG(dtype == SS_F16 || dtype == SS_F32 || dtype == SS_BF16, "%s: bad dtype %d", who,
               dtype);
  SS_CHECK_ARG(rows >= 0 && drafts >= 0 && vocab > 0 && vocab <= INT32_MAX - kChunk,
               "%s: bad sizes (rows %d, drafts %d, vocabulary %lld)", who, rows, drafts,
               (long long)vocab);
  SS_CHECK_ARG(temperature >= 0.0 && temperature < INFINITY,
               "%s: temperature must be finite and not negative", who);
  if (rows == 0) return SS_OK;
  const bool greedy = temperature == 0.0;
  SS_CHECK_ARG(target && accepted && out && (drafts == 0 || tokens) && (greedy || uniform),
               "%s: null pointer", who);
  SS_CHECK_ARG(drafts < 32768 && (int64_t)rows * (2 * (int64_t)drafts + 1) <= 65535,
               "%s: too many rows in one call", who);
  const size_t need = ss_verify_drafts_workspace_size(rows, drafts, vocab, draft != nullptr);
  SS_CHECK_ARG(need <= workspace_bytes && workspace && aligned16(workspace),
               "%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, need);
  const int64_t size = dtype == SS_F32 ? 4 : 2;
  const int chunks = (int)cdiv(vocab, kChunk);
  VerifyArgs a{(const char*)target, t_seq * size, t_row * size,
               greedy ? nullptr : (const char*)draft, d_seq * size, d_row * size, tokens, counts,
               uniform, rows, drafts, chunks, drafts + 1, vocab,
               // a finite number, or the maximum's own 0 times it is none
               greedy ? 1.0 : std::min(1.4426950408889634 / temperature, 1e300), accepted,
               out, (Stat*)workspace, nullptr, nullptr};
  if (a.draft) a.per += drafts;
  else a.d_seq = a.d_row = 0;
  a.parts = (double*)(a.stats + (int64_t)rows * (2 * drafts + 1) * chunks);
  a.choices = (Choice*)(a.parts + (int64_t)rows * chunks);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == SS_F16) return launch<half_t>(a, greedy, st);
  if (dtype == SS_BF16) return launch<bhalf_t>(a, greedy, st);
  return launch<float>(a, greedy, st);
}
