// Drafted tokens checked against the target's logits from given uniform numbers.
//
// p = softmax(target / T), q = softmax(draft / T); draft i is accepted while u_i q_i(x_i) <
// p_i(x_i).  At the first refusal the next token has the distribution max(p_i - q_i, 0), so
// that accepted and drawn tokens together are distributed as p; after no refusal it is drawn
// from p of the row behind the last draft.  Drawing inverts the running sum in token order.
//
// Probabilities and sums are fp64: a drawn token is the place of one number among up to
// 151936 running sums, and sums that are off by 1e-7 would name another token once in a
// hundred draws from a flat distribution.
//
// Three launches, each logit read once but for the chosen rows:
//   1. per (row, chunk of 8192 logits): maximum and sum of exp((l - max) / T) (or the
//      place of the maximum at T = 0);
//   2. per (sequence, chunk): the decisions, then the chunk's part of the chosen row's
//      max(p - q, 0) and p;
//   3. per sequence: the chunk in which the drawn number lies, and the token in it.
#include "paged.h"
#include "elementwise.h"

namespace ss {
namespace {

constexpr int kChunk = 8192;  // logits of a workgroup: 256 threads x 4 groups of 8

struct Stat {  // of a chunk, or of a row
  double sum;  // of weight(l, max)
  float max;
  int at;      // first place of the maximum (T = 0)
};

struct Choice {  // of a sequence
  double p_sum, q_sum;
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
  double inv_t;
  int32_t* accepted;
  int64_t* out;
  Stat* stats;      // target [rows][drafts + 1][chunks], then draft [rows][drafts][chunks]
  Choice* choices;  // [rows]
  double* parts;    // [2][rows][chunks]: max(p - q, 0), p

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

// exp((l - top) / T): 1 at the maximum (an infinite one included), 0 where there is none.
__device__ __forceinline__ double weight(float l, float top, double inv_t) {
  if (top == -INFINITY) return 0.0;
  if (l == top) return 1.0;
  return exp(((double)l - (double)top) * inv_t);
}

template <class T>
using Vec8 = T __attribute__((ext_vector_type(8)));

// Logits j .. j + 7 of a row; NaN and what lies behind the row's end are -inf.
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
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = x[e] == x[e] ? x[e] : -INFINITY;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

__device__ __forceinline__ double block_sum(double v, double* lds) {
  v = wave_sum_f64(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0] + lds[1] + lds[2] + lds[3];
  __syncthreads();
  return v;
}

template <class T, bool VEC, bool GREEDY>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs a) {
  __shared__ float tops[4];
  __shared__ double sums[4];
  __shared__ int places[4];
  const int chunk = blockIdx.x;
  const int b = blockIdx.y / a.per;
  const int i = blockIdx.y - b * a.per;
  const int n = a.count(b);
  const bool is_draft = i > a.drafts;
  if (is_draft ? i - a.drafts - 1 >= n : i > n) return;
  const char* row = is_draft ? a.draft + b * a.d_seq + (i - a.drafts - 1) * a.d_row
                             : a.target + b * a.t_seq + i * a.t_row;
  const int64_t j0 = (int64_t)chunk * kChunk + threadIdx.x * 8;
  float x[4][8];
#pragma unroll
  for (int g = 0; g < 4; ++g) load8<T, VEC>(row, j0 + g * 2048, a.vocab, x[g]);
  float top = -INFINITY;
#pragma unroll
  for (int g = 0; g < 4; ++g)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, x[g][e]);
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  Stat s{0.0, top, 0};
  if (GREEDY) {
    int at = INT32_MAX;
#pragma unroll
    for (int g = 3; g >= 0; --g)
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (x[g][e] == top) at = (int)(j0 + g * 2048 + e);
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) at = min(at, __shfl_xor(at, m, kWave));
    if ((threadIdx.x & 63) == 0) places[threadIdx.x >> 6] = at;
    __syncthreads();
    s.at = min(min(places[0], places[1]), min(places[2], places[3]));
  } else {
    double sum = 0.0;
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += weight(x[g][e], top, a.inv_t);
    s.sum = block_sum(sum, sums);
  }
  if (threadIdx.x == 0)
    (is_draft ? a.draft_stats(b, i - a.drafts - 1) : a.target_stats(b, i))[chunk] = s;
}

// Statistics of a whole row from its chunks', by one wave.
__device__ __forceinline__ Stat row_stat(const Stat* chunk, int chunks, double inv_t) {
  const int lane = threadIdx.x & 63;
  float top = -INFINITY;
  for (int c = lane; c < chunks; c += 64) top = fmaxf(top, chunk[c].max);
  top = wave_max(top);
  double sum = 0.0;
  int at = INT32_MAX;
  for (int c = lane; c < chunks; c += 64) {
    const Stat s = chunk[c];
    sum += s.sum * weight(s.max, top, inv_t);
    if (s.max == top) at = min(at, s.at);
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) at = min(at, __shfl_xor(at, m, kWave));
  return Stat{wave_sum_f64(sum), top, at};
}

template <class T>
__device__ __forceinline__ float logit(const char* row, int64_t j) {
  const float l = (float)reinterpret_cast<const T*>(row)[j];
  return l == l ? l : -INFINITY;
}

template <class T>
__device__ __forceinline__ bool accepts(const VerifyArgs& a, int b, int i) {
  const int64_t x = a.tokens[(int64_t)b * a.drafts + i];
  if (x < 0 || x >= a.vocab) return false;
  const Stat p = row_stat(a.target_stats(b, i), a.chunks, a.inv_t);
  const double px = weight(logit<T>(a.target + b * a.t_seq + i * a.t_row, x), p.max, a.inv_t);
  double qx = 1.0, q_sum = 1.0;
  if (a.draft) {
    const Stat q = row_stat(a.draft_stats(b, i), a.chunks, a.inv_t);
    qx = weight(logit<T>(a.draft + b * a.d_seq + i * a.d_row, x), q.max, a.inv_t);
    q_sum = q.sum;
  }
  const double u = a.uniform[(int64_t)b * (a.drafts + 1) + i];
  return u * (q_sum > 0.0 ? qx / q_sum : 0.0) < (p.sum > 0.0 ? px / p.sum : 0.0);
}

// max(p - q, 0) and p of eight logits of the chosen row.
struct Mass {
  double rest[8], p[8];
};
template <class T, bool VEC>
__device__ __forceinline__ Mass masses(const VerifyArgs& a, const Choice& c, int b, int64_t j) {
  Mass m;
  float x[8];
  load8<T, VEC>(a.target + b * a.t_seq + c.accepted * a.t_row, j, a.vocab, x);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    m.rest[e] = m.p[e] = c.p_sum > 0.0 ? weight(x[e], c.p_max, a.inv_t) / c.p_sum : 0.0;
  if (c.refused) {
    if (a.draft) {
      load8<T, VEC>(a.draft + b * a.d_seq + c.accepted * a.d_row, j, a.vocab, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double q = c.q_sum > 0.0 ? weight(x[e], c.q_max, a.inv_t) / c.q_sum : 0.0;
        m.rest[e] = fmax(m.p[e] - q, 0.0);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (j + e == c.drafted) m.rest[e] = 0.0;
    }
  }
  return m;
}

template <class T, bool VEC>
__global__ __launch_bounds__(256) void verify_rest_kernel(VerifyArgs a) {
  __shared__ int first;
  __shared__ Choice choice;
  __shared__ double sums[4];
  const int chunk = blockIdx.x, b = blockIdx.y;
  const int wave = threadIdx.x >> 6;
  const int n = a.count(b);
  if (threadIdx.x == 0) first = n;
  __syncthreads();
  for (int i = wave; i < n; i += 4) {
    if (!accepts<T>(a, b, i)) {
      if ((threadIdx.x & 63) == 0) atomicMin(&first, i);
      break;
    }
  }
  __syncthreads();
  if (wave == 0) {
    Choice c;
    c.accepted = first;
    c.refused = first < n;
    const Stat p = row_stat(a.target_stats(b, first), a.chunks, a.inv_t);
    c.p_sum = p.sum;
    c.p_max = p.max;
    c.q_sum = 0.0;
    c.q_max = -INFINITY;
    c.drafted = -1;
    if (c.refused) {
      const int64_t x = a.tokens[(int64_t)b * a.drafts + first];
      if (x >= 0 && x < a.vocab) c.drafted = (int)x;
      if (a.draft) {
        const Stat q = row_stat(a.draft_stats(b, first), a.chunks, a.inv_t);
        c.q_sum = q.sum;
        c.q_max = q.max;
      }
    }
    if (threadIdx.x == 0) {
      choice = c;
      if (chunk == 0) a.choices[b] = c;
    }
  }
  __syncthreads();
  const Choice c = choice;
  double rest = 0.0, p = 0.0;
  const int64_t j0 = (int64_t)chunk * kChunk + threadIdx.x * 8;
  for (int g = 0; g < 4; ++g) {
    const Mass m = masses<T, VEC>(a, c, b, j0 + g * 2048);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      rest += m.rest[e];
      p += m.p[e];
    }
  }
  rest = block_sum(rest, sums);
  p = block_sum(p, sums);
  if (threadIdx.x == 0) {
    a.parts[(int64_t)b * a.chunks + chunk] = rest;
    a.parts[(int64_t)(a.rows + b) * a.chunks + chunk] = p;
  }
}

template <class T, bool VEC>
__global__ __launch_bounds__(256) void verify_pick_kernel(VerifyArgs a) {
  __shared__ double scan[256];
  __shared__ int64_t drawn, last;
  const int b = blockIdx.x;
  const Choice c = a.choices[b];
  const double* rest = a.parts + (int64_t)b * a.chunks;
  const double* whole = a.parts + (int64_t)(a.rows + b) * a.chunks;
  double total = 0.0;
  for (int i = 0; i < a.chunks; ++i) total += rest[i];
  const bool use_p = !(total > 0.0);
  if (use_p) {
    total = 0.0;
    for (int i = 0; i < a.chunks; ++i) total += whole[i];
  }
  const double* part = use_p ? whole : rest;
  const double goal = (double)a.uniform[(int64_t)b * (a.drafts + 1) + a.drafts] * total;
  // The first chunk whose running sum exceeds the goal, or the last one that holds any.
  int chunk = -1;
  double sum = 0.0, ahead = 0.0;
  for (int i = 0; i < a.chunks; ++i) {
    if (part[i] > 0.0) {
      chunk = i;
      ahead = sum;
      if (sum + part[i] > goal) break;
    }
    sum += part[i];
  }
  if (threadIdx.x == 0) drawn = INT64_MAX, last = -1;
  int64_t token = -1;
  if (chunk >= 0) {
    const int64_t j0 = (int64_t)chunk * kChunk + threadIdx.x * 32;
    double mine = 0.0;
    double m[32];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const Mass q = masses<T, VEC>(a, c, b, j0 + g * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m[g * 8 + e] = use_p ? q.p[e] : q.rest[e];
        mine += m[g * 8 + e];
      }
    }
    scan[threadIdx.x] = mine;
    __syncthreads();
    double start = ahead;
    for (int i = 0; i < (int)threadIdx.x; ++i) start += scan[i];
    // Place of the first running sum above the goal, and of the last logit with any mass
    // (taken where rounding leaves the chunk's own sum at or below the goal).
    int64_t hit = INT64_MAX, any = -1;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      start += m[e];
      if (m[e] > 0.0) {
        any = j0 + e;
        if (start > goal && hit == INT64_MAX) hit = j0 + e;
      }
    }
    atomicMin((long long*)&drawn, (long long)hit);
    atomicMax((long long*)&last, (long long)any);
    __syncthreads();
    token = drawn != INT64_MAX ? drawn : last;
  }
  int64_t* out = a.out + (int64_t)b * (a.drafts + 1);
  for (int i = threadIdx.x; i <= a.drafts; i += 256)
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
  const dim3 block(256);
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
                     block, 0, st, a);
  SS_CHECK_LAUNCH("verify_rest_kernel");
  hipLaunchKernelGGL((verify_pick_kernel<T, VEC>), dim3((unsigned)a.rows), block, 0, st, a);
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
                         2 * chunks * sizeof(double));
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
               uniform, rows, drafts, chunks, drafts + 1, vocab, greedy ? 1.0 : 1.0 / temperature, accepted,
               out, (Stat*)workspace, nullptr, nullptr};
  if (a.draft) a.per += drafts;
  else a.d_seq = a.d_row = 0;
  a.parts = (double*)(a.stats + (int64_t)rows * (2 * drafts + 1) * chunks);
  a.choices = (Choice*)(a.parts + 2 * (int64_t)rows * chunks);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == SS_F16) return launch<half_t>(a, greedy, st);
  if (dtype == SS_BF16) return launch<bhalf_t>(a, greedy, st);
  return launch<float>(a, greedy, st);
}
