// Beam search: the best continuations of every request, and what follows from them.
//
//   c(b, v) = s_b + (x_bv - lse_b),   lse_b = log sum_v exp(x_bv)          of all beams b and tokens v the ``keep`` largest
//
// What bounds it is one pass over the logits (beams x vocabulary, 0.6 MB a row of the released models).  First kernel: every warp takes a group of a row's
// logits, 256 or 1024 of them, and leaves their maximum and sum of exponentials: no barriers, so the pass is as fast as memory.  Second
// kernel, a CTA per request: the rows' normalisers; a bound from below, the keep-th largest of the groups' maxima as scores, so only about as many
// groups as continuations are kept can hold one, and those are read again; what is not below the bound is ranked by counting.  Then the beams'
// bookkeeping, so that a whole step is captured without a look by the host.
//
// 151936 fp32 logits a row, in a graph: 16 requests of 8 beams 18.0 us, where their bytes alone take 11.9 and the second kernel 5; 4 beams 10.4, of which
// the second kernel's seven dependent phases are 7; a first step of 2 x 32 beams, 64 kept, 18.8.  A search's step (follow) takes 2 to 6 more: 20.9 for the 16
// requests, 12.8 for the 4 beams.  What is kept is ranked by one CTA, so that many beams with many ending tokens take longer: 2 x 64 beams
// with one 51, with two 64, with eight (576 kept) 211.  A first kernel that also chose the best of its
// slice of a row had barriers in its pass: 30 us for the 16 requests.
//
// Candidates of different beams may be closer than fp32 tells apart: a group's sum is of fp32 terms, from 32 terms on in 64 bits, and scores are compared in 64
// bits.  The largest term of a row is 1 exactly.  Another one, exp(-d), has an error of 2^-22 of itself from ex2, up to d 2^-24 from its rounded argument and
// d 2^-26 from the constant, the last always of one sign, and where many terms are alike so are the others.  So normalisers are good to some 1e-8 for random
// logits, to 3e-7 where one logit is far above 151935 others that are alike, and candidates of different beams are told apart to that; those of one beam always
// are.  Equal scores: the lower beam, then the lower token.
// A row with NaN, + inf or nothing but - inf has no candidates.
#include <float.h>
#include <math.h>
#include <string.h>

#include <mutex>

#include "host_common.h"
#include "sm100_common.cuh"

namespace snu1 {
namespace beam {

constexpr int THREADS = 256;
constexpr int MAX_BEAMS = 64;
constexpr int MAX_EOS = 8;
// A search's step: every beam may end in each of the ending tokens, so that the beams' number of others is only certain among as many.
constexpr int MAX_KEEP = MAX_BEAMS * (1 + MAX_EOS);

__device__ __forceinline__ uint32_t order32(float x) {          // keeps the order, - 0 equal to 0
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order64(double x) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(x + 0.0);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double value64(unsigned long long k) {
  return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Group {         // of a row's logits
  double sum;          // of exp(x - max)
  float quarter[4];    // maxima of its quarters; NaN if the group holds one
};
__device__ __forceinline__ float top_of(const Group& g) { return fmaxf(fmaxf(g.quarter[0], g.quarter[1]), fmaxf(g.quarter[2], g.quarter[3])); }

struct PassArgs {
  const void* logits;
  long long ld;        // elements from row to row
  int V, rows, groups; // groups of a row
  Group* out;          // [rows][groups]
};

// Token of a lane's value j of a group of 32 E; a lane has 16 bytes of every 512, eight lanes a quarter.
template <typename T, int E>
__device__ __forceinline__ int token_of(int group, int lane, int j) {
  constexpr int VEC = 16 / sizeof(T);
  return group * 32 * E + ((j / VEC) * 32 + lane) * VEC + j % VEC;
}
// A lane's values of a group, by token and not by address: the sum of a row does not depend on where it lies, so that beams with the same logits have
// the same scores.  - inf behind the last.
template <typename T, int E>
__device__ __forceinline__ void load_group(const T* x, int V, int group, int lane, float (&v)[E]) {
  constexpr int VEC = 16 / sizeof(T);
  const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
#pragma unroll
  for (int j = 0; j < E; j += VEC) {
    const int i = token_of<T, E>(group, lane, j);
    if (aligned && i + VEC <= V) {
      const uint4 u = *reinterpret_cast<const uint4*>(x + i);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (sizeof(T) == 4) v[j + e] = __uint_as_float(w[e & 3]);
        else v[j + e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[j + e] = i + e < V ? (float)x[i + e] : -INFINITY;
    }
  }
}

// A warp: a group's maxima and sum.
template <typename T, int E>
__device__ __forceinline__ void sum_group(const T* x, int V, int group, Group* out) {
  const int lane = threadIdx.x & 31;
  float v[E];
  load_group<T, E>(x, V, group, lane, v);
  float m = v[0];                                        // (NaN is passed over)
#pragma unroll
  for (int j = 1; j + 1 < E; j += 2) m = fmaxf(m, fmaxf(v[j], v[j + 1]));
  m = fmaxf(m, v[E - 1]);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float quarter = m;                               // eight lanes'
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  constexpr float LOG2E = 1.44269502162933349609375f;
  const float from = m > -INFINITY ? m : 0.f;
  float sum = 0.f;                                       // NaN if there is one
#pragma unroll
  for (int j = 0; j < E; ++j) sum += ex2((v[j] - from) * LOG2E);
  double total = sum;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if ((lane & 7) == 0) out->quarter[lane >> 3] = total == total ? quarter : __int_as_float(0x7fffffff);
  if (lane == 0) out->sum = total;
}

template <typename T, int E>
__global__ void __launch_bounds__(THREADS) pass_kernel(const PassArgs a) {
  const int row = blockIdx.y, group = blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  pdl_wait();
  pdl_trigger();
  if (group >= a.groups) return;
  sum_group<T, E>(reinterpret_cast<const T*>(a.logits) + row * a.ld, a.V, group, a.out + (long long)row * a.groups + group);
}

constexpr int JOIN_THREADS = 1024;
constexpr int JOIN_LIST = 2048;      // candidates that fit; where more are not below the bound, it is raised to the keep-th best of these
constexpr int RANKED = 384;          // as many are ranked at once
constexpr int JOIN_GROUPS = 1024;    // groups that fit a list; more are looked for by every warp in its own share

// A search's state (all on the device); see ops/beam.py.
struct State {
  float* scores;           // [requests][beams]
  long long* tokens;       // [requests * beams] what the next step reads
  int* parents;            // [requests * beams] row that a beam goes on from
  int* history_token;      // [steps][requests][beams]
  int* history_parent;     // [steps][requests][beams] beam of the step before
  float* pool_score;       // [requests][beams] finished ones, by score / length^penalty
  int* pool_step;          // their last step, -1: free
  int* pool_parent;        // the beam that they left ...
  int* pool_token;         // ... with this token
  int* done;               // [requests]
  int* step;               // [requests]
  int steps, pad;
  float penalty;
  int early;               // 0: until no beam can be better at its present length; 1: as soon as there are enough; 2: at any length
  int eos_count;
  int eos[MAX_EOS];
};

struct JoinArgs {
  const void* logits;
  long long ld;
  int V, groups;
  Group* group;            // [requests * beams][groups]
  const float* scores;     // [requests][beams]
  float* out_scores;       // [requests][keep]
  int* out_beams;
  int* out_tokens;
  int beams, keep, has_state;
  int* status;
  State st;
};

// Which is first: the larger score, then the lower beam, then the larger logit (two logits may give one score), then the lower token.
struct Best {
  unsigned long long s, key;
  uint32_t beam;
};
__device__ __forceinline__ bool before(const Best& x, const Best& y) {
  return x.s > y.s || (x.s == y.s && (x.beam < y.beam || (x.beam == y.beam && x.key > y.key)));
}

struct Chosen {
  float score[MAX_KEEP];
  int beam[MAX_KEEP], token[MAX_KEEP];
  int pick[MAX_BEAMS];                                    // the candidate that a beam goes on with
  float pool_score[MAX_BEAMS];
  int pool_step[MAX_BEAMS], pool_pick[MAX_BEAMS];         // pool_pick: the candidate that has just come in, -1: none, -2 - beam: a beam as it is
  int beams, done;
};

// The search's next step; all threads of the block, after ``c``'s candidates are written and seen.
__device__ void follow(const JoinArgs& a, int r, Chosen& c) {
  const State& s = a.st;
  const int K = a.beams, tid = threadIdx.x, t = s.step[r];
  const long long at = (long long)r * K;
  if (t >= s.steps) {                                     // more steps than the search has room for
    if (tid == 0) report_status(a.status, kBadShape, 11);
    return;
  }
  if (tid < K) {
    c.pool_score[tid] = s.pool_score[at + tid];
    c.pool_step[tid] = s.pool_step[at + tid];
    c.pool_pick[tid] = -1;
  }
  if (tid == 0) c.done = s.done[r];
  __syncthreads();
  if (tid == 0) {
    int n = 0;
    if (c.done == 0) {
      const float len = powf((float)(t + 1), s.penalty);
      auto worst = [&]() {                                // a free place, else the lowest score (of equal ones the last)
        int w = 0;
        for (int i = 0; i < K; ++i) {
          if (c.pool_step[i] < 0) return i;
          if (c.pool_score[i] <= c.pool_score[w]) w = i;
        }
        return w;
      };
      auto finish = [&](float x, int step, int pick) {
        const int w = worst();
        if (c.pool_step[w] < 0 || x > c.pool_score[w]) {
          c.pool_score[w] = x;
          c.pool_step[w] = step;
          c.pool_pick[w] = pick;
        }
      };
      for (int i = 0; i < a.keep && n < K; ++i) {
        if (c.score[i] == -INFINITY) break;
        bool eos = false;
        for (int k = 0; k < s.eos_count; ++k) eos |= c.token[i] == s.eos[k];
        if (!eos) {
          c.pick[n++] = i;
        } else if (i < K) {
          finish(c.score[i] / len, t, i);
        }
      }
      if (c.score[0] == -INFINITY && t > 0) {        // no beam has a continuation: they count as they are
        const float now = powf((float)t, s.penalty);
        for (int b = 0; b < K; ++b)
          if (s.scores[at + b] > -INFINITY) finish(s.scores[at + b] / now, t - 1, -2 - b);
      }
      const int w = worst();
      bool done = n == 0;
      if (c.pool_step[w] >= 0 && n > 0) {
        const float most = s.early == 2 && s.penalty > 0.f ? powf((float)s.steps, s.penalty) : len;
        done = s.early == 1 || c.pool_score[w] >= c.score[c.pick[0]] / most;
      }
      c.done = done ? 2 : 0;                              // 2: now
    }
    c.beams = n;
    s.step[r] = t + 1;
  }
  __syncthreads();
  if (tid >= K) return;
  const int n = c.done ? 0 : c.beams, pad = s.eos_count > 0 && s.eos[0] < a.V ? s.eos[0] : 0;        // (its embedding is looked up)
  const bool on = tid < n;                                // (a row that does not go on stays where it is)
  const int pick = on ? c.pick[tid] : 0, token = on ? c.token[pick] : pad, from = on ? c.beam[pick] : tid;
  const long long h = ((long long)t * gridDim.x + r) * K + tid;
  if (c.done != 1) s.scores[at + tid] = on ? c.score[pick] : -INFINITY;
  s.tokens[at + tid] = token;
  s.parents[at + tid] = r * K + from;
  s.history_token[h] = token;
  s.history_parent[h] = from;
  const int in = c.pool_pick[tid];
  if (in != -1) {
    const long long was = ((long long)(t - 1) * gridDim.x + r) * K - 2 - in;          // (of a beam as it is: its last token)
    s.pool_score[at + tid] = c.pool_score[tid];
    s.pool_step[at + tid] = c.pool_step[tid];
    s.pool_parent[at + tid] = in >= 0 ? c.beam[in] : s.history_parent[was];
    s.pool_token[at + tid] = in >= 0 ? c.token[in] : s.history_token[was];
  }
  if (tid == 0 && c.done == 2) s.done[r] = 1;
}

// Groups of a request up to which its one CTA takes them all: one launch less, no scratch.  Us in a graph (called from Python), with / without: 12 groups
// 7.6 / 8.2 (12.9 / 17.1), 32 7.9 / 8.3 (12.9 / 16.8), 64 8.9 / 8.3 (12.8 / 17.2), 128 10.5 / 8.5 (12.9 / 17.5).
constexpr int ALONE_GROUPS = 64;

struct JoinShared {
  double lse[MAX_BEAMS];
  float base[MAX_BEAMS], least[MAX_BEAMS];
  unsigned long long set[JOIN_THREADS], top[JOIN_THREADS], nth, list_s[JOIN_LIST];      // (list_s: the candidates' scores once more, to be counted)
  Best list[JOIN_LIST];
  int pass[JOIN_GROUPS], quarter[JOIN_GROUPS];
  short pick[JOIN_LIST];
  Best bound;
  int passing, count;
  Chosen out;
  Group alone[ALONE_GROUPS];
};

// ALONE: the groups' maxima and sums too, in shared memory.
template <typename T, int E, bool ALONE>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const JoinArgs a) {
  extern __shared__ unsigned long long s_raw[];
  JoinShared& sh = *reinterpret_cast<JoinShared*>(s_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.x, K = a.beams, keep = a.keep;
  if (tid == 0) sh.bound = Best{1, 0, 0xffffffffu};        // everything that is a candidate
  for (int i = tid; i < keep; i += JOIN_THREADS) {
    sh.out.score[i] = -INFINITY;
    sh.out.beam[i] = sh.out.token[i] = 0;
  }
  pdl_wait();
  pdl_trigger();
  const int all = K * a.groups;
  Group* group = ALONE ? sh.alone : a.group + (long long)r * all;
  const T* logits = reinterpret_cast<const T*>(a.logits) + (long long)r * K * a.ld;
  if (ALONE) {
    for (int i = warp; i < all; i += JOIN_THREADS / 32) sum_group<T, E>(logits + i / a.groups * a.ld, a.V, i % a.groups, group + i);
    __syncthreads();
  }
  // normalisers: NaN where the row has no candidates
  for (int b = warp; b < K; b += JOIN_THREADS / 32) {
    const Group* p = group + (long long)b * a.groups;
    constexpr int HELD = 5;                                // of a lane; more are looked up again
    const float base = a.scores[(long long)r * K + b];
    double sums[HELD];
    float tops[HELD];
    float m = -INFINITY;
    bool bad = !(fabsf(base) < INFINITY);                  // (a beam that is not there)
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      tops[i] = -INFINITY;
      sums[i] = 0.0;
      if (lane + 32 * i < a.groups) {
        tops[i] = top_of(p[lane + 32 * i]);
        sums[i] = p[lane + 32 * i].sum;
      }
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      bad |= !(tops[i] < INFINITY);
      m = fmaxf(m, tops[i]);
    }
#pragma unroll 4
    for (int i = lane + 32 * HELD; i < a.groups; i += 32) {
      const float y = top_of(p[i]);
      bad |= !(y < INFINITY);
      m = fmaxf(m, y);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    bad = __any_sync(0xffffffffu, bad) || m == -INFINITY;
    double sum = 0.0;
    if (!bad) {
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        if (tops[i] > -INFINITY) sum += sums[i] * exp((double)tops[i] - (double)m);
#pragma unroll 4
      for (int i = lane + 32 * HELD; i < a.groups; i += 32) {
        const float y = top_of(p[i]);
        if (y > -INFINITY) sum += p[i].sum * exp((double)y - (double)m);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      sh.lse[b] = bad ? (double)NAN : (double)m + log(sum);
      sh.base[b] = base;
    }
  }
  __syncthreads();
  // a logit's score as a number that can be compared; 0: it is no candidate
  auto score_of = [&](float x, int b) -> unsigned long long {
    const double score = (double)sh.base[b] + ((double)x - sh.lse[b]);
    return x > -INFINITY && score > -INFINITY && score < INFINITY ? order64(score) : 0ull;       // (false for NaN)
  };
  constexpr int OWN = 2;                                   // the first groups of a thread: their maxima as scores, looked up once
  unsigned long long own[OWN];
#pragma unroll
  for (int k = 0; k < OWN; ++k) {
    const int i = tid + k * JOIN_THREADS;
    own[k] = i < all ? score_of(top_of(group[i]), i / a.groups) : 0ull;
  }
  // The keep-th largest of the largest of 64 to 1024 sets of the threads' values, every 64th to 1024th thread a set (threads side by side are in
  // different ones, so that few values are a set each); 0 if fewer sets have any.  Its place is counted by ``share`` threads.
  auto nth_of = [&](unsigned long long mine) -> unsigned long long {
    const int share = keep <= 32 ? 16 : keep <= 64 ? 8 : keep <= 128 ? 4 : keep <= 256 ? 2 : 1, values = JOIN_THREADS / share, sub = tid & (share - 1);
    sh.set[tid] = mine;
    if (tid == 0) sh.nth = 0;
    __syncthreads();
    mine = sh.set[tid / share + sub * values];
    for (int o = 1; o < share; o <<= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if (sub == 0) sh.top[tid / share] = mine;
    __syncthreads();
    int above = 0, equal = 0;
#pragma unroll 4
    for (int i = sub; i < values; i += share) {
      const unsigned long long x = sh.top[i];
      above += x > mine;
      equal += x == mine;
    }
    for (int o = 1; o < share; o <<= 1) {
      above += __shfl_xor_sync(0xffffffffu, above, o);
      equal += __shfl_xor_sync(0xffffffffu, equal, o);
    }
    if (sub == 0 && mine != 0 && above < keep && above + equal >= keep) sh.nth = mine;            // (whoever writes, writes the same)
    __syncthreads();
    return sh.nth;
  };
  {
    // the bound, from the groups' maxima
    unsigned long long mine = 0;
#pragma unroll
    for (int k = 0; k < OWN; ++k) mine = max(mine, own[k]);
#pragma unroll 4
    for (int i = tid + OWN * JOIN_THREADS; i < all; i += JOIN_THREADS) mine = max(mine, score_of(top_of(group[i]), i / a.groups));
    // (of few groups, the first step's one beam, say, from their quarters)
    if (all <= JOIN_THREADS / 4 || __syncthreads_count(mine != 0) < 2 * keep) {
      mine = 0;
#pragma unroll 4
      for (int i = tid; i < 4 * all; i += JOIN_THREADS) mine = max(mine, score_of(group[i >> 2].quarter[i & 3], (i >> 2) / a.groups));
    }
    const unsigned long long nth = nth_of(mine);
    if (tid == 0 && nth != 0) sh.bound.s = nth;
  }
  if (tid == 0) sh.count = sh.passing = 0;
  __syncthreads();
  int n;
  for (bool exactly = false;; exactly = true) {
    const Best bound = sh.bound;
    // The groups that can hold a candidate, and for every beam a logit that is a little below what the bound's score asks for.
    auto see = [&](unsigned long long s, int i) {
      if (s >= bound.s) {
        const int at = atomicAdd(&sh.passing, 1);
        if (at < JOIN_GROUPS) sh.pass[at] = i;
      }
    };
#pragma unroll
    for (int k = 0; k < OWN; ++k) see(own[k], tid + k * JOIN_THREADS);
#pragma unroll 4
    for (int i = tid + OWN * JOIN_THREADS; i < all; i += JOIN_THREADS) see(score_of(top_of(group[i]), i / a.groups), i);
    if (tid < K) {
      const double to = value64(bound.s), from = sh.base[tid], x = to - from + sh.lse[tid];
      sh.least[tid] = bound.s == 1 ? -FLT_MAX
                                   : fmaxf((float)(x - 1e-6 * fabs(x) - 1e-15 * (fabs(to) + fabs(from) + fabs(sh.lse[tid]))) - FLT_MIN, -FLT_MAX);
    }
    __syncthreads();
    const int passing = sh.passing;
    const bool listed = passing <= JOIN_GROUPS;
    // More of them than warps: only their quarters that can, four to a warp (2 x 32 beams of 151936, first step 21.3 -> 18.7 us; for 8 groups 0.7 more).
    int quarters = -1;
    if (listed && passing > JOIN_THREADS / 32) {
      if (tid == 0) sh.count = 0;
      __syncthreads();
      for (int i = tid; i < 4 * passing; i += JOIN_THREADS) {
        const int g = sh.pass[i >> 2];
        if (score_of(group[g].quarter[i & 3], g / a.groups) >= bound.s) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < JOIN_GROUPS) sh.quarter[at] = 4 * g + (i & 3);
        }
      }
      __syncthreads();
      if (sh.count <= JOIN_GROUPS) quarters = sh.count;
      __syncthreads();
      if (tid == 0) sh.count = 0;
      __syncthreads();
    }
    for (int i = warp; i < (quarters >= 0 ? (quarters + 3) / 4 : listed ? passing : all); i += JOIN_THREADS / 32) {     // eight lanes have a quarter
      const int sub = lane >> 3;
      const int at = quarters < 0 ? 4 * (listed ? sh.pass[i] : i) + sub : 4 * i + sub < quarters ? sh.quarter[4 * i + sub] : 0;
      const int g = at >> 2, b = g / a.groups, from = (at & 3) * 8 + (lane & 7);
      const bool on = quarters < 0 ? listed || score_of(group[g].quarter[at & 3], b) >= bound.s : 4 * i + sub < quarters;
      if (!__any_sync(0xffffffffu, on)) continue;
      float v[E];
      load_group<T, E>(logits + b * a.ld, a.V, g - b * a.groups, from, v);
      const float least = on ? sh.least[b] : INFINITY;
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (v[j] >= least) {
          const unsigned long long key = (unsigned long long)order32(v[j]) << 32 | (uint32_t)~token_of<T, E>(g - b * a.groups, from, j);
          if (!exactly || !before(bound, Best{score_of(v[j], b), key, (uint32_t)b})) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < JOIN_LIST) sh.list[at] = Best{(unsigned long long)__float_as_uint(v[j]), key, (uint32_t)b};
          }
        }
    }
    __syncthreads();
    n = sh.count;
    const int here = min(n, JOIN_LIST);
    for (int i = tid; i < here; i += JOIN_THREADS) sh.list_s[i] = sh.list[i].s = score_of(__uint_as_float((uint32_t)sh.list[i].s), (int)sh.list[i].beam);
    __syncthreads();                                       // (everybody has read the count)
    if (tid == 0) sh.count = sh.passing = 0;
    // of many only those are ranked that can be among the best
    int few = here;
    const bool picked = here > RANKED;
    if (picked) {
      unsigned long long mine = 0;
      for (int i = tid; i < here; i += JOIN_THREADS) mine = max(mine, sh.list_s[i]);
      const unsigned long long nth = max(nth_of(mine), 1ull);
      for (int i = tid; i < here; i += JOIN_THREADS)
        if (sh.list_s[i] >= nth) sh.pick[atomicAdd(&sh.count, 1)] = (short)i;
      __syncthreads();
      few = sh.count;
      __syncthreads();
      if (tid == 0) sh.count = 0;
    }
    int share = 1;                                         // threads for one candidate (a power of two, neighbours)
    while (2 * share * few <= JOIN_THREADS && share < 32) share *= 2;
    for (int i0 = 0; i0 < few; i0 += JOIN_THREADS / share) {
      const int i = i0 + tid / share, sub = tid & (share - 1), at = i < few && picked ? sh.pick[i] : i;
      const Best e = i < few ? sh.list[at] : Best{0, 0, 0};
      int rank = 0;
#pragma unroll 4
      for (int k = sub; k < few; k += share) {
        const int other = picked ? sh.pick[k] : k;
        const unsigned long long s = sh.list_s[other];
        rank += s > e.s;
        if (s == e.s) rank += before(sh.list[other], e);   // (itself, seldom another)
      }
      for (int o = 1; o < share; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
      if (sub == 0 && e.s != 0 && rank < keep) {
        sh.out.score[rank] = (float)value64(e.s);
        sh.out.beam[rank] = (int)e.beam;
        sh.out.token[rank] = (int)~(uint32_t)e.key;
        if (rank == keep - 1) sh.bound = e;
      }
    }
    __syncthreads();
    // Where more pass than fit (equal logits, say), the keep-th best of these is a better bound, and is kept to exactly: every time at
    // least those of them that are behind it pass no more.
    if (n <= JOIN_LIST) break;
  }
  if (a.has_state) {
    follow(a, r, sh.out);
    return;
  }
  for (int i = tid; i < keep; i += JOIN_THREADS) {
    a.out_scores[(long long)r * keep + i] = sh.out.score[i];
    a.out_beams[(long long)r * keep + i] = sh.out.beam[i];
    a.out_tokens[(long long)r * keep + i] = sh.out.token[i];
  }
}

// Values per lane of a group: of short rows 8, so that there are several times as many groups as continuations are kept.
static int group_of(int V) { return V >= 32768 ? 32 : 8; }
static int groups_of(int E, int V) { return (V + 32 * E - 1) / (32 * E); }

static bool alone(int beams, int V) { return group_of(V) == 8 && (long long)beams * groups_of(8, V) <= ALONE_GROUPS; }

template <typename T, int E, bool ALONE>
static int launch_join(const JoinArgs& j, int requests, cudaStream_t st) {
  int dev = 0;
  SNU1_CUDA_CHECK(cudaGetDevice(&dev));
  static std::once_flag once[64];
  cudaError_t err = cudaSuccess;
  std::call_once(once[dev & 63], [&]() { err = cudaFuncSetAttribute(join_kernel<T, E, ALONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(JoinShared)); });
  SNU1_CUDA_CHECK(err);
  SNU1_CUDA_CHECK(launch_pdl(join_kernel<T, E, ALONE>, dim3(requests), dim3(JOIN_THREADS), sizeof(JoinShared), st, j));
  return kHostOk;
}

template <typename T, int E>
static int launch(const PassArgs& a, const JoinArgs& j, int requests, cudaStream_t st) {
  constexpr int WARPS = THREADS / 32;
  SNU1_CUDA_CHECK(launch_pdl(pass_kernel<T, E>, dim3((a.groups + WARPS - 1) / WARPS, a.rows), dim3(THREADS), 0, st, a));
  return launch_join<T, E, false>(j, requests, st);
}

}  // namespace beam
}  // namespace snu1

using namespace snu1;

SNU1_API int snu1_beam_state_bytes() { return (int)sizeof(beam::State); }

// Launches of a step.
SNU1_API int snu1_beam_launches(int beams, int V) { return beam::alone(beams, V) ? 1 : 2; }

// Bytes of scratch for ``rows`` rows of ``V`` logits, ``beams`` of each request; may be 0.
SNU1_API long long snu1_beam_scratch_bytes(int rows, int beams, int V) {
  return beam::alone(beams, V) ? 0 : (long long)rows * beam::groups_of(beam::group_of(V), V) * (long long)sizeof(beam::Group);
}

// logits [requests * beams][V] (fp32, or bf16 with is_bf16), rows ld elements apart; scores [requests][beams] fp32.  Without ``state`` the best
// ``keep`` of every request go to out_*; with it (a beam::State) they become the search's next step.
SNU1_API int snu1_beam_step(const void* logits, long long ld, int is_bf16, int V, const void* scores, int requests, int beams, int keep,
                            void* scratch, void* out_scores, void* out_beams, void* out_tokens, const void* state, void* stream) {
  using namespace beam;
  const long long rows = (long long)requests * beams;
  if (requests <= 0 || beams <= 0 || beams > MAX_BEAMS || rows > 65535 || V <= 0 || V > (1 << 24) || keep <= 0 || keep > MAX_KEEP ||
      keep > (long long)beams * V || ld < V || ((reinterpret_cast<uintptr_t>(scratch) & 15) != 0)) {
    set_last_error("beam_step: %d requests of %d beams (at most %d), %d tokens, %d kept (at most %d)", requests, beams, MAX_BEAMS, V, keep,
                   MAX_KEEP);
    return kHostBadArg;
  }
  const int E = group_of(V);
  PassArgs a;
  a.logits = logits;
  a.ld = ld;
  a.V = V;
  a.rows = (int)rows;
  a.groups = groups_of(E, V);
  a.out = (Group*)scratch;
  JoinArgs j;
  memset(&j, 0, sizeof(j));
  j.logits = logits;
  j.ld = ld;
  j.V = V;
  j.groups = a.groups;
  j.group = a.out;
  j.scores = (const float*)scores;
  j.out_scores = (float*)out_scores;
  j.out_beams = (int*)out_beams;
  j.out_tokens = (int*)out_tokens;
  j.beams = beams;
  j.keep = keep;
  j.status = device_status_word();
  if (state != nullptr) {
    j.has_state = 1;
    memcpy(&j.st, state, sizeof(State));
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (alone(beams, V))
    return is_bf16 ? launch_join<__nv_bfloat16, 8, true>(j, requests, st) : launch_join<float, 8, true>(j, requests, st);
  if (is_bf16) return E == 32 ? launch<__nv_bfloat16, 32>(a, j, requests, st) : launch<__nv_bfloat16, 8>(a, j, requests, st);
  return E == 32 ? launch<float, 32>(a, j, requests, st) : launch<float, 8>(a, j, requests, st);
}
