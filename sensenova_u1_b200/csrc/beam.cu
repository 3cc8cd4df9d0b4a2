// Beam search: the best continuations of every request, and what follows from them.
//
//   c(b, v) = s_b + (x_bv - lse_b),   lse_b = log sum_v exp(x_bv)          of all beams b and tokens v the ``keep`` largest
//
// What bounds it is one pass over the logits (beams x vocabulary, 0.6 MB a row of the released models).  First kernel: a CTA
// holds a slice of a row in registers, leaves its maximum and sum of exponentials, and its ``keep`` largest logits: within a row the
// order of the candidates is that of the logits, so no normaliser is needed to choose them.  A bound from below comes from
// the largest values of small groups of threads (the keep-th of them), few values pass it, and those are ranked by counting.  Second kernel, a
// CTA per request: the rows' normalisers, the slices' lists (sorted, so their heads give a bound the same way), the ``keep``
// best by score, and the beams' bookkeeping, so that a whole step is captured without a look by the host.
//
// Candidates of different beams may be closer than fp32 tells apart: a slice's sum is of fp32 terms, from 32 terms on in 64 bits (the largest
// term of a row is 1 exactly, the errors of the others, 2^-22 of each at most, are of either sign: 1e-8 of the normaliser where they were measured),
// and scores are compared in 64 bits.  Equal scores: the lower beam, then the lower token.
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
constexpr int MAX_KEEP = 128;
constexpr int MAX_EOS = 8;

__device__ __forceinline__ uint32_t order32(float x) {          // keeps the order, - 0 equal to 0
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value32(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
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

struct Part {          // of a slice
  double sum;          // of exp(x - max)
  float max;           // NaN if the slice holds one
  int pad;
};

struct PickArgs {
  const void* logits;
  long long ld;                      // elements from row to row
  int V, keep, slices;
  int share, second, room;           // threads of a group and which of its values gives the bound, see launch_pick; candidates that fit
  Part* part;                        // [rows][slices]
  unsigned long long* cand;          // [rows][slices][keep] (logit, complement of the token), largest first, 0: none
};

// E values per thread, by token and not by address: the sum of a row does not depend on where it lies, so that beams with the same logits have the
// same scores.  16 bytes are loaded at once if rows are aligned to them.
template <typename T, int E>
__global__ void __launch_bounds__(THREADS, 4) pick_kernel(const PickArgs a) {
  constexpr int VEC = 16 / sizeof(T), LOADS = E / VEC;
  extern __shared__ unsigned long long s_list[];       // [keep * most values of a group]
  __shared__ float s_top[THREADS];
  __shared__ unsigned long long s_key[THREADS];
  __shared__ double s_sum[THREADS / 32];
  __shared__ float s_max[THREADS / 32], s_least;
  __shared__ unsigned long long s_bound;
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.y, slice = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld;
  const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  if (tid == 0) {
    s_count = 0;
    s_bound = 1;
    s_least = -FLT_MAX;                                  // everything but - inf and NaN
  }
  pdl_wait();
  pdl_trigger();
  float v[E];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int i = ((slice * LOADS + j) * THREADS + tid) * VEC;                    // token of the first of VEC
    if (aligned && i + VEC <= a.V) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4*>(x + i));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (sizeof(T) == 4) v[j * VEC + e] = __uint_as_float(w[e & 3]);
        else v[j * VEC + e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[j * VEC + e] = i + e < a.V ? (float)x[i + e] : -INFINITY;
    }
  }
  const auto token = [&](int j) { return ((slice * LOADS + j / VEC) * THREADS + tid) * VEC + j % VEC; };
  const auto key = [&](float y, int j) -> unsigned long long { return (unsigned long long)order32(y) << 32 | (uint32_t)~token(j); };
  float top = v[0];                                      // (NaN is passed over)
#pragma unroll
  for (int j = 1; j + 1 < E; j += 2) top = fmaxf(top, fmaxf(v[j], v[j + 1]));
  top = fmaxf(top, v[E - 1]);
  if (!(top > -INFINITY)) top = -INFINITY;
  // The group's value: its threads' largest, or with ``second`` their second largest, which has two values that are not below it.
  const int share = a.share;
  float mine = top, other = -INFINITY;
  for (int o = 1; o < share; o <<= 1) {
    const float x = __shfl_xor_sync(0xffffffffu, mine, o), y = __shfl_xor_sync(0xffffffffu, other, o);
    other = fmaxf(fminf(mine, x), fmaxf(other, y));
    mine = fmaxf(mine, x);
  }
  if (a.second) mine = other;
  if ((tid & (share - 1)) == 0) s_top[tid / share] = mine;
  float m = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) s_max[warp] = m;
  __syncthreads();
  m = -INFINITY;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) m = fmaxf(m, s_max[w]);
  // The bound: of the groups' values the keep-th largest (with ``second`` half as many suffice), found by counting those above each; the
  // threads of a group share the count.
  {
    const int sub = tid & (share - 1), groups = THREADS / share, nth = a.second ? (a.keep + 1) / 2 : a.keep;
    int above = 0, equal = 0;
#pragma unroll 4
    for (int i = sub; i < groups; i += share) {
      const float x = s_top[i];
      above += x > mine;
      equal += x == mine;
    }
    for (int o = 1; o < share; o <<= 1) {
      above += __shfl_xor_sync(0xffffffffu, above, o);
      equal += __shfl_xor_sync(0xffffffffu, equal, o);
    }
    if (sub == 0 && above < nth && above + equal >= nth && mine > -INFINITY) s_least = mine;      // (whoever writes, writes the same)
  }
  // The sum; NaN if there is one.
  float sum = 0.f;
  constexpr float LOG2E = 1.44269502162933349609375f;
#pragma unroll
  for (int j = 0; j < E; ++j) sum += ex2((v[j] - (m > -INFINITY ? m : 0.f)) * LOG2E);
  double total = sum;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s_sum[warp] = total;
  __syncthreads();
  if (tid == 0) {
    Part p;
    p.sum = 0.0;
    for (int w = 0; w < THREADS / 32; ++w) p.sum += s_sum[w];
    p.max = p.sum == p.sum ? m : __int_as_float(0x7fffffff);
    p.pad = 0;
    a.part[(long long)row * a.slices + slice] = p;
  }
  {
    const float least = s_least;
    if (top >= least) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (v[j] >= least) {
          const int at = atomicAdd(&s_count, 1);
          if (at < a.room) s_list[at] = key(v[j], j);
        }
    }
  }
  __syncthreads();
  if (s_count > a.room) {
    // Too many pass: equal values, or all that are large in a few threads.  Once more by value and token, which are never equal, and with the threads' own
    // best, of which ``keep`` have any that passes.
    unsigned long long best = 0;
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (v[j] > -INFINITY) best = max(best, key(v[j], j));
    __syncthreads();
    s_key[tid] = best;
    if (tid == 0) s_count = 0;
    __syncthreads();
    int above = 0;
    for (int i = 0; i < THREADS; ++i) above += s_key[i] > best;
    if (above == a.keep - 1 && best > 0) s_bound = best;
    __syncthreads();
    const unsigned long long bound = s_bound;
    if (best >= bound) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (v[j] > -INFINITY && key(v[j], j) >= bound) s_list[atomicAdd(&s_count, 1)] = key(v[j], j);
    }
    __syncthreads();
  }
  const int n = s_count;
  unsigned long long* out = a.cand + ((long long)row * a.slices + slice) * a.keep;
  for (int i = tid; i < n; i += THREADS) {
    const unsigned long long mine = s_list[i];
    int rank = 0;
    for (int k = 0; k < n; ++k) rank += s_list[k] > mine;
    if (rank < a.keep) out[rank] = mine;
  }
  for (int i = n + tid; i < a.keep; i += THREADS) out[i] = 0;
}

constexpr int JOIN_THREADS = 512;
constexpr int JOIN_LISTS = 1280;     // lists with candidates whose heads are held; of more the bound is that of every thread's best head
constexpr int JOIN_LIST = 1024;      // candidates that are ranked by counting; more than that are taken one by one
constexpr int JOIN_GROUPS = 256;     // values that the bound is found among, by counting
constexpr int MAX_BEAMS = 64;

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
  const Part* part;
  const unsigned long long* cand;
  const float* scores;     // [requests][beams]
  float* out_scores;       // [requests][keep]
  int* out_beams;
  int* out_tokens;
  int beams, keep, slices, has_state;
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
  int pool_step[MAX_BEAMS], pool_pick[MAX_BEAMS];         // pool_pick: the candidate that has just come in, -1: none
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
      for (int i = 0; i < a.keep && n < K; ++i) {
        if (c.score[i] == -INFINITY) break;
        bool eos = false;
        for (int k = 0; k < s.eos_count; ++k) eos |= c.token[i] == s.eos[k];
        if (!eos) {
          c.pick[n++] = i;
        } else if (i < K) {
          const float x = c.score[i] / len;
          const int w = worst();
          if (c.pool_step[w] < 0 || x > c.pool_score[w]) {
            c.pool_score[w] = x;
            c.pool_step[w] = t;
            c.pool_pick[w] = i;
          }
        }
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
  const int n = c.done ? 0 : c.beams, pad = s.eos_count > 0 ? s.eos[0] : 0;
  const bool on = tid < n;                                // (a row that does not go on stays where it is)
  const int pick = on ? c.pick[tid] : 0, token = on ? c.token[pick] : pad, from = on ? c.beam[pick] : tid;
  const long long h = ((long long)t * gridDim.x + r) * K + tid;
  if (c.done != 1) s.scores[at + tid] = on ? c.score[pick] : -INFINITY;
  s.tokens[at + tid] = token;
  s.parents[at + tid] = r * K + from;
  s.history_token[h] = token;
  s.history_parent[h] = from;
  const int in = c.pool_pick[tid];
  if (in >= 0) {
    s.pool_score[at + tid] = c.pool_score[tid];
    s.pool_step[at + tid] = t;
    s.pool_parent[at + tid] = c.beam[in];
    s.pool_token[at + tid] = c.token[in];
  }
  if (tid == 0 && c.done == 2) s.done[r] = 1;
}

// The heads of the lists while the bound is looked for, then the candidates above it.
struct JoinShared {
  double lse[MAX_BEAMS];
  float base[MAX_BEAMS];
  unsigned long long top_s[JOIN_THREADS], list_s[JOIN_LIST];      // the first words once more, to be counted
  Best list[JOIN_LISTS > JOIN_LIST ? JOIN_LISTS : JOIN_LIST];
  Best top[JOIN_THREADS];
  short id[JOIN_LISTS];
  Best bound;
  int heads, count;
  Chosen out;
};

__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const JoinArgs a) {
  extern __shared__ unsigned long long s_raw[];
  JoinShared& sh = *reinterpret_cast<JoinShared*>(s_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.x, K = a.beams, keep = a.keep;
  if (tid == 0) {
    sh.heads = sh.count = 0;
    sh.bound = Best{1, 0, 0xffffffffu};                    // everything that is a candidate
  }
  for (int i = tid; i < keep; i += JOIN_THREADS) {
    sh.out.score[i] = -INFINITY;
    sh.out.beam[i] = sh.out.token[i] = 0;
  }
  pdl_wait();
  pdl_trigger();
  const int lists = K * a.slices;
  const unsigned long long* cand = a.cand + (long long)r * lists * keep;
  // the first list's head of this thread is on its way while the normalisers are made
  const unsigned long long first = tid < lists ? cand[(long long)tid * keep] : 0ull;
  // normalisers: NaN where the row has no candidates
  for (int b = warp; b < K; b += JOIN_THREADS / 32) {
    const Part* p = a.part + ((long long)r * K + b) * a.slices;
    constexpr int HELD = 3;                                // of a lane; more slices are looked up again
    const float base = a.scores[(long long)r * K + b];
    Part x[HELD];
    float m = -INFINITY;
    bool bad = !(fabsf(base) < INFINITY);                  // (a beam that is not there)
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      x[i].max = -INFINITY;
      x[i].sum = 0.0;
      if (lane + 32 * i < a.slices) x[i] = p[lane + 32 * i];
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      bad |= !(x[i].max < INFINITY);
      m = fmaxf(m, x[i].max);
    }
    for (int i = lane + 32 * HELD; i < a.slices; i += 32) {
      bad |= !(p[i].max < INFINITY);
      m = fmaxf(m, p[i].max);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    bad = __any_sync(0xffffffffu, bad) || m == -INFINITY;
    double sum = 0.0;
    if (!bad) {
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        if (x[i].max > -INFINITY) sum += x[i].sum * exp((double)x[i].max - (double)m);
      for (int i = lane + 32 * HELD; i < a.slices; i += 32)
        if (p[i].max > -INFINITY) sum += p[i].sum * exp((double)p[i].max - (double)m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      sh.lse[b] = bad ? (double)NAN : (double)m + log(sum);
      sh.base[b] = base;
    }
  }
  __syncthreads();
  // a candidate; s = 0 if it is none
  auto made = [&](unsigned long long k, int b) -> Best {
    const double score = (double)sh.base[b] + ((double)value32((uint32_t)(k >> 32)) - sh.lse[b]);
    const bool on = k != 0 && score > -INFINITY && score < INFINITY;              // (false for NaN)
    return Best{on ? order64(score) : 0ull, k, (uint32_t)b};
  };
  auto entry = [&](int list, int i) -> Best { return made(i < keep ? cand[(long long)list * keep + i] : 0ull, list / a.slices); };
  // the heads of all lists that have any
  Best mine{0, 0, 0};
  for (int l = tid; l < lists; l += JOIN_THREADS) {
    const Best e = l == tid ? made(first, l / a.slices) : entry(l, 0);
    if (e.s == 0) continue;
    if (before(e, mine)) mine = e;
    const int at = atomicAdd(&sh.heads, 1);
    if (at < JOIN_LISTS) {
      sh.list[at] = e;
      sh.id[at] = (short)min(l, 32767);                    // (not read if there are more lists than fit)
    }
  }
  __syncthreads();
  const int heads = sh.heads;
  const bool held = heads <= JOIN_LISTS && lists <= 32767;
  // The bound.  d entries of a list are at least as good as its d-th, so of the lists' d-th entries (or of the best of groups of lists) the
  // ceil(keep / d)-th largest has ``keep`` candidates that are not behind it.
  int values = JOIN_THREADS, nth = keep;
  if (held) {
    const int d = heads == 0 ? 1 : (keep + heads - 1) / heads;
    nth = (keep + d - 1) / d;
    const int groups = min(heads, max(64, min(2 * nth, JOIN_GROUPS)));
    values = groups;
    mine = Best{0, 0, 0};
    if (tid < groups)
      for (int i = tid; i < heads; i += groups) {
        const Best e = d == 1 ? sh.list[i] : entry(sh.id[i], d - 1);
        if (before(e, mine)) mine = e;
      }
  }
  sh.top[tid] = mine;
  sh.top_s[tid] = mine.s;
  __syncthreads();
  // A value's place is counted by as many threads as there are for it (a power of two, neighbours).
  {
    int share = 1;
    while (2 * share * values <= JOIN_THREADS && share < 32) share *= 2;
    const int v = tid / share, sub = tid % share;
    const Best e = v < values ? sh.top[v] : Best{0, 0, 0};
    int above = 0;
    if (e.s != 0)
#pragma unroll 4
      for (int i = sub; i < values; i += share) {
        const unsigned long long s = sh.top_s[i];
        above += s > e.s;
        if (s == e.s) above += before(sh.top[i], e);       // (itself, seldom another)
      }
    for (int o = 1; o < share; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
    if (sub == 0 && e.s != 0 && above == nth - 1) sh.bound = e;
  }
  __syncthreads();
  const Best bound = sh.bound;
  // What is not behind it.  (Heads and candidates share their place, so the heads are looked at again first.)
  constexpr int OWN = (JOIN_LISTS + JOIN_THREADS - 1) / JOIN_THREADS, DEEP = 4;
  int go[OWN];
#pragma unroll
  for (int k = 0; k < OWN; ++k) {
    const int i = k * JOIN_THREADS + tid;
    go[k] = held && i < heads && !before(bound, sh.list[i]) ? sh.id[i] : -1;
  }
  __syncthreads();
  auto walk = [&](int l) {
    const int b = l / a.slices;
    for (int i0 = 0; i0 < keep; i0 += DEEP) {
      unsigned long long k[DEEP];
#pragma unroll
      for (int i = 0; i < DEEP; ++i) k[i] = i0 + i < keep ? cand[(long long)l * keep + i0 + i] : 0ull;
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        const Best e = made(k[i], b);
        if (e.s == 0 || before(bound, e)) return;          // sorted: so is the rest
        const int at = atomicAdd(&sh.count, 1);
        if (at < JOIN_LIST) {
          sh.list[at] = e;
          sh.list_s[at] = e.s;
        }
      }
    }
  };
  if (held) {
#pragma unroll
    for (int k = 0; k < OWN; ++k)
      if (go[k] >= 0) walk(go[k]);
  } else {
    for (int l = tid; l < lists; l += JOIN_THREADS) walk(l);
  }
  __syncthreads();
  const int n = sh.count;
  if (n <= JOIN_LIST) {
    int share = 1;                                         // threads for one candidate
    while (2 * share * n <= JOIN_THREADS && share < 32) share *= 2;
    for (int i0 = 0; i0 < n; i0 += JOIN_THREADS / share) {
      const int i = i0 + tid / share, sub = tid % share;
      const Best e = i < n ? sh.list[i] : Best{0, 0, 0};
      int rank = 0;
#pragma unroll 4
      for (int k = sub; k < n; k += share) {
        const unsigned long long s = sh.list_s[k];
        rank += s > e.s;
        if (s == e.s) rank += before(sh.list[k], e);
      }
      for (int o = 1; o < share; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
      if (sub == 0 && i < n && rank < keep) {
        sh.out.score[rank] = (float)value64(e.s);
        sh.out.beam[rank] = (int)e.beam;
        sh.out.token[rank] = (int)~(uint32_t)e.key;
      }
    }
  } else {
    // Many lists share their best (rows that are alike, say): the best of all threads' next entries, ``keep`` times.  Behind the last one
    // taken a list goes on with its first entry that is not before it.
    Best last{~0ull, 0, 0};
    for (int c = 0; c < keep; ++c) {
      Best next{0, 0, 0};
      for (int l = tid; l < lists; l += JOIN_THREADS)
        for (int i = 0; i < keep; ++i) {
          const Best e = entry(l, i);
          if (e.s == 0) break;
          if (!before(last, e)) continue;                  // taken
          if (before(e, next)) next = e;
          break;
        }
      __syncthreads();
      sh.top[tid] = next;
      __syncthreads();
      for (int o = JOIN_THREADS / 2; o > 0; o >>= 1) {
        if (tid < o && before(sh.top[tid + o], sh.top[tid])) sh.top[tid] = sh.top[tid + o];
        __syncthreads();
      }
      last = sh.top[0];
      if (last.s == 0) break;
      if (tid == 0) {
        sh.out.score[c] = (float)value64(last.s);
        sh.out.beam[c] = (int)last.beam;
        sh.out.token[c] = (int)~(uint32_t)last.key;
      }
    }
  }
  __syncthreads();
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

// Values per thread of the first kernel: 8 where slices of 32 values would leave SMs without one (1 x 4 beams of 151936 tokens).
static int slice_of(long long rows, int V) {
  const long long slices = ((long long)V + THREADS * 32 - 1) / (THREADS * 32);
  return rows * slices >= num_sms() ? 32 : 8;
}
static int slices_of(int E, int V) { return (V + THREADS * E - 1) / (THREADS * E); }

template <typename T, int E>
static int launch_pick(PickArgs a, int rows, cudaStream_t st) {
  // Groups by how many values have to pass: fewer groups are sooner counted, as long as there are several times as many.  The room is for
  // what the exact bound lets pass, and four times as many where that is little.
  a.share = a.keep <= 32 ? 4 : a.keep <= 64 ? 2 : 1;
  a.second = a.keep > 16 && a.keep <= 64;
  a.room = a.keep * E * (a.keep <= 16 ? 4 : 1);
  SNU1_CUDA_CHECK(launch_pdl(pick_kernel<T, E>, dim3(a.slices, rows), dim3(THREADS), a.room * 8, st, a));
  return kHostOk;
}

}  // namespace beam
}  // namespace snu1

using namespace snu1;

SNU1_API int snu1_beam_state_bytes() { return (int)sizeof(beam::State); }

// Bytes of scratch for ``rows`` rows of ``V`` logits of which ``keep`` are kept.
SNU1_API long long snu1_beam_scratch_bytes(int rows, int V, int keep) {
  const long long slices = beam::slices_of(beam::slice_of(rows, V), V);
  return rows * slices * ((long long)sizeof(beam::Part) + 8ll * keep);
}

// logits [requests * beams][V] (fp32, or bf16 with is_bf16), rows ld elements apart; scores [requests][beams] fp32.  Without ``state`` the best
// ``keep`` of every request go to out_*; with it (a beam::State) they become the search's next step.
SNU1_API int snu1_beam_step(const void* logits, long long ld, int is_bf16, int V, const void* scores, int requests, int beams, int keep,
                            void* scratch, void* out_scores, void* out_beams, void* out_tokens, const void* state, void* stream) {
  using namespace beam;
  const long long rows = (long long)requests * beams;
  if (requests <= 0 || beams <= 0 || beams > MAX_BEAMS || rows > 65535 || V <= 0 || V > (1 << 30) || keep <= 0 || keep > MAX_KEEP ||
      keep > (long long)beams * V || ld < V || ((reinterpret_cast<uintptr_t>(scratch) & 15) != 0)) {
    set_last_error("beam_step: %d requests of %d beams (at most %d), %d tokens, %d kept (at most %d)", requests, beams, MAX_BEAMS, V, keep,
                   MAX_KEEP);
    return kHostBadArg;
  }
  cudaStream_t st = (cudaStream_t)stream;
  const int E = slice_of(rows, V);
  PickArgs a;
  a.logits = logits;
  a.ld = ld;
  a.V = V;
  a.keep = keep;
  a.slices = slices_of(E, V);
  a.part = (Part*)scratch;
  a.cand = (unsigned long long*)(a.part + rows * a.slices);
  int rc = is_bf16 ? (E == 32 ? launch_pick<__nv_bfloat16, 32>(a, (int)rows, st) : launch_pick<__nv_bfloat16, 8>(a, (int)rows, st))
                   : (E == 32 ? launch_pick<float, 32>(a, (int)rows, st) : launch_pick<float, 8>(a, (int)rows, st));
  if (rc != kHostOk) return rc;
  JoinArgs j;
  memset(&j, 0, sizeof(j));
  j.part = a.part;
  j.cand = a.cand;
  j.scores = (const float*)scores;
  j.out_scores = (float*)out_scores;
  j.out_beams = (int*)out_beams;
  j.out_tokens = (int*)out_tokens;
  j.beams = beams;
  j.keep = keep;
  j.slices = a.slices;
  j.status = device_status_word();
  if (state != nullptr) {
    j.has_state = 1;
    memcpy(&j.st, state, sizeof(State));
  }
  int dev = 0;
  SNU1_CUDA_CHECK(cudaGetDevice(&dev));
  static std::once_flag once[64];
  cudaError_t err = cudaSuccess;
  std::call_once(once[dev & 63], [&]() { err = cudaFuncSetAttribute(join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(JoinShared)); });
  SNU1_CUDA_CHECK(err);
  SNU1_CUDA_CHECK(launch_pdl(join_kernel, dim3(requests), dim3(JOIN_THREADS), sizeof(JoinShared), st, j));
  return kHostOk;
}
