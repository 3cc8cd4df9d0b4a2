// Attention of a few new rows per key/value head over a paged cache: decode steps, drafted tokens, and the joining of
// partial results (also those of attn_paged_sm100.cu).
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp(scale q_r k_j - m_r),   j < limit_r
//
// The rows of a (sequence, key/value head) are its new tokens times the query heads of the group, up to 32 per CTA.  What
// bounds it is the stream of keys and values, so the work is split over keys: a work item is one part of a sequence, the
// parts are made as equal as they can be over the whole batch (ops/paged.py), and their unnormalised results (maximum, sum,
// weighted values, fp32) are joined in a fixed order.  Where every sequence can have as many parts as the longest, up to
// eight, and all CTAs still run at once, the parts of a sequence are a cluster and meet in distributed shared memory: a
// small batch, where latency counts.  Otherwise they meet in scratch, see last_part and paged_join_kernel.
//
// Pages come whole through TMA (keys and values of one head in one box), several stages ahead.  Four warps compute with
// mma.sync m16n8k16, keys (then the width of a head) on the 16-side and rows on the 8-side: S^T = K q^T,
// o^T = V^T p^T.  So a step of a group of 4 or 8 heads fills the product, and what a warp has read and widened of the cache
// serves all rows.  At 1 - 2 products per KB of cache the legacy tensor path is far from its limit.
//
// e4m3 codes are widened to fp16, which is exact, two per instruction.  For that the queries go to fp16 as well, each row
// times the power of two that brings its largest value to [2^13, 2^14): values down to 2^-27 of the largest keep all their
// bits, and what smaller ones lose is below the rounding of the fp32 sum.  The scale of a key goes into its score.  The
// scale of a value goes into its probability, in the exponent: p' = exp2(s + log2(scale) - m') with a maximum of its own,
// so that the fp16 probabilities of the product are relative to the largest p' whatever sizes the values have (the largest
// is brought to 2^7, so that one is only lost below 2^-32 of it; rounding 2^-11 each).  The sum of the probabilities is taken in
// fp32 from p itself.  bf16 caches take a probability as two bf16 numbers (2^-16): one alone, 2^-8, would make the error of
// the result 1.4 times that of its rounding, and the second product costs nothing beside the stream of the cache.
//
// Masked places: scores of keys at or beyond a row's limit are -inf whatever the cache holds, and places that no row of the
// tile may read are cleared in shared memory.  A probability of zero does not hide an infinite or NaN value from the
// matrix product, so in a tile that some row may not read whole, bf16 values that are not finite are cleared too and the
// first key that held one is kept: rows that may read it give NaN, the others are as if it were not there.  (e4m3 codes are
// finite; what is not finite there is the row's scale, and that is only used where the mask allows.)
//
// Measured (32 / 8 heads unless said, of a measured copy bandwidth of 6456 GB/s): e4m3, 48 x 1 token over 32700 keys, 4 heads, 152 us,
// 5.9 TB/s or 0.91; 24 x 1 over up to 4096 keys 23 us, 0.65, of which 6 are a launch's start and end and the join; one
// conversation of 840 bf16 keys 6.3 us in a graph, 7.8 called one by one, latency alone.  8 x 5 tokens over up to 12000 bf16 keys 44 us,
// 0.73.  From 16 rows on instructions count: e4m3 8 x 12000 keys 4 / 16 / 24 / 32 rows 37 / 47 / 63 / 86 us.
#include <math.h>
#include <string.h>

#include <mutex>

#include "host_common.h"
#include "paged.cuh"

namespace snu1 {
namespace paged {

constexpr int FEW_WARPS = 4;                              // warps that compute
constexpr int FEW_LD = 132;                               // a row of 128 values where warps meet, padded

// Up to eight rows: their registers let three CTAs run on an SM, with two stages each instead of three.
// SELF: a fifth warp asks for pages, except with 24 rows per warp.  Five warps of two CTAs are three in a quarter of the SM,
// 168 registers each; four have 255, which 24 rows need, so there the warp that is the last to be done with a stage asks
// for what goes there next.  (17 to 24 rows, 8 x 12000 keys: e4m3 62 us, as 2 x 2 groups of eight rows 85, each code then
// widened by two warps; bf16 71 and 75.  32 rows as four groups per warp: 152 and 89.  Up to 16 rows without the fifth warp: 1 to 4 % slower.)
template <bool FP8, int NR, int WR>
struct Few {
  static constexpr bool SMALL = NR * WR == 1, SELF = NR == 3;
  static constexpr int THREADS = (FEW_WARPS + !SELF) * 32;
  static constexpr int KT = FP8 ? 128 : 64;               // keys of a stage
  static constexpr int HALVES = FP8 ? 1 : 2;              // boxes of 128 bytes per row
  static constexpr int DATA = KT * 2 * 128 * HALVES;      // keys and values of a stage
  static constexpr int SCALES = FP8 ? KT * 2 * 4 : 0;
  static constexpr int CTAS = SMALL ? 3 : 2;
  static constexpr int STAGES = SMALL ? 2 : 3;
  static constexpr int RING = STAGES * (DATA + SCALES);
  static constexpr int SMEM = RING + 1024;
};

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// transposes an 8x8 matrix of 16-bit elements held as a fragment
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool HALF>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the two codes in the low or the high half of ``w`` as fp16
__device__ __forceinline__ uint32_t widen_lo(uint32_t w) {
  uint32_t r;
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %1;\ncvt.rn.f16x2.e4m3x2 %0, l;\n}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t widen_hi(uint32_t w) {
  uint32_t r;
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %1;\ncvt.rn.f16x2.e4m3x2 %0, h;\n}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ float fast_log2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct FewArgs {
  const __nv_bfloat16* q;
  __nv_bfloat16* o;
  long long ldq, ldo;
  float* part;        // [partial rows][heads][128]
  float2* part_ml;    // [partial rows][heads] maximum (log2 units), sum
  unsigned long long* flags;   // [parts of few rows][heads], see last_part
  unsigned long long word;
  int pages, heads;   // of the cache
  float scale_log2;
  int* status;
  int beside;         // the launch in front is that of the chunks: run beside it
  int cluster;        // parts of every sequence, which are a cluster; 1: parts meet in scratch
};

// Up to so many rows the parts join themselves, more are joined by a launch of their own (paged_join_kernel, which has as many
// warps as rows and not four): 24 x 1 token, 4 rows each, 27.7 -> 26.6 us, one conversation 12.2 -> 10.4; 8 x 5 tokens, 20 rows
// each, 44.5 -> 47.9.
constexpr int JOIN_ROWS = 8;

// Joins ``parts`` results of a row, ``step`` apart from ``at`` on; a whole warp, four values per lane.
__device__ __forceinline__ void join_row(const FewArgs& a, long long at, long long step, int parts, __nv_bfloat16* out) {
  const int lane = threadIdx.x & 31;
  float mt = -INFINITY;
  for (int s = lane; s < parts; s += 32) mt = fmaxf(mt, __ldcg(&a.part_ml[at + s * step].x));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  float lt = 0.f;
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const float2 ml = __ldcg(&a.part_ml[at + s * step]);
    const float4 y = __ldcg(reinterpret_cast<const float4*>(a.part + (at + s * step) * HEAD) + lane);
    const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - mt);
    x.x += f * y.x;
    x.y += f * y.y;
    x.z += f * y.z;
    x.w += f * y.w;
    lt += ml.x == -INFINITY ? 0.f : f * ml.y;
  }
  const float inv = lt == 0.f ? 0.f : 1.f / lt;                  // a row without keys gives zeros
  uint2 u;
  u.x = pack_bf16x2(x.x * inv, x.y * inv);
  u.y = pack_bf16x2(x.z * inv, x.w * inv);
  *reinterpret_cast<uint2*>(out + lane * 4) = u;
}

// The same with 16 lanes per row, eight values each, and four parts on their way at a time.
__device__ __forceinline__ void join_eight(const FewArgs& a, long long at, long long step, int parts, __nv_bfloat16* out) {
  constexpr int U = 4;
  const int c = threadIdx.x & 15;
  float x[8], lt = 0.f, mt = -INFINITY;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  for (int s0 = 0; s0 < parts; s0 += U) {
    float2 ml[U];
    float4 y[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long r = at + min(s0 + u, parts - 1) * step;
      ml[u] = __ldcg(&a.part_ml[r]);
      y[u][0] = __ldcg(reinterpret_cast<const float4*>(a.part + r * HEAD) + 2 * c);
      y[u][1] = __ldcg(reinterpret_cast<const float4*>(a.part + r * HEAD) + 2 * c + 1);
    }
    float mn = mt;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u < parts) mn = fmaxf(mn, ml[u].x);
    const float old = mt == -INFINITY ? 0.f : fast_exp2(mt - mn);
    mt = mn;
    lt *= old;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= old;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u >= parts || ml[u].x == -INFINITY) continue;
      const float f = fast_exp2(ml[u].x - mt);
      lt += f * ml[u].y;
      x[0] += f * y[u][0].x;
      x[1] += f * y[u][0].y;
      x[2] += f * y[u][0].z;
      x[3] += f * y[u][0].w;
      x[4] += f * y[u][1].x;
      x[5] += f * y[u][1].y;
      x[6] += f * y[u][1].z;
      x[7] += f * y[u][1].w;
    }
  }
  const float inv = lt == 0.f ? 0.f : 1.f / lt;                  // a row without keys gives zeros
  *reinterpret_cast<uint4*>(out + c * 8) = make_uint4(pack_bf16x2(x[0] * inv, x[1] * inv), pack_bf16x2(x[2] * inv, x[3] * inv),
                                                      pack_bf16x2(x[4] * inv, x[5] * inv), pack_bf16x2(x[6] * inv, x[7] * inv));
}

// Whether this CTA has to join the parts that it is one of; all its threads call it, after their last store of a result.
// A part that is done sets its flag and then looks at all flags: the one that sets its flag last sees the others (stores and
// loads on both sides of a fence.sc), others may see them too and join as well, to the same bits.  Scratch starts with
// whatever was there, so a flag is set to a word of this call (64 random bits), and is cleared again by those who joined:
// the same launch replayed from a graph finds no flag of its last run.
__device__ __forceinline__ bool last_part(unsigned long long* flags, int part, int parts, int step, unsigned long long word, int* s_vote,
                                          int threads) {
  named_bar_sync(1, threads);
  if (threadIdx.x < 32) {
    __threadfence();                                             // of all stores before the barrier
    if (threadIdx.x == 0) *reinterpret_cast<volatile unsigned long long*>(flags + (long long)part * step) = word;
    __threadfence();
    __syncwarp();
    bool all = true;
    for (int s = threadIdx.x; s < parts; s += 32) {
      unsigned long long f;
      asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(f) : "l"(flags + (long long)s * step) : "memory");
      all &= s == part || f == word;
    }
    all = __all_sync(0xffffffffu, all);
    if (threadIdx.x == 0) *s_vote = all;
  }
  named_bar_sync(1, threads);
  return *s_vote != 0;
}

// NR: groups of eight rows that a warp computes.  WR: sets of warps with other rows; the warps of a set take other keys.  TAIL: keys from the
// sequence's ``skip`` on, results always to scratch (attn_prefix_sm100.cu reads the keys before).
template <bool FP8, int NR, int WR, bool TAIL>
__global__ void __launch_bounds__(Few<FP8, NR, WR>::THREADS, Few<FP8, NR, WR>::CTAS)
    paged_few_kernel(const __grid_constant__ CUtensorMap tm_kv, const __grid_constant__ CUtensorMap tm_scale, const Plan p,
                     const FewArgs a) {
  using F = Few<FP8, NR, WR>;
  constexpr int KT = F::KT, WK = FEW_WARPS / WR, M = 8 * NR * WR;
  constexpr bool JOIN = M <= JOIN_ROWS && !TAIL;
  constexpr int BLOCKS = KT / 16 / WK, NB = BLOCKS < 2 ? BLOCKS : 2;     // blocks of 16 keys of a warp, and how many at a time
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* s_scales = reinterpret_cast<float*>(smem + F::STAGES * F::DATA);   // [stage][page box][keys, values][box rows]
  __shared__ uint64_t full[F::STAGES], empty[F::STAGES];
  __shared__ int s_done[F::STAGES];                              // SELF: warps that are done with a stage, all its tiles so far
  __shared__ int abort_word, s_poison, s_vote;
  __shared__ float s_m[FEW_WARPS][8 * NR], s_l[FEW_WARPS][8 * NR];
  __shared__ float s_rs[M];                                      // a row's score scale, log2 units
  // in the ring, behind where warps meet at the end: this CTA's results, read by its cluster
  float* s_part = reinterpret_cast<float*>(smem) + FEW_WARPS * 8 * NR * FEW_LD;      // [rows][128]
  float2* s_part_ml = reinterpret_cast<float2*>(s_part + M * HEAD);
  static_assert(FEW_WARPS * 8 * NR * FEW_LD * 4 + M * (HEAD * 4 + 8) <= F::SMEM - 1024, "results fit the ring");
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_kv);
    if (FP8) tma_prefetch_desc(&tm_scale);
    for (int i = 0; i < F::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], FEW_WARPS);
      s_done[i] = 0;
    }
    abort_word = 0;
    s_poison = 0x7fffffff;
    mbar_fence_init();
  }
  __syncthreads();
  // what the plan's host side has set, before the wait: no launch in front writes it
  const int4 item = (TAIL ? p.tail : p.few)[blockIdx.x];
  const int b = item.x, row0 = item.y, part = item.z & 0xffff, parts = item.z >> 16;
  const int head = blockIdx.y, G = p.group;
  const int shared = TAIL ? p.skip[b] : 0;
  const int q0 = p.q_start[b], q_len = p.q_start[b + 1] - q0;
  // Chunks in front (attn_paged_sm100.cu) have waited for all work before them when this kernel may start, and nothing that
  // they write is read here: it only has to end after them.
  if (!a.beside) pdl_wait();
  pdl_trigger();

  if (threadIdx.x == 0) report_grown(p, b, a.status);
  const int kv_len = seq_len(p, b);
  const int skip = TAIL ? still_shared(p, b, kv_len, shared) / KT : 0;         // tiles
  const int rows = min(M, q_len * G - row0);
  // the furthest key that a row of this tile may read, and the nearest limit
  int max_lim = 0, min_lim = kv_len;
  {
    const int t0 = row0 / G, t1 = (row0 + rows - 1) / G;
    for (int t = t0 + lane; t <= t1; t += 32) {
      const int l = row_limit(p, q0, q_len, kv_len, t);
      max_lim = max(max_lim, l);
      min_lim = min(min_lim, l);
    }
    max_lim = __reduce_max_sync(0xffffffffu, max_lim);
    min_lim = __reduce_min_sync(0xffffffffu, min_lim);
  }
  const int tiles = max(0, (max_lim + KT - 1) / KT - skip);
  const int j0 = skip + (int)((long long)tiles * part / parts), j1 = skip + (int)((long long)tiles * (part + 1) / parts);
  const int page_log = __ffs(p.page) - 1;
  const int bx_log = min(page_log, KT == 128 ? 7 : 6), bx = 1 << bx_log;      // rows of a box
  const int box_bytes = 2 * 128 << bx_log;

  // a lane per box of the stage
  const int boxes = KT >> bx_log;
  const int* table = p.table + (long long)b * p.width;
  auto page_of = [&](int j) -> int {
    const int k = j * KT + (lane << bx_log);
    return j < j1 && lane < boxes && k < max_lim ? table[k >> page_log] : 0;
  };
  auto ask = [&](int j, int s, int pg) {               // (a whole warp)
    const int live = min(boxes, (max_lim - j * KT + bx - 1) >> bx_log);
    if (lane == 0) mbar_expect_tx(&full[s], live * (box_bytes * F::HALVES + (FP8 ? bx * 8 : 0)));
    __syncwarp();
    if (lane < live) {
      if (pg < 0 || pg >= a.pages) report_status(a.status, kBadPage, 10);     // reads as zeros
      const int y = (j * KT + (lane << bx_log)) & (p.page - 1);
#pragma unroll
      for (int h = 0; h < F::HALVES; ++h)
        tma_load_5d(smem_u32(smem + s * F::DATA + (lane * F::HALVES + h) * box_bytes), &tm_kv, &full[s], h * 64, y, head, 0, pg);
      if (FP8) tma_load_4d(s_scales + (s * KT + (lane << bx_log)) * 2, &tm_scale, &full[s], y, head, 0, pg);
    }
    __syncwarp();
  };
  if (!F::SELF && warp == FEW_WARPS) {
    int next = page_of(j0);                              // read a stage ahead
    for (int j = j0; j < j1; ++j) {
      const int n = j - j0, s = n % F::STAGES;
      const int pg = next;
      next = page_of(j + 1);
      if (!mbar_wait_warp(&empty[s], ((n / F::STAGES) & 1) ^ 1, abort_flag, a.status, 10)) break;
      ask(j, s, pg);
    }
  } else {
    int first[F::STAGES], next = 0;
    if (F::SELF) {
#pragma unroll
      for (int s = 0; s < F::STAGES; ++s) first[s] = warp == 0 ? page_of(j0 + s) : 0;
      next = page_of(j0 + F::STAGES);                    // of the tile that goes where this one is
    }
    const int wr = warp / WK, wk = warp % WK;
    const int g = lane >> 2, c = lane & 3;
    // Query fragments of eight rows: values 2 c + {0, 1} and 2 c + 8 + {0, 1} of every 16, or for e4m3 4 c + {0 .. 3}: there a
    // thread's four codes of 16 stand side by side.  Rows behind the last are zeros.
    auto fetch_q = [&](int rg, uint32_t (&f)[8][2]) {
      const int row = rg * 8 + g;
      const bool on = row < rows;
      const __nv_bfloat16* qp = a.q + (long long)(q0 + (row0 + row) / G) * a.ldq + (long long)(head * G + (row0 + row) % G) * HEAD;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f[k][0] = f[k][1] = 0u;
        if (on) {
          if (FP8) {
            const uint2 u = *reinterpret_cast<const uint2*>(qp + k * 16 + c * 4);
            f[k][0] = u.x;
            f[k][1] = u.y;
          } else {
            f[k][0] = *reinterpret_cast<const uint32_t*>(qp + k * 16 + c * 2);
            f[k][1] = *reinterpret_cast<const uint32_t*>(qp + k * 16 + c * 2 + 8);
          }
        }
      }
    };
    auto widen_q = [&](int rg, uint32_t (&f)[8][2]) {
      float rs = a.scale_log2;
      if (FP8) {
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) top = max(top, max((f[k][i] << 16) & 0x7fffffffu, f[k][i] & 0x7fff0000u));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = (int)(top >> 23) - 127;                    // of the largest value; zero and what is not finite: as it is
        const int up = top == 0 || e == 128 ? 0 : min(13 - e, 120);
        const float f2 = __int_as_float((127 + up) << 23);
        rs *= __int_as_float((127 - up) << 23);
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            f[k][i] = pack_f16x2(__uint_as_float(f[k][i] << 16) * f2, __uint_as_float(f[k][i] & 0xffff0000u) * f2);
      }
      if (c == 0) s_rs[rg * 8 + g] = rs;
    };
    uint32_t qf[NR][8][2];
#pragma unroll
    for (int i = 0; i < NR; ++i) fetch_q(wr * NR + i, qf[i]);
    if (F::SELF && warp == 0) {
#pragma unroll
      for (int s = 0; s < F::STAGES; ++s)
        if (j0 + s < j1) ask(j0 + s, s, first[s]);
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) widen_q(wr * NR + i, qf[i]);
    named_bar_sync(1, FEW_WARPS * 32);
    // this thread's rows of a group of eight: 2 c and 2 c + 1
    float rs[NR][2];
    int lim[NR][2];
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = (wr * NR + i) * 8 + 2 * c + e;
        rs[i][e] = s_rs[row];
        lim[i][e] = row < rows ? row_limit(p, q0, q_len, kv_len, (row0 + row) / G) : 0;
      }
    float acc[NR][8][4];                   // o^T: 16 values x 8 rows
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][d][e] = 0.f;
    // running maxima of the scores (for the sums l) and of scores + log2 of the values' scales (for acc; relative to m: beside a large
    // score a small logarithm would be rounded away, and the value's scale with it); bf16: the same
    float m[NR][2], mv[NR][2], l[NR][2];
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[i][e] = mv[i][e] = -INFINITY;
        l[i][e] = 0.f;
      }
    bool ok = true;
    const int krow = (lane & 7) + ((lane >> 3) & 1) * 8, vrow = (lane & 7) + (lane >> 4) * 8;
    for (int j = j0; j < j1; ++j) {
      const int n = j - j0, s = n % F::STAGES, k0 = j * KT;
      const int pg = next;
      if (F::SELF) next = page_of(j + 1 + F::STAGES);
      ok &= mbar_wait(&full[s], (n / F::STAGES) & 1, abort_flag, a.status, 10);
      const uint32_t data = smem_u32(smem + s * F::DATA);
      const bool partial = k0 + KT > min_lim;
      if (partial && (!FP8 || k0 + KT > max_lim)) {
        // values that no row may read, and bf16 values that are not finite
        for (int i = threadIdx.x; i < KT * 8 * F::HALVES; i += FEW_WARPS * 32) {
          const int key = FP8 ? i >> 3 : i >> 4, ch = FP8 ? i & 7 : i & 15;
          uint4* at = reinterpret_cast<uint4*>(smem + s * F::DATA + ((key >> bx_log) * F::HALVES + (ch >> 3)) * box_bytes + (bx << 7) +
                                               swz128_offset(key & (bx - 1), ch & 7));
          if (k0 + key >= max_lim) {
            *at = make_uint4(0, 0, 0, 0);
          } else if (!FP8) {
            uint4 x = *at;
            uint32_t* w = reinterpret_cast<uint32_t*>(&x);
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool lo = (w[e] & 0x7f80u) == 0x7f80u, hi = (w[e] & 0x7f800000u) == 0x7f800000u;
              bad |= lo || hi;
              w[e] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0xffffu : 0xffffffffu);
            }
            if (bad) {
              *at = x;
              atomicMin(&s_poison, k0 + key);
            }
          }
        }
        fence_proxy_async_smem();          // TMA writes here again
        named_bar_sync(1, FEW_WARPS * 32);
      }
#pragma unroll 1
      for (int u0 = wk * BLOCKS; u0 < (wk + 1) * BLOCKS; u0 += NB) {
        float sv[NR][NB][4];                 // S^T: keys g, g + 8 x rows 2 c, 2 c + 1
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) sv[i][nb][e] = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k += 2) {     // 32 values at a time
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const int key0 = (u0 + nb) * 16;
            const uint32_t kb = data + (key0 >> bx_log) * F::HALVES * box_bytes + ((key0 & (bx - 1)) << 7);
            if (FP8) {
              // matrices: keys 0-7 and 8-15 of a 16-value piece, then of the next piece
              uint32_t r[4];
              ldsm_x4(kb + swz128_offset(krow, k + (lane >> 4)), r);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t w0 = r[2 * h], w1 = r[2 * h + 1];
                const uint32_t f[4] = {widen_lo(w0), widen_lo(w1), widen_hi(w0), widen_hi(w1)};
#pragma unroll
                for (int i = 0; i < NR; ++i) mma_16816<true>(sv[i][nb], f, qf[i][k + h][0], qf[i][k + h][1]);
              }
            } else {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t r[4];
                ldsm_x4(kb + (k >> 2) * box_bytes + swz128_offset(krow, ((k + h) & 3) * 2 + (lane >> 4)), r);
#pragma unroll
                for (int i = 0; i < NR; ++i) mma_16816<false>(sv[i][nb], r, qf[i][k + h][0], qf[i][k + h][1]);
              }
            }
          }
        }
        // scores in log2 units, masked, relative to m; largest of this thread's keys
        float lv[NB][2];                     // log2 of the values' scales
        float mx[NR][2], mxv[NR][2];
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) mx[i][e] = mxv[i][e] = -INFINITY;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int key = (u0 + nb) * 16 + g;
          float ks[2] = {1.f, 1.f};
          lv[nb][0] = lv[nb][1] = 0.f;
          if (FP8) {
            const int key0 = (u0 + nb) * 16;
            const float* sc = s_scales + s * KT * 2 + ((key0 >> bx_log) << (bx_log + 1)) + (key0 & (bx - 1)) + g;
            ks[0] = sc[0];
            ks[1] = sc[8];
            lv[nb][0] = fast_log2(sc[bx]);
            lv[nb][1] = fast_log2(sc[bx + 8]);
          }
#pragma unroll
          for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x = __fmul_rn(sv[i][nb][e], FP8 ? rs[i][e & 1] * ks[e >> 1] : rs[i][e & 1]);      // (never fused with the difference)
              if (partial && k0 + key + (e >> 1) * 8 >= lim[i][e & 1]) x = -INFINITY;
              x -= m[i][e & 1] == -INFINITY ? 0.f : m[i][e & 1];
              sv[i][nb][e] = x;
              mx[i][e & 1] = fmaxf(mx[i][e & 1], x);
              if (FP8) mxv[i][e & 1] = fmaxf(mxv[i][e & 1], x + lv[nb][e >> 1]);
            }
        }
        // A running maximum moves only when it is outgrown by more than 2^8 (see attn_infer_sm100.cu), so most tiles need no
        // reduction over the lanes.
        bool move = false;
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) move |= mx[i][e] > (m[i][e] == -INFINITY ? -INFINITY : 8.f) || (FP8 && mxv[i][e] > mv[i][e] + 8.f);
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) mx[i][e] = fmaxf(mx[i][e], __shfl_xor_sync(0xffffffffu, mx[i][e], o));
              const bool fresh = m[i][e] == -INFINITY;
              // (by the difference itself, not by that of two rounded maxima: the largest score here is 0 then)
              const float by = fresh ? (mx[i][e] == -INFINITY ? 0.f : mx[i][e]) : fmaxf(mx[i][e], 0.f);
              const float f = fresh ? 0.f : fast_exp2(-by);
              m[i][e] = fresh ? mx[i][e] : m[i][e] + by;
              l[i][e] *= f;
              float fv = f;
              mxv[i][e] = -INFINITY;
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  sv[i][nb][2 * h + e] -= by;
                  if (FP8) mxv[i][e] = fmaxf(mxv[i][e], sv[i][nb][2 * h + e] + lv[nb][h]);
                }
              if (FP8) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) mxv[i][e] = fmaxf(mxv[i][e], __shfl_xor_sync(0xffffffffu, mxv[i][e], o));
                const float nv = fmaxf(mv[i][e] - by, mxv[i][e]);
                fv = mv[i][e] == -INFINITY ? 0.f : fast_exp2(mv[i][e] - by - nv);
                mv[i][e] = nv;
              }
#pragma unroll
              for (int d = 0; d < 8; ++d) {
                acc[i][d][e] *= fv;
                acc[i][d][2 + e] *= fv;
              }
            }
        }
        uint32_t pf[NR][NB][2];              // p^T: rows g x keys 2 c + {0, 1}, then + 8
        uint32_t pr[NR][NB][2];              // bf16: what rounding has left
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          float muv[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) muv[e] = FP8 && mv[i][e] != -INFINITY ? mv[i][e] - P_TOP : 0.f;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[e] = fast_exp2(sv[i][nb][e]);
              l[i][e & 1] += x[e];
              // (the logarithm of a masked key's scale may be anything)
              if (FP8) x[e] = partial && sv[i][nb][e] == -INFINITY ? 0.f : fast_exp2(sv[i][nb][e] + lv[nb][e >> 1] - muv[e & 1]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t w = FP8 ? pack_f16x2(x[2 * h], x[2 * h + 1]) : pack_bf16x2(x[2 * h], x[2 * h + 1]);
              pf[i][nb][h] = transpose_8x8(w);
              if (!FP8)
                pr[i][nb][h] = transpose_8x8(pack_bf16x2(x[2 * h] - __uint_as_float(w << 16), x[2 * h + 1] - __uint_as_float(w & 0xffff0000u)));
            }
          }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int key0 = (u0 + nb) * 16;
          const uint32_t vb = data + (key0 >> bx_log) * F::HALVES * box_bytes + ((bx + (key0 & (bx - 1))) << 7);
          if (FP8) {
#pragma unroll
            for (int d = 0; d < 8; d += 2) {
              // matrices: keys 0-7 and 8-15 of a piece, then of the next.  A thread has two values of two keys: the even values of a
              // piece are the upper eight lines of the product, the odd ones the lower.
              uint32_t r[4];
              ldsm_x4_t(vb + swz128_offset(krow, d + (lane >> 4)), r);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t w0 = __byte_perm(r[2 * h], 0, 0x3120), w1 = __byte_perm(r[2 * h + 1], 0, 0x3120);
                const uint32_t f[4] = {widen_lo(w0), widen_hi(w0), widen_lo(w1), widen_hi(w1)};
#pragma unroll
                for (int i = 0; i < NR; ++i) mma_16816<true>(acc[i][d + h], f, pf[i][nb][0], pf[i][nb][1]);
              }
            }
          } else {
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              uint32_t r[4];                 // matrices: two pieces of keys 0-7, two of keys 8-15
              ldsm_x4_t(vb + (d >> 2) * box_bytes + swz128_offset(vrow, (d & 3) * 2 + ((lane >> 3) & 1)), r);
#pragma unroll
              for (int i = 0; i < NR; ++i) {
                mma_16816<false>(acc[i][d], r, pf[i][nb][0], pf[i][nb][1]);
                mma_16816<false>(acc[i][d], r, pr[i][nb][0], pr[i][nb][1]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (!F::SELF) {
        if (lane == 0) mbar_arrive(&empty[s]);
      } else if (j + F::STAGES < j1) {
        int before = 0;
        if (lane == 0)
          asm volatile("atom.acq_rel.cta.shared::cta.add.s32 %0, [%1], 1;" : "=r"(before) : "r"(smem_u32(&s_done[s])) : "memory");
        before = __shfl_sync(0xffffffffu, before, 0);
        if (before % FEW_WARPS == FEW_WARPS - 1) ask(j + F::STAGES, s, pg);
      }
    }
    ok = __all_sync(0xffffffffu, ok);
    // Warps of the same rows meet in the ring: every stage has been read (the barrier), and TMA asks for nothing more.
    named_bar_sync(1, FEW_WARPS * 32);
    float* ring = reinterpret_cast<float*>(smem);                // [warp][8 NR][FEW_LD]
    constexpr int LD = FEW_LD;
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], o);
        if (!FP8 && lim[i][e] > s_poison) l[i][e] = __int_as_float(0x7fffffff);
        if (l[i][e] != l[i][e] && m[i][e] == -INFINITY) m[i][e] = 0.f;       // all NaN: not to be taken for no keys at all
        // acc relative to the scores' maximum
        const float f = !FP8 || mv[i][e] == -INFINITY ? 1.f : exp2f(mv[i][e] - P_TOP);
        const int row = i * 8 + 2 * c + e;
        if (g == 0) {
          s_m[warp][row] = m[i][e];
          s_l[warp][row] = l[i][e];
        }
        float* at = ring + (warp * 8 * NR + row) * LD;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          if (FP8) {
            *reinterpret_cast<float2*>(at + d * 16 + 2 * g) = make_float2(acc[i][d][e] * f, acc[i][d][2 + e] * f);
          } else {
            at[d * 16 + g] = acc[i][d][e];
            at[d * 16 + g + 8] = acc[i][d][2 + e];
          }
        }
      }
    named_bar_sync(1, FEW_WARPS * 32);
    const bool direct = !TAIL && item.w < 0;
    const bool near = !TAIL && a.cluster > 1;
    // a warp finishes one row at a time, four values per lane
    for (int row = warp; row < rows; row += FEW_WARPS) {
      const int w0 = row / (8 * NR) * WK, rr = row % (8 * NR);
      float mt = s_m[w0][rr];
#pragma unroll
      for (int w = 1; w < WK; ++w) mt = fmaxf(mt, s_m[w0 + w][rr]);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      float lt = 0.f;
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const float mw = s_m[w0 + w][rr];
        const float f = mw == -INFINITY ? 0.f : fast_exp2(mw - mt);
        const float4 y = *reinterpret_cast<const float4*>(ring + ((w0 + w) * 8 * NR + rr) * LD + lane * 4);
        x.x += f * y.x;
        x.y += f * y.y;
        x.z += f * y.z;
        x.w += f * y.w;
        lt += mw == -INFINITY ? 0.f : f * s_l[w0 + w][rr];
      }
      if (!ok) continue;
      if (near) {
        *reinterpret_cast<float4*>(s_part + row * HEAD + lane * 4) = x;
        if (lane == 0) s_part_ml[row] = make_float2(mt, lt);
      } else if (direct) {
        const float inv = lt == 0.f ? 0.f : 1.f / lt;            // a row without keys gives zeros
        const int t = (row0 + row) / G;
        uint2 u;
        u.x = pack_bf16x2(x.x * inv, x.y * inv);
        u.y = pack_bf16x2(x.z * inv, x.w * inv);
        *reinterpret_cast<uint2*>(a.o + (long long)(q0 + t) * a.ldo + (long long)(head * G + (row0 + row) % G) * HEAD + lane * 4) = u;
      } else {
        const long long at = (long long)(item.w + row) * a.heads + head;
        *reinterpret_cast<float4*>(a.part + at * HEAD + lane * 4) = x;
        if (lane == 0) a.part_ml[at] = make_float2(mt, lt);
      }
    }
    if (JOIN && !direct) {
      const int first = item.w - part * M;                       // partial rows of part 0
      unsigned long long* flags = a.flags + (long long)(first / M) * a.heads + head;
      if (last_part(flags, part, parts, a.heads, a.word, &s_vote, FEW_WARPS * 32)) {
        const int row = threadIdx.x >> 4;
        if (row < rows && ok)
          join_eight(a, (long long)(first + row) * a.heads + head, (long long)M * a.heads, parts,
                     a.o + (long long)(q0 + (row0 + row) / G) * a.ldo + (long long)(head * G + (row0 + row) % G) * HEAD);
        for (int s = threadIdx.x; s < parts; s += FEW_WARPS * 32) flags[(long long)s * a.heads] = 0;
      }
    }
  }
  if (*abort_flag) {                       // copies may be on their way into this CTA's memory
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) {
    }
  }
  if (!TAIL && a.cluster > 1) {
    __syncwarp();
    cluster_sync_all();
    if (warp < FEW_WARPS) {
      for (int row = part * FEW_WARPS + warp; row < rows; row += parts * FEW_WARPS) {
        const float* ml = reinterpret_cast<const float*>(s_part_ml + row);
        float mt = -INFINITY;
        for (int s = 0; s < parts; ++s) mt = fmaxf(mt, ld_cluster(ml[0], s));
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        float lt = 0.f;
#pragma unroll 4
        for (int s = 0; s < parts; ++s) {
          const float ms = ld_cluster(ml[0], s), ls = ld_cluster(ml[1], s);
          const float4 y = ld_cluster_f4(smem_u32(s_part + row * HEAD + lane * 4), s);
          const float f = ms == -INFINITY ? 0.f : fast_exp2(ms - mt);
          x.x += f * y.x;
          x.y += f * y.y;
          x.z += f * y.z;
          x.w += f * y.w;
          lt += ms == -INFINITY ? 0.f : f * ls;
        }
        const float inv = lt == 0.f ? 0.f : 1.f / lt;            // a row without keys gives zeros
        const int t = (row0 + row) / G;
        uint2 u;
        u.x = pack_bf16x2(x.x * inv, x.y * inv);
        u.y = pack_bf16x2(x.z * inv, x.w * inv);
        *reinterpret_cast<uint2*>(a.o + (long long)(q0 + t) * a.ldo + (long long)(head * G + (row0 + row) % G) * HEAD + lane * 4) = u;
      }
    }
    __syncwarp();
    cluster_sync_all();                    // nobody leaves while its results are read
  }
  if (a.beside) pdl_wait();
}

// Joins the parts of the chunk kernel, and of more than JOIN_ROWS few rows: a block per four rows of a key/value head, a warp per row.
constexpr int JOIN_THREADS = 128;

__global__ void __launch_bounds__(JOIN_THREADS) paged_join_kernel(const Plan p, const FewArgs a) {
  pdl_wait();
  pdl_trigger();
  const int4 e = p.merge[blockIdx.x];
  const int b = e.x, parts = e.z & 0xfff, rows = e.z >> 16, warp = threadIdx.x >> 5, head = blockIdx.y;
  const int q0 = p.q_start[b], row = e.y + warp, G = p.group;
  if (warp >= (e.z >> 12 & 15)) return;
  join_row(a, (long long)(e.w + warp) * a.heads + head, (long long)rows * a.heads, parts,
           a.o + (long long)(q0 + row / G) * a.ldo + (long long)(head * G + row % G) * HEAD);
}

// Joins what rows with shared tokens have of them and of their own: a warp per row and head.
__global__ void __launch_bounds__(JOIN_THREADS) paged_share_join_kernel(const Plan p, const FewArgs a) {
  const int i = blockIdx.x * (JOIN_THREADS / 32) + (threadIdx.x >> 5), head = blockIdx.y, lane = threadIdx.x & 31;
  int4 e[2];
  if (i < p.join_count) {
    e[0] = p.joins[2 * i];
    e[1] = p.joins[2 * i + 1];
  }
  pdl_wait();
  pdl_trigger();
  if (i >= p.join_count) return;
  // a lane has the maximum and the sum of one part, 32 parts at a time; eight parts' values are on their way
  const int shared = e[0].w, all = shared + e[1].y;
  float mt = -INFINITY, lt = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < all; s0 += 32) {
    const int s = s0 + lane;
    const int row = s < shared ? e[0].z + s * e[1].w : e[1].x + (s - shared) * e[1].z;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (s < all) ml = __ldcg(&a.part_ml[(long long)row * a.heads + head]);
    float top = fmaxf(ml.x, mt);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // (-1: the part has nothing.  One that is far below still counts: its NaN is the row's.)
    const float old = mt == -INFINITY ? 0.f : fast_exp2(mt - top), f = ml.x == -INFINITY ? -1.f : fast_exp2(ml.x - top);
    mt = top;
    float l = f < 0.f ? 0.f : f * ml.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    lt = lt * old + l;
    x.x *= old;
    x.y *= old;
    x.z *= old;
    x.w *= old;
    const int here = min(32, all - s0);
    for (int k = 0; k < here; k += 8) {
      float4 y[8];
      float g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int from = __shfl_sync(0xffffffffu, row, min(k + i, here - 1));
        g[i] = __shfl_sync(0xffffffffu, f, k + i & 31);
        y[i] = __ldcg(reinterpret_cast<const float4*>(a.part + ((long long)from * a.heads + head) * HEAD) + lane);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (k + i >= here || g[i] < 0.f) continue;               // (nothing is written where there is nothing)
        x.x += g[i] * y[i].x;
        x.y += g[i] * y[i].y;
        x.z += g[i] * y[i].z;
        x.w += g[i] * y[i].w;
      }
    }
  }
  const float inv = lt == 0.f ? 0.f : 1.f / lt;                  // a row without keys gives zeros
  uint2 u;
  u.x = pack_bf16x2(x.x * inv, x.y * inv);
  u.y = pack_bf16x2(x.z * inv, x.w * inv);
  *reinterpret_cast<uint2*>(a.o + (long long)e[0].x * a.ldo + (long long)(head * p.group + e[0].y) * HEAD + lane * 4) = u;
}

template <bool FP8, int NR, int WR, bool TAIL>
static int launch_few(const Cache& c, const Plan& p, const FewArgs& a, cudaStream_t st) {
  auto kernel = paged_few_kernel<FP8, NR, WR, TAIL>;
  constexpr int SMEM = Few<FP8, NR, WR>::SMEM;
  int dev = 0;
  SNU1_CUDA_CHECK(cudaGetDevice(&dev));
  static std::once_flag once[64];
  cudaError_t err = cudaSuccess;
  std::call_once(once[dev & 63], [&]() {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  });
  SNU1_CUDA_CHECK(err);
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(TAIL ? p.tail_count : p.few_count, c.heads);
  cfg.blockDim = dim3(Few<FP8, NR, WR>::THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = a.cluster > 1 ? 2 : 1;
  SNU1_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, c.kv, c.scale, p, a));
  return kHostOk;
}

template <bool FP8>
static int launch_few(const Cache& c, const Plan& p, const FewArgs& a, cudaStream_t st) {
  switch (p.few_rows) {
    case 8: return launch_few<FP8, 1, 1, false>(c, p, a, st);
    case 16: return launch_few<FP8, 2, 1, false>(c, p, a, st);
    case 24: return launch_few<FP8, 3, 1, false>(c, p, a, st);
    case 32: return launch_few<FP8, 2, 2, false>(c, p, a, st);
    default: set_last_error("paged_attention: no kernel for %d rows", p.few_rows); return kHostBadArg;
  }
}

template <bool FP8>
static int launch_tail(const Cache& c, const Plan& p, const FewArgs& a, cudaStream_t st) {
  switch (p.tail_rows) {
    case 8: return launch_few<FP8, 1, 1, true>(c, p, a, st);
    case 16: return launch_few<FP8, 2, 1, true>(c, p, a, st);
    case 32: return launch_few<FP8, 2, 2, true>(c, p, a, st);
    default: set_last_error("paged_attention: no kernel for tails of %d rows", p.tail_rows); return kHostBadArg;
  }
}

}  // namespace paged
}  // namespace snu1

using namespace snu1;

// o_r = attention of row r over its sequence's first keys, rows [rows][heads of queries][128] bf16, ldq / ldo apart.
// scratch: partial results (partial_rows x heads x (128 values, maximum, sum) in fp32) and a 64-bit flag per part of the few
// rows (few_parts x heads), to a multiple of 128 bytes; then unpack_count fp16 pages of 128 tokens and their factors (a float4
// per page and head).  word: see last_part; another one for every call.
SNU1_API int snu1_paged_attention(const void* cache, const void* plan, const void* q, long long ldq, void* o, long long ldo,
                                  float scale, void* scratch, unsigned long long word, void* stream) {
  using namespace paged;
  Cache c;
  Plan p;
  memcpy(&c, cache, sizeof(c));
  memcpy(&p, plan, sizeof(p));
  if (p.layout != paged::PLAN_LAYOUT) {
    set_last_error("paged: this plan was made for another version of the library");
    return kHostBadArg;
  }
  if (p.rows <= 0) return kHostOk;
  if (p.page != c.page || ldq % 8 || ldo % 8 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(scratch)) & 15) != 0) {
    set_last_error("paged_attention: rows must be 16-byte aligned, and the plan made for this page size");
    return kHostBadArg;
  }
  FewArgs a;
  if (!(scale > 0.f) || isinf(scale)) {
    set_last_error("paged_attention: the scale must be a positive number");
    return kHostBadArg;
  }
  a.q = (const __nv_bfloat16*)q;
  a.o = (__nv_bfloat16*)o;
  a.ldq = ldq;
  a.ldo = ldo;
  a.part = (float*)scratch;
  a.part_ml = (float2*)(a.part + (long long)p.partial_rows * c.heads * HEAD);
  a.flags = (unsigned long long*)(a.part_ml + (long long)p.partial_rows * c.heads);
  a.word = word;
  a.pages = c.pages;
  a.heads = c.heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = device_status_word();
  a.beside = p.chunk_count + p.one_count > 0;
  a.cluster = p.few_cluster;
  cudaStream_t st = (cudaStream_t)stream;
  int rc = kHostOk;
  if (a.beside) {
    void* wide = a.flags + (((long long)(p.partial_rows + p.few_parts) * c.heads + 15) / 16 * 16 - (long long)p.partial_rows * c.heads);
    float4* factors = (float4*)((uint8_t*)wide + 2ll * 128 * HEAD * 2 * p.unpack_count * c.heads);
    if (c.fp8 && p.chunk_count > 0 && (rc = launch_widen(c, p, wide, factors, st)) != kHostOk) return rc;
    if ((rc = launch_chunks(c, p, q, ldq, o, ldo, a.part, a.part_ml, a.scale_log2, wide, factors, st)) != kHostOk) return rc;
  }
  if (p.many_count > 0) {                  // the products of many rows are long: in front of what runs beside
    Plan r = p;
    r.q_start = p.run_start;
    r.kv_len = r.cap = p.run_len;
    r.own_q_start = p.q_start;
    r.own_kv_len = p.kv_len;
    r.own_cap = p.cap;
    (c.fp8 ? r.one : r.chunk) = p.many;
    r.one_count = c.fp8 ? p.many_count : 0;
    r.chunk_count = c.fp8 ? 0 : p.many_count;
    if ((rc = launch_chunks(c, r, q, ldq, o, ldo, a.part, a.part_ml, a.scale_log2, nullptr, nullptr, st)) != kHostOk) return rc;
    a.beside = 1;
  }
  if (p.few_count > 0) {
    if (c.fp8) rc = launch_few<true>(c, p, a, st);
    else rc = launch_few<false>(c, p, a, st);
    if (rc != kHostOk) return rc;
  }
  a.beside = a.beside || p.few_count > 0;
  // Shared tokens first, on the SMs that the plan gives them: a CTA of them fills an SM, tails take what is left.  Both run beside the launch in
  // front, if that is one of this call (see ``beside`` in paged_few_kernel).
  if (p.prefix_count > 0) {
    if ((rc = launch_prefix(c, p, q, ldq, a.part, a.part_ml, a.scale_log2, a.beside, st)) != kHostOk) return rc;
    a.beside = 1;
  }
  if (p.tail_count > 0) {
    a.cluster = 1;
    if ((rc = c.fp8 ? launch_tail<true>(c, p, a, st) : launch_tail<false>(c, p, a, st)) != kHostOk) return rc;
    SNU1_CUDA_CHECK(launch_pdl(paged_share_join_kernel, dim3((p.join_count + JOIN_THREADS / 32 - 1) / (JOIN_THREADS / 32), c.heads),
                               dim3(JOIN_THREADS), 0, st, p, a));
  }
  if (p.merge_count > 0)
    SNU1_CUDA_CHECK(launch_pdl(paged_join_kernel, dim3(p.merge_count, c.heads), dim3(JOIN_THREADS), 0, st, p, a));
  return kHostOk;
}
