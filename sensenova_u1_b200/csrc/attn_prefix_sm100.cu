// Attention of many sequences' few new rows to the tokens that all of them share, over a paged cache: the first part of a row's
// keys, read once for the whole run of sequences.  The rest of the keys is each sequence's own (attn_paged.cu, TAIL); both leave unnormalised results
// (maximum, sum, weighted values, fp32) that paged_share_join_kernel puts together.
//
//   S^T = K q^T,   p = exp2(S^T - m),   o^T = V^T p^T
//
// The rows of a run are its new tokens times the query heads of the group, up to 64 per CTA.  They are the N of both products
// (tcgen05.mma, accumulators in tensor memory), the 128 keys of a tile (the 128 values of a head) the M: eight rows cost an eighth of 64,
// where rows as the M would fill 128 lanes whatever their number.  A thread of the softmax has one key and a column per row, so the
// maximum over keys lies across lanes.  It begins at that of 32 keys and moves only when a probability would be too large (Range), and a vote per
// tile is all that costs.  Sums stay with the threads until the end.
//
// e4m3 codes go to the first product as they are; a query is two e4m3 numbers, each row times a power of two: hi has 4 of the 8 bits
// of bf16, lo the others, 16 times as large, as 64 more columns.  A value of less than 2^-14 of its row's largest loses bits below 2^-22 of it.  A key's
// scale is a number of the thread's.  For the second product four warps widen codes to fp16, which is exact; a value's scale goes into its probability,
// times a power of two per row that keeps the largest product between 2^4 and 2^15 (W_TOP), and what that leaves of fp16's range is 28 bits below
// the largest.  bf16: probabilities are two bf16 numbers, hi and lo as 64 columns each.
//
// What bounds it: with bf16 memory (8 heads, 80000 shared tokens: 8 rows 57 us, 64 rows 62, their bytes alone 50).  With e4m3 8 rows
// read 5 TB/s, and every eight rows more that a warp has take 0.15 us a tile, 1.45 at 64 rows (43 and 62 us, the bytes alone 26): their arithmetic, of which no part
// (exponentials, conversions, products) is the bound by itself.  Short prefixes: the start and the end of a CTA, 8 us together, of
// which the first page look-up, its copy, the first product and the last one follow each other (8 heads, 16000 tokens: 17 us and 25 to 27).
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <math.h>
#include <string.h>

#include <mutex>

#include "host_common.h"
#include "paged.cuh"

namespace snu1 {
namespace paged {

constexpr int PR = PREFIX_ROWS;                 // rows of a CTA
constexpr int PK = 128;                         // keys of a tile

template <bool FP8>
struct Prefix {
  static constexpr int THREADS = FP8 ? 512 : 384;
  static constexpr int K_STAGES = 3, V_STAGES = FP8 ? 3 : 2, W_STAGES = 2, P_STAGES = FP8 ? 2 : 1;
  // Scales of a tile's keys and values.  Those of tile n are read before S(n + 2) is asked for, and the keys of tile n + K_STAGES + 2 come after that.
  static constexpr int C_STAGES = 8;
  static constexpr int TILE = PK * HEAD * (FP8 ? 1 : 2), WIDE = PK * HEAD * 2, Q = 16384, P = FP8 ? PK * PR * 2 : 2 * PK * PR * 2;
  static constexpr int SCALES = FP8 ? C_STAGES * PK * 8 : 0;
  static constexpr int SMEM = Q + (K_STAGES + V_STAGES) * TILE + (FP8 ? W_STAGES * WIDE : 0) + P_STAGES * P + SCALES + 1024;
  static constexpr int COLS = FP8 ? 512 : 256;  // of tensor memory: scores twice, output
  static constexpr int S_COLS = FP8 ? 2 * PR : PR, O_AT = 2 * S_COLS;
};

struct PrefixArgs {
  const __nv_bfloat16* q;
  long long ldq;
  float* part;
  float2* part_ml;
  int pages, heads;
  float scale_log2;
  int beside;
  int* status;
};

__device__ __forceinline__ void tmem_ld_x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void umma_f8_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// whether any of the barrier's threads says so
__device__ __forceinline__ bool named_bar_any(int id, int threads, bool x) {
  uint32_t r;
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbarrier.cta.red.or.pred q, %2, %3, p;\nselp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"((uint32_t)x), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ uint32_t e4m3x2_of(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// four codes as fp16
__device__ __forceinline__ uint2 widen4(uint32_t w) {
  uint2 r;
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}" : "=r"(r.x), "=r"(r.y) : "r"(w));
  return r;
}
__device__ __forceinline__ float log2_of(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The maximum that probabilities are relative to moves when one would pass 2^MOST.  bf16: it begins, and is moved, LEAD above the largest score that has
// been seen, so scores may rise by LEAD + MOST before it moves, and products with values of up to 2^100 still fit fp32 sums (p is at most 2^8, as in
// the kernel for chunks).  What is 2^-100 of the largest probability or less is lost.  e4m3: values' scales have a power of two of their
// own (W_TOP), which bounds the products.
template <bool FP8> struct Range {
  static constexpr float MOST = FP8 ? 60.f : 8.f, LEAD = FP8 ? 0.f : 24.f;
};
// e4m3: exponent of the factor of probabilities times values' scales, whose largest is 2^mv: 2^W_TOP then, as fp16 numbers, and up to 2^15 before it
// moves.  What is 2^-28 of the largest or less is lost.  (2^7 lets it move in one CTA in five of random scores, 5 us each time.)
constexpr float W_TOP = 4.f;
__device__ __forceinline__ int exponent_of(float mv) { return mv == -INFINITY ? 120 : max(-120, min(120, (int)floorf(W_TOP - mv))); }

// What the softmax knows of a row; column n.
struct RowState {
  float m;           // running maximum, log2 units; -inf as long as there is none
  float rs;          // e4m3: the power of two that the scores are multiplied by; NaN: a query that is not finite
};

struct PrefixShared {
  alignas(16) int lim[PR];                       // limits of the rows, by column
  // e4m3: the powers of two of RowState::rs and of ec, as bf16: read eight at a time (registers do not suffice for them)
  alignas(16) uint16_t rs[PR];
  alignas(16) uint16_t vf[PR];
  RowState row[PR];
  float by[PR], f[PR], fo[PR], mv[PR];           // of a move: by how much, factors of the sums and of the output; e4m3: see exponent_of
  int ec[PR];                                    // e4m3: exponent of a row's factor of p times the value's scale
  float red[8][32], sum[8][32];
};

// The largest scores of eight rows over a warp's keys, row i in lane i: log2 units, or relative to the row's maximum plus ``more``.  S: the rows'
// products; lim: their limits, or null.  Every step takes half of the rows across half of the lanes.
template <bool FP8>
__device__ __forceinline__ float row_tops(uint32_t S, const RowState* row, const int* lim, int key, float ks, bool rel, float more) {
  uint32_t h[8], lo[8];
  tmem_ld_x8(S, h);
  if (FP8) tmem_ld_x8(S + PR, lo);
  tmem_ld_wait();
  const int lane = threadIdx.x & 31;
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    y[e] = __uint_as_float(h[e]);
    if (FP8) y[e] = fmaf(__uint_as_float(lo[e]), 0.0625f, y[e]);
    y[e] = __fmul_rn(y[e], FP8 ? __fmul_rn(row[e].rs, ks) : ks);
    if (rel) y[e] -= row[e].m;
    if (lim != nullptr && key >= lim[e]) y[e] = -INFINITY;
    y[e] = y[e] > -INFINITY ? y[e] + more : -INFINITY;           // (NaN counts for nothing)
  }
#pragma unroll
  for (int n = 4; n > 0; n >>= 1)
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float send = lane & 4 * n ? y[i] : y[i + n], keep = lane & 4 * n ? y[i + n] : y[i];
      y[i] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, send, 4 * n));
    }
  y[0] = fmaxf(y[0], __shfl_xor_sync(0xffffffffu, y[0], 2));
  y[0] = fmaxf(y[0], __shfl_xor_sync(0xffffffffu, y[0], 1));
  return __shfl_sync(0xffffffffu, y[0], lane << 2 & 31);         // (lane / 4 was the row)
}

// Moves the maxima of a set of four softmax warps to the largest scores of a tile, and the output with them.  Out of the loop's way.
template <bool FP8>
__device__ __noinline__ void move_maxima(PrefixShared& sh, uint32_t S, uint32_t O, int side, int active, int key, float ks, float lv, bool dirty, bool first) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = warp - 4, c0 = side * 32, col = c0 + lane;
  const bool mine = (w & 3) == 0 && lane < 8 * active;
#pragma unroll 1
  for (int i = 0; i < active; ++i) {
    const int c = c0 + 8 * i;
    const float top = row_tops<FP8>(S + 8 * i, sh.row + c, dirty ? sh.lim + c : nullptr, key, ks, false, 0.f);
    if (lane < 8) sh.red[w][8 * i + lane] = top;
  }
  named_bar_sync(2 + side, 128);
  if (mine) {
    const float m = sh.row[col].m;
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) top = fmaxf(top, sh.red[side * 4 + k][lane]);
    const bool fresh = m == -INFINITY;
    const float now = fmaxf(m, top + Range<FP8>::LEAD);
    sh.by[col] = fresh ? 0.f : now - m;
    sh.f[col] = fresh ? 0.f : fast_exp2(m - now);
    sh.row[col].m = now;
  }
  named_bar_sync(2 + side, 128);
  if (FP8) {
#pragma unroll 1
    for (int i = 0; i < active; ++i) {
      const int c = c0 + 8 * i;
      const float top = row_tops<FP8>(S + 8 * i, sh.row + c, dirty ? sh.lim + c : nullptr, key, ks, true, lv);
      if (lane < 8) sh.red[w][8 * i + lane] = top;
    }
    named_bar_sync(2 + side, 128);
    if (mine) {
      float top = sh.mv[col] - sh.by[col];
#pragma unroll
      for (int k = 0; k < 4; ++k) top = fmaxf(top, sh.red[side * 4 + k][lane]);
      const int ec = exponent_of(top);
      sh.fo[col] = sh.f[col] == 0.f ? 0.f : exp2f((float)(ec - sh.ec[col]) - sh.by[col]);
      sh.mv[col] = top;
      sh.ec[col] = ec;
      sh.vf[col] = (uint16_t)((127 + ec) << 7);
    }
    named_bar_sync(2 + side, 128);
  }
  if (!first) {
#pragma unroll 1
    for (int i = 0; i < active * (FP8 ? 1 : 2); ++i) {
      const int c = c0 + 8 * (FP8 ? i : i >> 1);
      const uint32_t at = O + (FP8 ? 0 : (i & 1) * PR) + c;
      uint32_t o[8];
      tmem_ld_x8(at, o);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * (FP8 ? sh.fo : sh.f)[c + e]);
      tmem_st_x8(at, o);
    }
    tmem_st_wait();
  }
}

template <bool FP8>
__global__ void __launch_bounds__(Prefix<FP8>::THREADS, 1)
    paged_prefix_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v /* e4m3: of the scales */, const __grid_constant__ Plan p,
                        const __grid_constant__ PrefixArgs args) {
  using F = Prefix<FP8>;
  constexpr int KS = F::K_STAGES, VS = F::V_STAGES, WS = F::W_STAGES, PS = F::P_STAGES, CS = F::C_STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;                            // e4m3: [hi 64, lo 64][128]; bf16: [half of the values][64][64]
  uint8_t* sK = sQ + F::Q;
  uint8_t* sV = sK + KS * F::TILE;
  uint8_t* sP = sV + VS * F::TILE;               // [key][64 rows] fp16; bf16: hi, then lo
  uint8_t* sW = sP + PS * F::P;                  // e4m3: widened values, [half][key][64]
  float* sC = reinterpret_cast<float*>(sW + WS * F::WIDE);      // e4m3: [stage][page][keys, values][token]
  __shared__ uint64_t q_ready, k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], w_full[WS], w_empty[WS], s_full[2], s_empty[2], p_full[PS], pv_done[PS], c_full[CS];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word, s_poison;
  __shared__ int s_most, s_least;
  __shared__ PrefixShared sh;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  // what the plan's host side has set, before the wait: no launch in front writes it
  const int4 item = p.prefix[blockIdx.x / args.heads], run = p.runs[item.x];
  const int head = blockIdx.x % args.heads, part = item.z & 0xffff, parts = item.z >> 16, G = p.group;
  const int t0 = run.x, row0 = item.y, rows = min(PR, run.y * G - row0), shared = run.w;
  const int groups = (rows + 7) / 8, sides = groups > 1 ? 2 : 1;      // of eight rows; sets of four softmax warps that have any
  if (tid == 0) {
    mbar_init(&q_ready, 8);
    for (int i = 0; i < KS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < VS; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], FP8 ? 4 : 1);
    }
    for (int i = 0; i < WS; ++i) {
      mbar_init(&w_full[i], 4);
      mbar_init(&w_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 4 * sides);
    }
    for (int i = 0; i < CS; ++i) mbar_init(&c_full[i], 1);
    for (int i = 0; i < PS; ++i) {
      mbar_init(&p_full[i], 4 * sides);
      mbar_init(&pv_done[i], 1);
    }
    abort_word = 0;
    s_poison = 0x7fffffff;
    mbar_fence_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, F::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // (also host-set: where the rows of warp 0's threads are)
  int q_first[2], q_len[2], seq[2];
  if (warp == 0) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = min(lane + 32 * k, rows - 1);
      seq[k] = p.row_seq[t0 + (row0 + r) / G];
      q_first[k] = p.q_start[seq[k]];
      q_len[k] = p.q_start[seq[k] + 1] - q_first[k];
    }
  }
  if (!args.beside) pdl_wait();                  // (see paged_few_kernel)
  pdl_trigger();
  const int* table = p.table + (long long)run.z * p.width;
  const int page = p.page, per = PK / page;      // pages of a tile
  // a tile's keys, values and scales; the whole of warp 0, a lane per page
  auto ask = [&](int n, int pg, int live, int kv) {
    const int s = n % (kv ? VS : KS);
    uint64_t* full = kv ? &v_full[s] : &k_full[s];
    uint8_t* dst = (kv ? sV : sK) + s * F::TILE + lane * page * 128;
    if (lane == 0) {
      mbar_expect_tx(full, live * page * (FP8 ? 128 : 256));
      if (FP8 && kv == 0) mbar_expect_tx(&c_full[n % CS], live * page * 8);
    }
    __syncwarp();
    if (lane < live) {
      if (pg < 0 || pg >= args.pages) report_status(args.status, kBadPage, 10);     // reads as zeros
      if (FP8) {
        if (kv == 0) tma_load_4d(sC + ((n % CS) * PK + lane * page) * 2, &tm_v, &c_full[n % CS], 0, head, 0, pg);
        tma_load_5d(smem_u32(dst), &tm_k, full, 0, 0, head, kv, pg);
      } else {
        tma_load_4d(dst, kv ? &tm_v : &tm_k, full, 0, 0, head, pg);
        tma_load_4d(dst + PK * 128, kv ? &tm_v : &tm_k, full, 64, 0, head, pg);
      }
    }
    __syncwarp();
  };
  if (warp == 0) {
    // column of row r: 8 (r / 8 / 2) + r % 8 of the half that its set of warps has
    const int guess = lane < per ? table[(int)((long long)(shared / PK) * part / parts) * per + lane] : 0;      // if all shared tokens are read
    int most = 0, least = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = lane + 32 * k, col = (r >> 3 & 1) * 32 + (r >> 4) * 8 + (r & 7);
      int lim = 0;
      if (r < rows) {
        const int len = seq_len(p, seq[k]);
        lim = min(still_shared(p, seq[k], len, shared), row_limit(p, q_first[k], q_len[k], len, t0 + (row0 + r) / G - q_first[k]));
        least = min(least, lim);
      }
      most = max(most, lim);
      sh.lim[col] = lim;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    least = __reduce_min_sync(0xffffffffu, least);
    if (lane == 0) {
      s_most = most;
      s_least = least;
    }
    // the first tile is on its way before anybody else is ready
    const int all = (most + PK - 1) / PK, first = (int)((long long)all * part / parts);
    if (first < (int)((long long)all * (part + 1) / parts)) {
      const int live = min(per, (most + page - 1) / page - first * per);
      const int pg = most == shared ? guess : lane < live ? table[first * per + lane] : 0;
      ask(0, pg, live, 0);
      ask(0, pg, live, 1);
    }
  } else if (warp >= 4 && warp < 12) {
    // queries: four threads per row
    const int s = tid - 128, r = s >> 2, c = s & 3, col = (r >> 3 & 1) * 32 + (r >> 4) * 8 + (r & 7), row = row0 + r;
    uint4 u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = make_uint4(0, 0, 0, 0);
    if (r < rows) {
      const uint4* from = reinterpret_cast<const uint4*>(args.q + (long long)(t0 + row / G) * args.ldq + (long long)(head * G + row % G) * HEAD + c * 32);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = from[i];
    }
    float rs = 1.f;
    if (!FP8) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(sQ + (c >> 1) * (PR * 128) + swz128_offset(col, (c & 1) * 4 + i)) = u[i];
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        top = max_u16x2(top, max_u16x2(max_u16x2(u[i].x & 0x7fff7fffu, u[i].y & 0x7fff7fffu), max_u16x2(u[i].z & 0x7fff7fffu, u[i].w & 0x7fff7fffu)));
      }
      top = max_u16x2(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max_u16x2(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = max(top << 16, top & 0xffff0000u);
      const int e = (int)(top >> 23) - 127, up = top == 0 || e == 128 ? 0 : min(7 - e, 120);
      const float f = __int_as_float((127 + up) << 23);
      rs = e == 128 ? __int_as_float(0x7fffffff) : __int_as_float((127 - up) << 23);      // not finite: NaN
      uint32_t hi[8], lo[8];                   // four codes each
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t x2 = i & 2 ? (i & 1 ? u[i >> 2].w : u[i >> 2].z) : (i & 1 ? u[i >> 2].y : u[i >> 2].x);
        const float x = __uint_as_float(x2 << 16) * f, y = __uint_as_float(x2 & 0xffff0000u) * f;
        const uint32_t h = e4m3x2_of(x, y);
        const float2 back = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)h, __NV_E4M3)));
        const uint32_t l = e4m3x2_of((x - back.x) * 16.f, (y - back.y) * 16.f);
        if (i & 1) {
          hi[i >> 1] |= h << 16;
          lo[i >> 1] |= l << 16;
        } else {
          hi[i >> 1] = h;
          lo[i >> 1] = l;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        *reinterpret_cast<uint4*>(sQ + swz128_offset(col, 2 * c + i)) = make_uint4(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
        *reinterpret_cast<uint4*>(sQ + swz128_offset(PR + col, 2 * c + i)) = make_uint4(lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
      }
    }
    if (c == 0) {
      sh.row[col] = RowState{-INFINITY, rs};
      sh.rs[col] = (uint16_t)(__float_as_uint(rs) >> 16);
      sh.ec[col] = 120;
      sh.vf[col] = (127 + 120) << 7;
      sh.mv[col] = -INFINITY;
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&q_ready);
  }
  __syncthreads();
  const int most = s_most, least = s_least;
  const int all = (most + PK - 1) / PK;
  const int j0 = (int)((long long)all * part / parts), n_tiles = (int)((long long)all * (part + 1) / parts) - j0;
  // e4m3: 512 threads start with 128 registers, 256 x 72 + 256 x 184 = 512 x 128; bf16: 384 with 168, 128 x 88 + 256 x 208 = 384 x 168
  if (warp < 4 || warp >= 12) {
    if (FP8) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) {
      // ------------------------------ pages --------------------------------
      const int used = (most + page - 1) / page;
      auto page_of = [&](int n) -> int {
        const int i = (j0 + n) * per + lane;
        return n < n_tiles && lane < per && i < used ? table[i] : 0;
      };
      int pg = page_of(1);
      bool ok = true;
      for (int n = 1; n < n_tiles && ok; ++n) {
        const int next = page_of(n + 1), live = min(per, used - (j0 + n) * per);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int stages = kv ? VS : KS;
          ok = ok && mbar_wait_warp(kv ? &v_empty[n % stages] : &k_empty[n % stages], ((n / stages) & 1) ^ 1, abort_flag, args.status, 1);
          if (ok) ask(n, pg, live, kv);
        }
        pg = next;
      }
    } else if (warp == 1) {
      // ------------------------------ products --------------------------------
      bool ok = mbar_wait(&q_ready, 0, abort_flag, args.status, 3);
      const uint64_t q_desc = make_smem_desc(smem_u32(sQ), 0, 1024), k_desc = make_smem_desc(smem_u32(sK), 0, 1024);
      const uint64_t v_desc = make_smem_desc(smem_u32(FP8 ? sW : sV), PK * 128, 1024), p_desc = make_smem_desc(smem_u32(sP), PK * 128, 1024);
      // (e4m3: bits [7,13) of the descriptor are 0 for e4m3 operands, and for fp16 ones)
      constexpr uint32_t types = 1u << 7 | 1u << 10;
      constexpr uint32_t idesc_s = FP8 ? make_idesc_bf16(128, 2 * PR, false, false) & ~types : make_idesc_bf16(128, PR, false, false);
      constexpr uint32_t idesc_o = FP8 ? make_idesc_bf16(128, PR, true, true) & ~types : make_idesc_bf16(128, 2 * PR, true, true);
      auto issue_s = [&](int n) {
        ok &= mbar_wait(&k_full[n % KS], (n / KS) & 1, abort_flag, args.status, 3);
        ok &= mbar_wait(&s_empty[n & 1], ((n >> 1) & 1) ^ 1, abort_flag, args.status, 2);
        tc_fence_after();
        const uint64_t kd = k_desc + (n % KS) * (F::TILE >> 4);
        const uint32_t d = tmem + (n & 1) * F::S_COLS;
        __syncwarp();
        if (elect_one()) {
          if (FP8) {
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_f8_ss(d, kd + 2 * k, q_desc + 2 * k, idesc_s, k > 0);
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              umma_bf16_ss(d, kd + (k >> 2) * (PK * 128 >> 4) + (k & 3) * 2, q_desc + (k >> 2) * (PR * 128 >> 4) + (k & 3) * 2, idesc_s, k > 0);
          }
          umma_commit(&s_full[n & 1]);
          umma_commit(&k_empty[n % KS]);
        }
        __syncwarp();
      };
      if (n_tiles > 0) issue_s(0);
      for (int n = 0; n < n_tiles; ++n) {          // all tiles also after a time-out
        if (n + 1 < n_tiles) issue_s(n + 1);
        ok &= mbar_wait(FP8 ? &w_full[n % WS] : &v_full[n % VS], FP8 ? (n / WS) & 1 : (n / VS) & 1, abort_flag, args.status, 3);
        ok &= mbar_wait(&p_full[n % PS], (n / PS) & 1, abort_flag, args.status, 2);
        tc_fence_after();
        const uint64_t vd = v_desc + (FP8 ? (n % WS) * (F::WIDE >> 4) : (n % VS) * (F::TILE >> 4)), pd = p_desc + (n % PS) * (F::P >> 4);
        __syncwarp();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 8; ++k) umma_bf16_ss(tmem + F::O_AT, vd + k * (2048 >> 4), pd + k * (2048 >> 4), idesc_o, n > 0 || k > 0);
          umma_commit(&pv_done[n % PS]);
          umma_commit(FP8 ? &w_empty[n % WS] : &v_empty[n % VS]);
        }
        __syncwarp();
      }
      ok = __all_sync(0xffffffffu, ok);            // (the warp goes on as one)
    } else if (FP8 && warp >= 12) {
      // ------------------------------ widening of values --------------------------------
      const int row = tid & 127, sw = (row & 7) << 4;
      bool ok = true;
      for (int n = 0; n < n_tiles && ok; ++n) {
        ok = mbar_wait_warp(&v_full[n % VS], (n / VS) & 1, abort_flag, args.status, 3);
        if (!ok) break;
        const uint8_t* from = sV + (n % VS) * F::TILE + row * 128;
        uint4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const uint4*>(from + ((i << 4) ^ sw));
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_empty[n % VS]);
        if ((j0 + n) * PK + row >= most) {         // nobody reads it, and its codes may be NaN
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = make_uint4(0, 0, 0, 0);
        }
        ok = mbar_wait_warp(&w_empty[n % WS], ((n / WS) & 1) ^ 1, abort_flag, args.status, 3);
        if (!ok) break;
        uint8_t* to = sW + (n % WS) * F::WIDE + row * 128;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint2 y0 = widen4(i & 1 ? x[i >> 1].z : x[i >> 1].x), y1 = widen4(i & 1 ? x[i >> 1].w : x[i >> 1].y);
          *reinterpret_cast<uint4*>(to + (i >> 3) * (PK * 128) + (((i & 7) << 4) ^ sw)) = make_uint4(y0.x, y0.y, y1.x, y1.y);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&w_full[n % WS]);
      }
    }
  } else {
    if (FP8) asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------ softmax --------------------------------
    const int w = warp - 4, side = w >> 2, c0 = side * 32, active = (groups + 1 - side) >> 1;      // groups of eight columns from c0 on
    const int in_tile = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    bool ok = true;
    if (active > 0 && n_tiles > 0) {
      const int page_log = __ffs(p.page) - 1, c_at = ((in_tile >> page_log) << page_log) * 2 + (in_tile & (p.page - 1));      // of this thread's key
      // Two rows in every 64-bit register: sums, maxima (negative; + inf as long as there is none, so that the first score moves it), and a
      // tile's probabilities.
      uint64_t l2[16], nm[16], p2[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        l2[i] = p2[i] = 0;
        nm[i] = pack_f32x2(INFINITY, INFINITY);
      }
      const uint64_t sixteenth = pack_f32x2(0.0625f, 0.0625f);
      // e4m3: scales of this thread's key and value.  A value that is not finite makes its key's scores NaN: rows that may read it are NaN, and
      // elsewhere it is not seen.
      auto scales_of = [&](int n) -> float2 {
        const float* c = sC + (n % CS) * PK * 2 + c_at;
        const float2 x = make_float2(c[0], c[p.page]);
        return fabsf(x.y) < INFINITY ? x : make_float2(__int_as_float(0x7fffffff), 0.f);
      };
      // the registers' copies of what has changed in shared memory
      auto take = [&](bool sums) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (i >= 4 * active) break;
          const int c = c0 + 2 * i;
          nm[i] = pack_f32x2(-sh.row[c].m, -sh.row[c + 1].m);
          if (sums) l2[i] = mul_f32x2(l2[i], pack_f32x2(sh.f[c], sh.f[c + 1]));
        }
      };
      {
        // Where the maxima begin: at those of 32 keys (of a tile that the mask cuts: nowhere, see move_maxima).  Every warp sets one group of rows.
        float2 sc = make_float2(1.f, 1.f);
        if (FP8) {
          ok &= mbar_wait(&c_full[0], 0, abort_flag, args.status, 5);
          sc = scales_of(0);
        }
        ok &= mbar_wait(&s_full[0], 0, abort_flag, args.status, 5);
        __syncwarp();
        tc_fence_after();
        const int i = w & 3, col = c0 + 8 * i;
        if (i < active && j0 * PK + PK <= least) {
          const float ks = sc.x * args.scale_log2;
          const uint32_t S = tmem + col + lanes;
          const float m = row_tops<FP8>(S, sh.row + col, nullptr, 0, ks, false, 0.f);
          if (lane < 8) sh.row[col + lane].m = m + Range<FP8>::LEAD;
          if (FP8) {
            __syncwarp();
            const float mv = row_tops<FP8>(S, sh.row + col, nullptr, 0, ks, true, log2_of(sc.y));
            if (lane < 8) {
              sh.mv[col + lane] = mv;
              sh.ec[col + lane] = exponent_of(mv);
              sh.vf[col + lane] = (uint16_t)((127 + exponent_of(mv)) << 7);
            }
          }
        }
        named_bar_sync(2 + side, 128);
        take(false);
      }
      for (int n = 0; n < n_tiles; ++n) {        // all tiles also after a time-out
        const int k0 = (j0 + n) * PK, key = k0 + in_tile;
        const bool dirty = k0 + PK > least;      // some row may not read all of it
        float2 sc = make_float2(1.f, 1.f);
        if (FP8) {
          ok &= mbar_wait(&c_full[n % CS], (n / CS) & 1, abort_flag, args.status, 5);
          sc = scales_of(n);
        }
        const float ks = sc.x * args.scale_log2;
        const uint64_t ks2 = pack_f32x2(ks, ks), vs2 = pack_f32x2(sc.y, sc.y);
        uint8_t* P = sP + (n % PS) * F::P;
        ok &= mbar_wait(&s_full[n & 1], (n >> 1) & 1, abort_flag, args.status, 5);
        // P's place is free.  (e4m3: PV(n - 2) was asked for before S(n), by the same thread, so s_full says so.)
        if (!FP8 && n > 0) ok &= mbar_wait(&pv_done[0], (n - 1) & 1, abort_flag, args.status, 6);
        __syncwarp();
        tc_fence_after();
        const uint32_t S = tmem + (n & 1) * F::S_COLS + c0 + lanes;
        bool again = false;                      // the maxima have moved: once more
        do {
          // Probabilities, and whether one is too large for where the maxima are; their products are written all the same, and once more after the
          // maxima have moved.
          float mx = -INFINITY, mw = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i < active) {
              uint32_t h[8], lo[8];
              tmem_ld_x8(S + 8 * i, h);
              if (FP8) tmem_ld_x8(S + PR + 8 * i, lo);
              uint4 rs4 = make_uint4(0, 0, 0, 0), vf4 = rs4;
              if (FP8) {
                rs4 = *reinterpret_cast<const uint4*>(sh.rs + c0 + 8 * i);
                vf4 = *reinterpret_cast<const uint4*>(sh.vf + c0 + 8 * i);
              }
              const uint32_t rs2[4] = {rs4.x, rs4.y, rs4.z, rs4.w}, vf2[4] = {vf4.x, vf4.y, vf4.z, vf4.w};
              tmem_ld_wait();
              uint64_t y[4];                       // log2 units; product and difference are never fused
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                y[e] = pack_f32x2(__uint_as_float(h[2 * e]), __uint_as_float(h[2 * e + 1]));
                if (FP8) {
                  y[e] = fma_f32x2(pack_f32x2(__uint_as_float(lo[2 * e]), __uint_as_float(lo[2 * e + 1])), sixteenth, y[e]);
                  y[e] = mul_f32x2(y[e], mul_f32x2(bf16x2_to_f32x2(rs2[e]), ks2));
                } else {
                  y[e] = mul_f32x2(y[e], ks2);
                }
                y[e] = add_f32x2(y[e], nm[4 * i + e]);
              }
              if (__builtin_expect(dirty, 0)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float a, b;
                  unpack_f32x2(y[e], a, b);
                  const int2 lim = *reinterpret_cast<const int2*>(sh.lim + c0 + 8 * i + 2 * e);
                  y[e] = pack_f32x2(key >= lim.x ? -INFINITY : a, key >= lim.y ? -INFINITY : b);
                }
              }
              uint32_t u[4], v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float a, b;
                unpack_f32x2(y[e], a, b);
                mx = max3(mx, a, b);
                const float pa = fast_exp2(a), pb = fast_exp2(b);
                const uint64_t pp = pack_f32x2(pa, pb);
                p2[4 * i + e] = pp;
                if (FP8) {
                  float wa, wb;
                  unpack_f32x2(mul_f32x2(mul_f32x2(pp, vs2), bf16x2_to_f32x2(vf2[e])), wa, wb);
                  mw = max3(mw, wa, wb);
                  u[e] = pack_f16x2(wa, wb);
                } else {
                  const uint32_t hi = pack_bf16x2(pa, pb);
                  float ra, rb;
                  unpack_f32x2(add_f32x2(pp, bf16x2_to_f32x2(hi ^ 0x80008000u)), ra, rb);
                  u[e] = hi;
                  v[e] = pack_bf16x2(ra, rb);
                }
              }
              const uint32_t to = swz128_offset(in_tile, side * 4 + i);
              *reinterpret_cast<uint4*>(P + to) = make_uint4(u[0], u[1], u[2], u[3]);
              if (!FP8) *reinterpret_cast<uint4*>(P + PK * 128 + to) = make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
          if (__builtin_expect(named_bar_any(2 + side, 128, !again && (mx > Range<FP8>::MOST || mw > 32768.f)), 0)) {
            if (n > 0) {
              ok &= mbar_wait(&pv_done[(n - 1) % PS], ((n - 1) / PS) & 1, abort_flag, args.status, 6);
              __syncwarp();
              tc_fence_after();
            }
            move_maxima<FP8>(sh, S, tmem + F::O_AT + lanes, side, active, key, ks, FP8 ? log2_of(sc.y) : 0.f, dirty, n == 0);
            take(true);
            again = true;
          } else {
            again = false;
          }
        } while (again);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[n & 1]);
#pragma unroll
        for (int i = 0; i < 16; ++i) l2[i] = add_f32x2(l2[i], p2[i]);
        if (!FP8 && __builtin_expect(dirty, 0)) {
          // values that some row may not read: what nobody may and what is not finite is cleared, see attn_paged.cu
          ok &= mbar_wait(&v_full[n % VS], (n / VS) & 1, abort_flag, args.status, 5);
          uint8_t* tile = sV + (n % VS) * F::TILE;
          for (int i = tid - 128; i < PK * 16; i += 128 * sides) {
            const int k = i >> 4;
            uint4* at = reinterpret_cast<uint4*>(tile + ((i & 15) >> 3) * (PK * 128) + swz128_offset(k, i & 7));
            uint4 x = *at;
            uint32_t* z = reinterpret_cast<uint32_t*>(&x);
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool a = (z[e] & 0x7f80u) == 0x7f80u, b = (z[e] & 0x7f800000u) == 0x7f800000u;
              bad |= a || b;
              z[e] &= (a ? 0xffff0000u : 0xffffffffu) & (b ? 0xffffu : 0xffffffffu);
            }
            if (k0 + k >= most) {
              *at = make_uint4(0, 0, 0, 0);
            } else if (bad) {
              *at = x;
              atomicMin(&s_poison, k0 + k);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[n % PS]);
      }
      // Sums over the keys' threads, row i in lane i: every step adds half of the rows across half of the lanes.  Then the output.
      float l[32];
#pragma unroll
      for (int i = 0; i < 16; ++i) unpack_f32x2(l2[i], l[2 * i], l[2 * i + 1]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < o; ++i) {
          const float send = lane & o ? l[i] : l[i + o], keep = lane & o ? l[i + o] : l[i];
          l[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      sh.sum[w][lane] = l[0];
      ok &= mbar_wait(&pv_done[(n_tiles - 1) % PS], ((n_tiles - 1) / PS) & 1, abort_flag, args.status, 6);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      named_bar_sync(2 + side, 128);
      if ((w & 3) == 0 && lane < 8 * active) {
        // The maximum that is left goes up by the whole part of the sum's logarithm: the part is then the mean of values, times less than two, and as
        // large as they are at most.
        const int col = c0 + lane;
        const float m = sh.row[col].m;
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) sum += sh.sum[side * 4 + k][lane];
        const float up = sum >= 2.f && sum < INFINITY ? m + (float)((int)(__float_as_uint(sum) >> 23) - 127) : m;
        const float f = up == m ? 1.f : exp2f(m - up);
        sum *= f;
        if (!FP8 && sh.lim[col] > *reinterpret_cast<volatile int*>(&s_poison)) sum = __int_as_float(0x7fffffff);
        sh.f[col] = f;
        sh.row[col].m = sum != sum && m == -INFINITY ? 0.f : up;       // all NaN: not to be taken for no keys at all
        sh.sum[side * 4][lane] = sum;
      }
      named_bar_sync(2 + side, 128);
#pragma unroll 1
      for (int i = 0; i < active; ++i) {
        uint32_t h[8], lo[8];
        tmem_ld_x8(tmem + F::O_AT + c0 + 8 * i + lanes, h);
        if (!FP8) tmem_ld_x8(tmem + F::O_AT + PR + c0 + 8 * i + lanes, lo);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int col = c0 + 8 * i + e, r = (2 * i + side) * 8 + e;
          const float o = FP8 ? __uint_as_float(h[e]) : __uint_as_float(h[e]) + __uint_as_float(lo[e]);
          if (r < rows && ok)
            args.part[((long long)(item.w + r) * args.heads + head) * HEAD + in_tile] = FP8 ? o * sh.f[col] * __int_as_float((127 - sh.ec[col]) << 23) : o * sh.f[col];
        }
      }
    }
    if ((w & 3) == 0 && lane < 8 * active) {
      const int col = c0 + lane, r = (2 * (lane >> 3) + side) * 8 + (lane & 7);
      if (r < rows)
        args.part_ml[(long long)(item.w + r) * args.heads + head] =
            n_tiles > 0 ? make_float2(sh.row[col].m, sh.sum[side * 4][lane]) : make_float2(-INFINITY, 0.f);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {                             // copies may be on their way into this CTA's memory
    const uint64_t t = globaltimer_ns();
    while (globaltimer_ns() - t < 2000000ull) {
    }
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, F::COLS);
  }
  if (args.beside) pdl_wait();
}

template <bool FP8>
static int launch(const Cache& c, const Plan& p, const PrefixArgs& a, cudaStream_t st) {
  int dev = 0;
  SNU1_CUDA_CHECK(cudaGetDevice(&dev));
  static std::once_flag once[64];
  cudaError_t err = cudaSuccess;
  std::call_once(once[dev & 63], [&]() {
    err = cudaFuncSetAttribute(paged_prefix_kernel<FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, Prefix<FP8>::SMEM);
  });
  SNU1_CUDA_CHECK(err);
  SNU1_CUDA_CHECK(launch_pdl(paged_prefix_kernel<FP8>, dim3(a.heads * p.prefix_count), dim3(Prefix<FP8>::THREADS), Prefix<FP8>::SMEM, st, c.k, FP8 ? c.scale : c.v, p, a));
  return kHostOk;
}

int launch_prefix(const Cache& c, const Plan& p, const void* q, long long ldq, float* part, float2* part_ml, float scale_log2, int beside, cudaStream_t st) {
  PrefixArgs a;
  a.q = (const __nv_bfloat16*)q;
  a.ldq = ldq;
  a.part = part;
  a.part_ml = part_ml;
  a.pages = c.pages;
  a.heads = c.heads;
  a.scale_log2 = scale_log2;
  a.beside = beside;
  a.status = device_status_word();
  return c.fp8 ? launch<true>(c, p, a, st) : launch<false>(c, p, a, st);
}

}  // namespace paged
}  // namespace snu1
