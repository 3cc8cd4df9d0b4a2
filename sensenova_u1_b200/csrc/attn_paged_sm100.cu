// Attention of chunks of new tokens over a paged cache: many rows per key/value head, so the products belong on the
// tensor cores (tcgen05.mma, scores and output of two row tiles in tensor memory).  The pipeline is that of attn_infer_sm100.cu:
// warp 0 asks for pages through TMA, warp 1 issues the products in the order S_A(j+1) PV_A(j) S_B(j+1) PV_B(j), eight softmax
// warps per tile of 16 rows each, probabilities over the other tile's scores as the A operand of the second product.
//
// What is different:
// * A row tile holds all query heads of one key/value head: 128 / group tokens, head after head (one TMA box from q).  A
//   chunk of a few dozen tokens fills the tensor cores' 128 rows, and the heads of a group read keys and values once.
// * Keys and values come page by page (a lane of the loading warp per page).  An e4m3 cache is widened to fp16 pages of scratch
//   first (paged_widen_kernel: code times scale, divided by one power of two per tile and head), and queries and probabilities
//   are fp16 as well.  So the softmax pays for the scales once per tile and row, not per score: the keys' power of two goes
//   into the factor of the scores, the values' into the exponent of the probabilities (and out of their sum).  Scales
//   applied per score and probability in fp32 took 2.33 us per pair of tiles instead of 1.78 (2 x 512 new tokens, 8192 keys);
//   keys rounded to bf16 would move every score by up to 2^-8 of the sum of |q k|.  The queries are scaled row by row, by the
//   softmax warps.
// * The mask is one number per row, the keys that it may read; tiles that all rows read whole need no test.
// * A work item is a part of the key tiles of two row tiles; unnormalised results of parts are joined by
//   paged_join_kernel.  ops/paged.py chooses the parts so that the waves of CTAs are full.
// * Two warps that have nothing else to do clear values that are not finite (and rows behind the last token) in the bf16 tiles
//   that some row may not read whole (widening does so for e4m3): a probability of zero does not hide them from the product.
//   Rows that may read such a value give NaN, the others are as if it were not there.
//
// Measured (32 / 8 heads): bf16, 2 x 512 new tokens over 8300 keys 138 us in a graph of 20 calls, 0.98 PFLOP/s, 146 to 153 when called for a
// second on end (the power limit takes the clocks down); a pair of tiles takes 1.78 us, 0.82 of the tensor cores' measured rate if all SMs
// were at it (128 CTAs on 148 SMs), and a CTA 8 to 10 us to start and end.  e4m3, 4096 tokens at the end of 32001: 1.73 ms, 1.16 PFLOP/s, or
// 2.01 to 2.08 in a loop.  Chunks of up to 256 rows over e4m3, 8 x 64 rows over 12000 keys: 94 us, 2.2 TB/s, 3300 clocks per tile of 128 rows.
// Four warps widen keys, four values, and two turn scales into factors two tiles ahead; with eight warps doing all three one after
// the other it took 1.13 times as long.  Without the multiplications 0.93, without the exponentials 0.88, without both 0.83 of the time: what
// bounds it is each warp's own chain.  Softmax warps without rows that only keep step made it 1.01, two places for P (so that its store need
// not wait for the product before) 1.10 times as long.
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <float.h>
#include <string.h>

#include <mutex>

#include "host_common.h"
#include "paged.cuh"

namespace snu1 {
namespace paged {

constexpr int BK = 128;                         // keys of a tile
constexpr int CHALF = 128 * 64 * 2;             // 64 columns of a 128-row tile
constexpr int CTILE = 2 * CHALF;
constexpr int CHUNK_THREADS = 640;
constexpr int RAW_UNIT = 128 * 128;             // codes of a tile's keys, or of its values
constexpr int RAW_STAGES = 3, SCALE_STAGES = 4;    // of units; of tiles

// What a CTA reads: bf16 pages, e4m3 pages that have been widened to fp16, or e4m3 pages as they are.
enum ChunkMode { kPages, kWide, kRaw };
template <int MODE>
struct Chunk {
  static constexpr bool FP16 = MODE != kPages, RAW = MODE == kRaw;
  static constexpr int TILES = RAW ? 1 : 2;     // row tiles
  static constexpr int K_STAGES = RAW ? 2 : 3, V_STAGES = 2;
  static constexpr int RING = RAW ? RAW_STAGES * RAW_UNIT + SCALE_STAGES * 2048 : 0;
  static constexpr int SMEM = (TILES + K_STAGES + V_STAGES) * CTILE + RING + 512 + 1024;
};

struct ChunkArgs {
  const __nv_bfloat16* q;
  long long ldq;
  __nv_bfloat16* o;
  long long ldo;
  float* part;
  float2* part_ml;
  const int* first_page;   // scratch of widened rows: a sequence's first page there; null: the cache's own pages
  const int4* items;
  const float4* factors;   // of the widened pages, see paged_widen_kernel
  int page, pages, heads;
  float scale_log2;
  const uint8_t* data;     // the cache itself
  const float* scales;
  int cache_pages;
  int* status;
};

// see attn_infer_sm100.cu
__device__ __forceinline__ void tally_add(int* c) {
  asm volatile("red.release.cta.shared::cta.add.s32 [%0], 1;" ::"r"(smem_u32(c)) : "memory");
}
__device__ __forceinline__ bool tally_wait(const int* c, int target, volatile int* abort_flag, int* status, int where) {
  const uint32_t a = smem_u32(c);
  uint64_t t0 = 0;
  for (uint32_t spins = 0;; ++spins) {
    int v;
    asm volatile("ld.acquire.cta.shared::cta.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    if (v >= target) return true;
    if ((spins & 0x3ff) == 32) {
      if (*abort_flag) return false;
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > kLocalWaitNs) {
        *abort_flag = 1;
        report_status(status, kWaitTimeout, where);
        return false;
      }
    }
  }
}

// The products with descriptors given by their lower words (the upper word is the same for all tiles here): the issuing
// warp has 64 registers, and pairs of them per product do not fit.
constexpr uint32_t DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;     // see make_smem_desc
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 da, db;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "mov.b64 da, {%1, %5};\n"
      "mov.b64 db, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n"
      "}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(DESC_HI)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 db;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "mov.b64 db, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n"
      "}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(DESC_HI)
      : "memory");
}

// Sums of probabilities over e4m3 are kept 2^12 times smaller.  A tile of zeros (or values below 2^-80) has 2^-93 as its power of two: a
// probability, up to 2^15, counts 2^96 then, and 2^30 keys of them stay below 2^128.  At the other end, 2^113, a factor is 2^-125.
constexpr float SUM_DOWN = 12.f;
constexpr uint32_t CLEAR_ROW = 0x80000000u;     // a row's factor: + 0 and - 0, which no scale gives

// One row's attention to keys [k0, k1) of its sequence by one warp, in fp32 on the cache as it is; four values per lane.  The softmax of the
// chunk kernel takes a score's product and the running maximum's difference in one step.  The maximum is rounded, the product is not, so
// 2^-24 of the score is left over: beyond 2^20 that would show, and from 2^26 on probabilities overflow.  A warp that meets such a
// row computes it again here.  (As a branch of the softmax's loop, rounding such scores first made all calls 5 to 18 % slower.)
constexpr float FAR = 1048576.f;                // 2^20, log2 units
template <bool FP8>
__noinline__ __device__ void far_row(const Plan& p, const ChunkArgs& a, int b, int row, int head, int kvh, int k0, int k1, float4* x, float2* ml) {
  const int lane = threadIdx.x & 31, group = 4;
  const uint2 u = *reinterpret_cast<const uint2*>(a.q + row * a.ldq + head * HEAD + lane * 4);
  const float q[4] = {__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u)};
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = k0; k < k1; k += group) {
    float v[group][4], s[group];
#pragma unroll
    for (int i = 0; i < group; ++i) {
      const int key = min(k + i, k1 - 1), pg = p.table[(long long)b * p.width + key / p.page];
      float c[2][4];
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const long long at = (((long long)pg * 2 + kv) * a.heads + kvh) * p.page + key % p.page;
        const bool there = pg >= 0 && pg < a.cache_pages;        // (reported by who asked for the page)
        if (FP8) {
          const uint32_t w = there ? *reinterpret_cast<const uint32_t*>(a.data + at * HEAD + lane * 4) : 0u;
          const float scale = there ? a.scales[at] : 0.f;
          const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3)));
          const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3)));
          c[kv][0] = lo.x * scale, c[kv][1] = lo.y * scale, c[kv][2] = hi.x * scale, c[kv][3] = hi.y * scale;
        } else {
          const uint2 w = there ? *reinterpret_cast<const uint2*>(a.data + at * (2 * HEAD) + lane * 8) : make_uint2(0, 0);
          c[kv][0] = __uint_as_float(w.x << 16), c[kv][1] = __uint_as_float(w.x & 0xffff0000u);
          c[kv][2] = __uint_as_float(w.y << 16), c[kv][3] = __uint_as_float(w.y & 0xffff0000u);
        }
      }
      s[i] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i] = fmaf(q[e], c[0][e], s[i]);
        v[i][e] = c[1][e];
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < group; ++i) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
      s[i] = k + i < k1 ? __fmul_rn(s[i], a.scale_log2) : -INFINITY;
      top = fmaxf(top, s[i]);
    }
    const float now = fmaxf(m, top), f = m == -INFINITY ? 0.f : fast_exp2(m - now);
    m = now;
    l *= f;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= f;
#pragma unroll
    for (int i = 0; i < group; ++i) {
      if (k + i >= k1) break;
      const float pr = fast_exp2(s[i] - m);
      l += pr;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(pr, v[i][e], acc[e]);
    }
  }
  *x = make_float4(acc[0], acc[1], acc[2], acc[3]);
  *ml = make_float2(m, l);
}

template <int MODE>
__global__ void __launch_bounds__(CHUNK_THREADS, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Plan p, const __grid_constant__ ChunkArgs args) {
  using C = Chunk<MODE>;
  constexpr bool FP16 = C::FP16, RAW = C::RAW;
  constexpr int TILES = C::TILES, CK_STAGES = C::K_STAGES, CV_STAGES = C::V_STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + TILES * CTILE;
  uint8_t* sV = sK + CK_STAGES * CTILE;
  uint8_t* s_raw = sV + CV_STAGES * CTILE;                 // [RAW_STAGES] codes of keys and of values in turn
  float* s_scale = reinterpret_cast<float*>(s_raw + RAW_STAGES * RAW_UNIT);     // [SCALE_STAGES][page][keys, values][token]
  uint32_t* s_mult = reinterpret_cast<uint32_t*>(s_scale + SCALE_STAGES * 256);  // [SCALE_STAGES][keys, values][token]: two fp16 numbers
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_raw + C::RING);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;
  uint64_t* k_empty = k_full + CK_STAGES;
  uint64_t* v_full = k_empty + CK_STAGES;
  uint64_t* v_empty = v_full + CV_STAGES;
  uint64_t* v_dirty = v_empty + CV_STAGES;      // [stages] the stage has to be cleaned
  uint64_t* v_clean = v_dirty + CV_STAGES;      // [stages] the cleaning warps are done with it
  uint64_t* s_full = v_clean + CV_STAGES;       // [2] per row tile
  uint64_t* s_empty = s_full + 2;
  uint64_t* p_full = s_empty + 2;
  uint64_t* pv_done = p_full + 2;
  uint64_t* q_ready = pv_done + 2;              // e4m3: the queries are fp16
  // (units of keys and of values go through one ring, but each has barriers of its own: who waits for every other phase of a
  // barrier cannot tell it from the one before)
  uint64_t* raw_full = q_ready + 1;             // [2 RAW_STAGES] by unit
  uint64_t* raw_empty = raw_full + 2 * RAW_STAGES;
  uint64_t* scale_full = raw_empty + 2 * RAW_STAGES;      // [SCALE_STAGES] by tile: s_scale
  uint64_t* mult_full = scale_full + SCALE_STAGES;        // [SCALE_STAGES] by tile: s_mult and s_factor
  float2* s_factor = reinterpret_cast<float2*>(mult_full + SCALE_STAGES);        // [2 SCALE_STAGES] of tiles: see ChunkArgs::factors
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_factor + 2 * SCALE_STAGES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* drained = reinterpret_cast<int*>(tmem_slot + 2);   // [2] softmax warps that have read a score tile, all tiles so far
  int* lim_max = drained + 2;                              // [2] the largest and the smallest limit of a row tile
  int* lim_min = lim_max + 2;
  int* poison = lim_min + 2;                               // first key of a tile not read whole whose value was not finite

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < CK_STAGES; ++i) {
      mbar_init(&k_full[i], RAW ? 4 : 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < 2 * RAW_STAGES; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 4);
    }
    for (int i = 0; i < SCALE_STAGES; ++i) {
      mbar_init(&scale_full[i], 1);
      mbar_init(&mult_full[i], 2);
    }
    for (int i = 0; i < CV_STAGES; ++i) {
      mbar_init(&v_full[i], RAW ? 4 : 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&v_dirty[i], 1);
      mbar_init(&v_clean[i], 2);
    }
    mbar_init(q_ready, 8 * TILES);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 8);
      mbar_init(&p_full[i], 8);
      mbar_init(&pv_done[i], 1);
      drained[i] = lim_max[i] = 0;
      lim_min[i] = *poison = 0x7fffffff;
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // what the plan's host side has set, before the wait: no launch in front writes it
  const int4 item = args.items[blockIdx.x / args.heads];
  const int b = item.x, part = item.z & 0xffff, parts = item.z >> 16;
  const int kvh = blockIdx.x % args.heads, G = p.group, T = 128 / G;       // tokens of a row tile
  const int q0 = p.q_start[b], q_len = p.q_start[b + 1] - q0;
  const int token0 = item.y / G;
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x == 0) {                       // the queries do not depend on what is looked up below
    mbar_expect_tx(q_full, 2 * TILES * T * G * 128);
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      tma_load_3d(sQ + t * CTILE, &tm_q, q_full, 0, kvh * G, q0 + token0 + t * T);
      tma_load_3d(sQ + t * CTILE + CHALF, &tm_q, q_full, 64, kvh * G, q0 + token0 + t * T);
    }
    report_grown(p, b, args.status);
  }
  const int kv_len = seq_len(p, b);
  int max_a, max_b, min_a, min_b;               // the largest and the smallest limit of row tiles A and B
  if (p.behind == nullptr) {                    // limits grow from token to token
    const int ends = min(token0 + TILES * T, q_len) - 1;
    min_a = row_limit(p, q0, q_len, kv_len, token0);
    max_a = row_limit(p, q0, q_len, kv_len, min(token0 + T - 1, ends));
    min_b = token0 + T <= ends ? row_limit(p, q0, q_len, kv_len, token0 + T) : 0x7fffffff;
    max_b = token0 + T <= ends ? row_limit(p, q0, q_len, kv_len, ends) : 0;
  } else {
    if (threadIdx.x < TILES * T) {
      const int t = threadIdx.x / T, token = token0 + threadIdx.x;
      if (token < q_len) {
        const int l = row_limit(p, q0, q_len, kv_len, token);
        atomicMax(&lim_max[t], l);
        atomicMin(&lim_min[t], l);
      }
    }
    __syncthreads();
    max_a = lim_max[0], max_b = lim_max[1], min_a = lim_min[0], min_b = lim_min[1];
  }
  const int most = max(max_a, max_b);
  const int all = (most + BK - 1) / BK;
  const int j0 = (int)((long long)all * part / parts), n = (int)((long long)all * (part + 1) / parts) - j0;
  // Row tile A (B) reads the part's first n_a (n_b) key tiles, all but the first full_a (full_b) of them with the mask.
  const int n_a = max(0, min(n, (max_a + BK - 1) / BK - j0)), n_b = max(0, min(n, (max_b + BK - 1) / BK - j0));
  const int full_a = min_a / BK - j0, full_b = min_b / BK - j0;
  auto dirty = [&](int j) -> bool { return !FP16 && ((j < n_a && j >= full_a) || (j < n_b && j >= full_b)); };
  // columns: S_A and P_B [0,128), S_B and P_A [128,256), O_A [256,384), O_B [384,512)

  // 640 threads start with 96 registers: 128 x 64 + 512 x 104 = 640 x 96
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 0) {
      if (n == 0) {
        mbar_wait_warp(q_full, 0, abort_flag, args.status, 1);      // nobody else does, and the CTA has to outlive the copy
      } else {
        const int page = args.page, per = BK / page, used = (most + page - 1) / page;   // pages of a tile, of the sequence
        const int* table = args.first_page == nullptr ? p.table + (long long)b * p.width : nullptr;
        const int base = args.first_page == nullptr ? 0 : args.first_page[b];
        // a lane's page of tile j, read a tile ahead
        auto page_of = [&](int j) -> int {
          const int i = (j0 + j) * per + lane;
          return j < n && lane < per && i < used ? (table != nullptr ? table[i] : base + i) : 0;
        };
        int pk = page_of(0), pv = pk, ahead = page_of(1);
        bool ok = true;
        auto load = [&](uint8_t* dst, const CUtensorMap* tm, uint64_t* full, int j, int pg) {
          const int live = min(per, used - (j0 + j) * per);
          if (lane == 0) mbar_expect_tx(full, live * page * 256);
          __syncwarp();
          if (lane < live) {
            if (pg < 0 || pg >= args.pages) report_status(args.status, kBadPage, 10);     // reads as zeros
            tma_load_4d(dst + lane * page * 128, tm, full, 0, 0, kvh, pg);
            tma_load_4d(dst + CHALF + lane * page * 128, tm, full, 64, 0, kvh, pg);
          }
          __syncwarp();
        };
        auto load_k = [&](int j, int pg) {
          const int s = j % CK_STAGES;
          ok = mbar_wait_warp(&k_empty[s], ((j / CK_STAGES) & 1) ^ 1, abort_flag, args.status, 1);
          if (ok) load(sK + s * CTILE, &tm_k, &k_full[s], j, pg);
        };
        if (RAW) {
          // Codes of keys and codes of values in turn into one ring, and two tiles ahead the scales of both.
          int far = page_of(2);
          auto load_scales = [&](int j, int pg) {
            if (j >= n) return;
            const int live = min(per, used - (j0 + j) * per), s = j % SCALE_STAGES;
            if (lane == 0) mbar_expect_tx(&scale_full[s], live * page * 8);
            __syncwarp();
            if (lane < live) tma_load_4d(s_scale + s * 256 + lane * page * 2, &tm_v, &scale_full[s], 0, kvh, 0, pg);
            __syncwarp();
          };
          load_scales(0, pk);
          load_scales(1, ahead);
          for (int j = 0; j < n && ok; ++j) {
            const int pg = pk, two = far, live = min(per, used - (j0 + j) * per);
            pk = ahead;
            ahead = far;
            far = page_of(j + 3);
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
              const int u = 2 * j + kv, s = u % RAW_STAGES, w = u - RAW_STAGES;
              if (w >= 0) ok = ok && mbar_wait_warp(&raw_empty[w % (2 * RAW_STAGES)], (w / (2 * RAW_STAGES)) & 1, abort_flag, args.status, 1);
              if (!ok) break;
              uint64_t* full = &raw_full[u % (2 * RAW_STAGES)];
              if (lane == 0) mbar_expect_tx(full, live * page * 128);
              __syncwarp();
              if (lane < live) {
                if (pg < 0 || pg >= args.pages) report_status(args.status, kBadPage, 10);     // reads as zeros
                tma_load_5d(smem_u32(s_raw + s * RAW_UNIT + lane * page * 128), &tm_k, full, 0, 0, kvh, kv, pg);
              }
              __syncwarp();
              // what was made of the scales four tiles before has been read: keys and values of that tile have left the ring
              if (kv == 0) load_scales(j + 2, two);
            }
          }
        } else {
          load_k(0, pk);
        }
        for (int j = 0; j < n && ok && !RAW; ++j) {
          if (j + 1 < n) {
            pk = ahead;
            ahead = page_of(j + 2);
            load_k(j + 1, pk);
          }
          if (!ok) break;
          const int s = j % CV_STAGES;
          ok = mbar_wait_warp(&v_empty[s], ((j / CV_STAGES) & 1) ^ 1, abort_flag, args.status, 1);
          if (!ok) break;
          load(sV + s * CTILE, &tm_v, &v_full[s], j, pv);
          pv = pk;
        }
      }
    } else if (warp == 1) {
      // The whole warp walks the tiles and one elected lane issues (see mbar_ready in attn_common.cuh).
      if (n > 0) {
        // bits [7,10) and [10,13) of the descriptor: bf16 (1) or fp16 (0) operands
        constexpr uint32_t type = FP16 ? ~(1u << 7 | 1u << 10) : ~0u;
        constexpr uint32_t idesc_s = make_idesc_bf16(128, 128, false, false) & type;
        constexpr uint32_t idesc_pv = make_idesc_bf16(128, 128, false, true) & type;
        const uint32_t q_desc = (uint32_t)make_smem_desc(smem_u32(sQ), 0, 1024);
        const uint32_t k_desc = (uint32_t)make_smem_desc(smem_u32(sK), 0, 1024);
        const uint32_t v_desc = (uint32_t)make_smem_desc(smem_u32(sV), CHALF, 1024);
        bool ok = mbar_wait(FP16 ? q_ready : q_full, 0, abort_flag, args.status, 3);   // this lane's; see mbar_wait_warp
        uint32_t cleaned = 0;                   // phase of every stage's v_clean
        auto issue_s = [&](int j, int t) {
          if (j < (t ? n_b : n_a)) {
            ok &= mbar_wait(&s_empty[t], (j & 1) ^ 1, abort_flag, args.status, 2);
            tc_fence_after();
            const uint32_t qd = q_desc + t * (CTILE >> 4), kd = k_desc + (j % CK_STAGES) * (CTILE >> 4);
            __syncwarp();
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                constexpr uint32_t half = CHALF >> 4;
                const uint32_t off = (k >> 2) * half + (k & 3) * 2;
                umma_ss(tmem_base + t * 128, qd + off, kd + off, idesc_s, k > 0 ? 1u : 0u);
              }
              umma_commit(&s_full[t]);
            }
            __syncwarp();
          }
        };
        auto issue_pv = [&](int j, int t) {
          if (j < (t ? n_b : n_a)) {
            ok &= mbar_wait(&p_full[t], j & 1, abort_flag, args.status, 2);
            tc_fence_after();
            const uint32_t vd = v_desc + (j % CV_STAGES) * (CTILE >> 4);
            const uint32_t p_tmem = tmem_base + (t ^ 1) * 128;
            const uint32_t acc0 = j > 0 ? 1u : 0u;
            __syncwarp();
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                umma_ts(tmem_base + 256 + t * 128, p_tmem + k * 8, vd + k * (2048 >> 4), idesc_pv, k > 0 ? 1u : acc0);
              umma_commit(&pv_done[t]);
            }
            __syncwarp();
          }
        };
        auto release = [&](uint64_t* bar) {
          if (elect_one()) umma_commit(bar);
          __syncwarp();
        };
        ok &= mbar_wait(&k_full[0], 0, abort_flag, args.status, 3);
        issue_s(0, 0);
        issue_s(0, 1);
        release(&k_empty[0]);
        if (n > 1) ok &= mbar_wait(&k_full[1], 0, abort_flag, args.status, 3);
        ok &= mbar_wait(&v_full[0], 0, abort_flag, args.status, 3);
        for (int j = 0; j < n; ++j) {      // all tiles also after a time-out
          const bool more = j + 1 < n, clean = dirty(j);
          if (clean && lane == 0) mbar_arrive(&v_dirty[j % CV_STAGES]);
          if (more) issue_s(j + 1, 0);
          if (clean) {
            const int s = j % CV_STAGES;
            ok &= mbar_wait(&v_clean[s], (cleaned >> s) & 1, abort_flag, args.status, 3);
            cleaned ^= 1u << s;
          }
          issue_pv(j, 0);
          if (more) {
            issue_s(j + 1, 1);
            release(&k_empty[(j + 1) % CK_STAGES]);
          }
          issue_pv(j, 1);
          if (more) {
            release(&v_empty[j % CV_STAGES]);
            if (j + 2 < n) ok &= mbar_wait(&k_full[(j + 2) % CK_STAGES], ((j + 2) / CK_STAGES) & 1, abort_flag, args.status, 3);
            ok &= mbar_wait(&v_full[(j + 1) % CV_STAGES], ((j + 1) / CV_STAGES) & 1, abort_flag, args.status, 3);
          }
        }
        ok = __all_sync(0xffffffffu, ok);       // (nothing here depends on it; the warp goes on as one)
      }
    } else if (RAW) {
      // ------------------------------ scales --------------------------------
      // A tile is scaled like those of paged_widen_kernel; a scale is two fp16 numbers then.  The exponents go to the softmax.  Rows that nobody reads and values that are not finite are to be cleared.
      const int tid = threadIdx.x - 64, page = args.page, page_log = __ffs(page) - 1;
      auto place = [&](int r, int kv) -> int { return (((r >> page_log) * 2 + kv) << page_log) + (r & (page - 1)); };
      bool ok = true;
      for (int j = 0; j < n && ok; ++j) {
        const int k0 = (j0 + j) * BK, s = j % SCALE_STAGES;
        ok = mbar_wait_warp(&scale_full[s], (j / SCALE_STAGES) & 1, abort_flag, args.status, 3);
        const float* sc = s_scale + s * 256;
        uint32_t* out = s_mult + s * 256;
        int ex[2];
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const float4 x = *reinterpret_cast<const float4*>(sc + place(4 * lane, kv));       // four rows, which lie in one page
          const float y[4] = {x.x, x.y, x.z, x.w};
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (k0 + 4 * lane + i < most && fabsf(y[i]) < INFINITY) top = max(top, __float_as_uint(fabsf(y[i])));
          ex[kv] = tile_exponent(__uint_as_float(__reduce_max_sync(0xffffffffu, top))) - WIDEN_UP;
          const float2 mine = *reinterpret_cast<const float2*>(sc + place(2 * tid, kv));
          uint32_t w[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int key = k0 + 2 * tid + i;
            const float f = (i ? mine.y : mine.x) * __int_as_float((127 - ex[kv]) << 23);
            w[i] = split_f16(f);
            if (key >= most) {
              w[i] = CLEAR_ROW;
            } else if (kv && !(fabsf(f) < INFINITY)) {
              w[i] = CLEAR_ROW;
              atomicMin(poison, key);
            }
          }
          *reinterpret_cast<uint2*>(out + kv * 128 + 2 * tid) = make_uint2(w[0], w[1]);
        }
        if (tid == 0) s_factor[j % (2 * SCALE_STAGES)] = make_float2(__int_as_float((127 + ex[0]) << 23), (float)ex[1]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&mult_full[s]);
      }
    } else if (!FP16) {
      // ------------------------------ cleaning --------------------------------
      bool ok = true;
      const int tid = threadIdx.x - 64;
      uint32_t told = 0;                        // phase of every stage's v_dirty
      for (int j = 0; j < n && ok; ++j) {
        if (!dirty(j)) continue;
        const int s = j % CV_STAGES, k0 = (j0 + j) * BK;
        // v_full alone would not do: its phases go on while these warps pass over tiles that are read whole
        ok = mbar_wait_warp(&v_dirty[s], (told >> s) & 1, abort_flag, args.status, 3);
        told ^= 1u << s;
        if (ok) ok = mbar_wait_warp(&v_full[s], (j / CV_STAGES) & 1, abort_flag, args.status, 3);
        // eight loads at a time, or a store in between holds the next load up: 5 -> 2 us for a last tile
        uint8_t* at = sV + s * CTILE + ((tid & 15) >> 3) * CHALF;
#pragma unroll 1
        for (int i = 0; i < 32; i += 8) {
          uint4 x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const uint4*>(at + swz128_offset((i + u) * 4 + (tid >> 4), tid & 7));
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&x[u]);
            constexpr uint32_t ex = 0x7f80u;         // an exponent of all ones
            // the upper bit of a half is set where its exponent is all ones
            uint32_t bad = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= ((w[e] & (ex | ex << 16)) + 0x00800080u) & 0x80008000u;
            if (bad) {
              const int key = (i + u) * 4 + (tid >> 4);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] &= ((w[e] & ex) == ex ? 0xffff0000u : 0xffffffffu) & ((w[e] & ex << 16) == ex << 16 ? 0xffffu : 0xffffffffu);
              *reinterpret_cast<uint4*>(at + swz128_offset(key, tid & 7)) = x[u];
              if (k0 + key < kv_len) atomicMin(poison, k0 + key);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_clean[s]);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    if (RAW && warp >= 12) {
      // ------------------------------ widening --------------------------------
      // Four warps widen keys, four values; a thread has a row: code times scale, three instructions per pair.
      const int row = threadIdx.x & 127, kv = (warp - 12) >> 2, sw = (row & 7) << 4;
      const int stages = kv ? CV_STAGES : CK_STAGES;
      uint64_t *const free = kv ? v_empty : k_empty, *const done = kv ? v_full : k_full;
      uint8_t* const tiles = (kv ? sV : sK) + row * 128;
      bool ok = true;
      for (int j = 0; j < n && ok; ++j) {
        const int u = 2 * j + kv, w = u % (2 * RAW_STAGES), to = j % stages;
        ok = mbar_wait_warp(&mult_full[j % SCALE_STAGES], (j / SCALE_STAGES) & 1, abort_flag, args.status, 3) &&
             mbar_wait_warp(&raw_full[w], (u / (2 * RAW_STAGES)) & 1, abort_flag, args.status, 3);
        if (!ok) break;
        const uint32_t f = s_mult[(j % SCALE_STAGES) * 256 + kv * 128 + row];
        const uint8_t* from = s_raw + u % RAW_STAGES * RAW_UNIT + row * 128;
        uint4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const uint4*>(from + ((i << 4) ^ sw));
        __syncwarp();
        if (lane == 0) mbar_arrive(&raw_empty[w]);
        if (__any_sync(0xffffffffu, f == CLEAR_ROW)) {      // (their codes may be NaN)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (f == CLEAR_ROW) x[i] = make_uint4(0, 0, 0, 0);
        }
        const uint32_t hi = __byte_perm(f, f, 0x1010), lo = __byte_perm(f, f, 0x3232);
        ok = mbar_wait_warp(&free[to], ((j / stages) & 1) ^ 1, abort_flag, args.status, 3);
        if (!ok) break;
        uint8_t* dst = tiles + to * CTILE;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint2 y0 = widen_scaled(i & 1 ? x[i >> 1].z : x[i >> 1].x, hi, lo), y1 = widen_scaled(i & 1 ? x[i >> 1].w : x[i >> 1].y, hi, lo);
          *reinterpret_cast<uint4*>(dst + (i >> 3) * CHALF + (((i & 7) << 4) ^ sw)) = make_uint4(y0.x, y0.y, y1.x, y1.y);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&done[to]);
      }
    } else {
    // ------------------------------ softmax --------------------------------
    // A warp owns 16 rows; its threads hold columns 2 (lane % 4) + 8 i + {0, 1} of rows lane / 4 and lane / 4 + 8.
    const int t = (warp - 4) >> 3;
    const int base = (warp & 3) * 32 + ((warp - 4) >> 2 & 1) * 16;
    const int q2 = (lane & 3) * 2;
    const uint32_t lane_sel = (uint32_t)base << 16;
    const uint32_t tmem_S = tmem_base + t * 128 + lane_sel;
    const uint32_t tmem_O = tmem_base + 256 + t * 128 + lane_sel;
    const uint32_t tmem_P = tmem_base + (t ^ 1) * 128 + lane_sel;   // over the other tile's scores
    uint8_t* sOt = sQ + t * CTILE;
    int lim[2];          // -1: no row of this sequence
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = base + (lane >> 2) + 8 * r, token = token0 + t * T + row / G;
      lim[r] = row < T * G && token < q_len ? row_limit(p, q0, q_len, kv_len, token) : -1;
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};      // running maximum, log2 units
    float sc[2] = {args.scale_log2, args.scale_log2};
    bool ok = true;
    if (FP16 && n > 0) {
      // This warp's 16 query rows to fp16, each times the power of two that brings its largest value to [2^13, 2^14): a value
      // loses 2^-38 of its row's largest at most.  (One power of two for all of them would let a large row take its neighbours' bits.)
      ok &= mbar_wait(q_full, 0, abort_flag, args.status, 5);
      __syncwarp();
      uint8_t* at = sOt + ((lane & 15) >> 3) * CHALF;
      uint4 u[8];                            // 16 lanes have a row: 2 i + lane / 16
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = *reinterpret_cast<const uint4*>(at + swz128_offset(base + 2 * i + (lane >> 4), lane & 7));
      const int mine = (min(token0 + (t + 1) * T, q_len) - (token0 + t * T)) * G - base;     // rows of this warp that are somebody's
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (2 * i + (lane >> 4) >= mine) u[i] = make_uint4(0, 0, 0, 0);
        uint32_t top = max_u16x2(max_u16x2(u[i].x & 0x7fff7fffu, u[i].y & 0x7fff7fffu), max_u16x2(u[i].z & 0x7fff7fffu, u[i].w & 0x7fff7fffu));
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) top = max_u16x2(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = max(top << 16, top & 0xffff0000u);
        const int e = (int)(top >> 23) - 127;                    // of the largest value; zero and what is not finite: as it is
        const int up = top == 0 || e == 128 ? 0 : min(13 - e, 120);
        const float f = __int_as_float((127 + up) << 23);
        const uint64_t f2 = pack_f32x2(f, f);
        uint32_t* w = reinterpret_cast<uint32_t*>(&u[i]);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          float x, y;
          unpack_f32x2(mul_f32x2(bf16x2_to_f32x2(w[h]), f2), x, y);
          w[h] = pack_f16x2(x, y);
        }
        *reinterpret_cast<uint4*>(at + swz128_offset(base + 2 * i + (lane >> 4), lane & 7)) = u[i];
        // to the threads that hold this row's scores: rows lane / 4 and lane / 4 + 8
        const float back = __shfl_sync(0xffffffffu, __int_as_float((127 - up) << 23), (lane & 4) << 2);
        if ((i & 3) == lane >> 3) sc[i >> 2] = args.scale_log2 * back;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    }
    const float4* factors = MODE == kWide ? args.factors + (long long)(args.first_page[b] + j0) * args.heads + kvh : nullptr;
    int bad = 0x7fffffff;                   // first key whose value is not finite
    const int mine = t ? n_b : n_a, full = t ? full_b : full_a;
    for (int j = 0; j < mine; ++j) {        // all tiles also after a time-out, see mbar_wait_warp
      float4 factor = make_float4(1.f, 0.f, 0.f, 0.f);      // of this tile's keys and values
      if (MODE == kWide) {
        factor = __ldg(factors + (long long)j * args.heads);
        bad = min(bad, __float_as_int(factor.z));
      }
      ok &= mbar_wait(&s_full[t], j & 1, abort_flag, args.status, 5);
      tc_fence_after();
      if (RAW) {                             // told before the keys were; the place is used again eight tiles on
        const float2 told = s_factor[j % (2 * SCALE_STAGES)];
        factor.x = told.x;
        factor.y = told.y;
      }
      float sv[2][32];   // [columns 0-63, 64-127][4 i + 2 row + e]
      {
        uint32_t r0[32], r1[32];
        tmem_ld_16x256b_x8(tmem_S, r0);
        tmem_ld_16x256b_x8(tmem_S + 64, r1);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          sv[0][c] = __uint_as_float(r0[c]);
          sv[1][c] = __uint_as_float(r1[c]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&s_empty[t]);
        if (TILES > 1) tally_add(&drained[t]);
      }
      if (j >= full) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int end = lim[r] - (j0 + j) * BK - q2;       // columns 8 i + e from here on are hidden
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (h * 64 + i * 8 + e >= end) sv[h][4 * i + 2 * r + e] = -INFINITY;
        }
      }
      float mx[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float m0 = fmaxf(sv[0][2 * r], sv[0][2 * r + 1]), m1 = fmaxf(sv[1][2 * r], sv[1][2 * r + 1]);
#pragma unroll
        for (int i = 1; i < 8; ++i) {
          m0 = max3(m0, sv[0][4 * i + 2 * r], sv[0][4 * i + 2 * r + 1]);
          m1 = max3(m1, sv[1][4 * i + 2 * r], sv[1][4 * i + 2 * r + 1]);
        }
        mx[r] = lim[r] < 0 ? -INFINITY : fmaxf(m0, m1);      // what other rows hold decides nothing here
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      }
      // the running maximum moves only when it is outgrown by more than 2^8, see attn_infer_sm100.cu
      float f[2];                            // scores in log2 units: s f
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        // (not 0, or a hidden score, -inf, would be NaN.  Sums are up to 2^34: where the factor is raised, all scores are below 2^-92.)
        f[r] = FP16 ? fmaxf(sc[r] * factor.x, FLT_MIN) : sc[r];
        mx[r] = FP16 ? fmaf(mx[r], f[r], factor.y) : mx[r] * f[r];
      }
      const bool rescale = __any_sync(0xffffffffu, mx[0] > m[0] + 8.f || mx[1] > m[1] + 8.f);
      float alpha[2];
      uint64_t nb2[2], sc2[2], acc[2][2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float m_new = rescale ? fmaxf(m[r], mx[r]) : m[r];
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        alpha[r] = rescale ? fast_exp2(m[r] - m_use) : 1.f;
        m[r] = m_new;
        const float nb = FP16 ? factor.y + P_TOP - m_use : -m_use;
        nb2[r] = pack_f32x2(nb, nb);
        sc2[r] = pack_f32x2(f[r], f[r]);
        acc[r][0] = acc[r][1] = 0ull;
      }
      uint32_t pk[32];      // probabilities, bf16 pairs: [2 (8-column group) + row]
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float x, y;
            unpack_f32x2(fma_f32x2(pack_f32x2(sv[h][4 * i + 2 * r], sv[h][4 * i + 2 * r + 1]), sc2[r], nb2[r]), x, y);
            x = fast_exp2(x);
            y = fast_exp2(y);
            acc[r][i & 1] = add_f32x2(acc[r][i & 1], pack_f32x2(x, y));
            pk[16 * h + 2 * i + r] = FP16 ? pack_f16x2(x, y) : pack_bf16x2(x, y);
          }
      const float out_of = FP16 ? fast_exp2(-SUM_DOWN - factor.y) : 1.f;       // the sum is of probabilities, without the values' power of two
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float s0, s1;
        unpack_f32x2(add_f32x2(acc[r][0], acc[r][1]), s0, s1);
        l[r] = l[r] * alpha[r] + (s0 + s1) * out_of;      // of this thread's columns; summed over the four threads at the end
      }
      if (j > 0) ok &= mbar_wait(&pv_done[t], (j - 1) & 1, abort_flag, args.status, 5);
      // The other tile's warps have read the scores that P goes over: of the score tiles issued before PV_t(j), which are key tiles
      // 0 .. j of B for A, 0 .. j + 1 of A for B.
      if (TILES > 1) ok &= tally_wait(&drained[t ^ 1], 8 * (t == 0 ? min(j + 1, n_b) : min(j + 2, n_a)), abort_flag, args.status, 5);
      tc_fence_after();
      tmem_st_16x128b_x16(tmem_P, pk);
      if (j > 0 && rescale) {
        const uint64_t al0 = pack_f32x2(alpha[0], alpha[0]), al1 = pack_f32x2(alpha[1], alpha[1]);
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t r[32];
          tmem_ld_16x256b_x8(tmem_O + c * 64, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float y0, y1;
            unpack_f32x2(mul_f32x2(pack_f32x2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), (i & 2) ? al1 : al0),
                         y0, y1);
            r[i] = __float_as_uint(y0);
            r[i + 1] = __float_as_uint(y1);
          }
          tmem_st_16x256b_x8(tmem_O + c * 64, r);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
    }
    if (mine > 0) ok &= mbar_wait(&pv_done[t], (mine - 1) & 1, abort_flag, args.status, 5);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      tc_fence_after();
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (lim[r] > (MODE == kWide ? bad : *poison)) l[r] = __int_as_float(0x7fffffff);
      }
      // rows with scores whose rounding counts; infinite ones stay what they are
      uint32_t done = 0;                     // this warp's rows that are computed again
      {
        const bool far[2] = {lim[0] >= 0 && fabsf(m[0]) > FAR && fabsf(m[0]) < INFINITY, lim[1] >= 0 && fabsf(m[1]) > FAR && fabsf(m[1]) < INFINITY};
        const uint32_t f0 = __ballot_sync(0xffffffffu, far[0]), f1 = __ballot_sync(0xffffffffu, far[1]);
        if (f0 | f1) {
#pragma unroll 1
          for (int i = 0; i < 16; ++i) {
            if (((i < 8 ? f0 : f1) >> (i & 7) * 4 & 1) == 0) continue;
            const int r = base + i, row = q0 + token0 + t * T + r / G, head = kvh * G + r % G;
            const int end = __shfl_sync(0xffffffffu, i < 8 ? lim[0] : lim[1], (i & 7) * 4);
            float4 x;
            float2 ml;
            far_row<FP16>(p, args, b, row, head, kvh, j0 * BK, min(end, (j0 + mine) * BK), &x, &ml);
            if (item.w < 0) {
              const float inv = ml.y == 0.f ? 0.f : 1.f / ml.y;
              *reinterpret_cast<uint2*>(args.o + row * args.ldo + head * HEAD + lane * 4) =
                  make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
            } else {
              const long long at = ((long long)item.w + t * T * G + r) * args.heads + kvh;
              *reinterpret_cast<float4*>(args.part + at * HEAD + lane * 4) = x;
              if (lane == 0) args.part_ml[at] = ml;
            }
            done |= 1u << i;
          }
        }
      }
      const float down = FP16 ? 1.f / 4096.f : 1.f;      // as the sums: SUM_DOWN
      if (item.w < 0) {
        // Output rows leave through this warp's rows of the row tile's buffer (no product reads it any more), so that 16
        // lanes store one row's 256 bytes.
        const uint32_t st_row = smem_u32(sOt) + (base + ((lane >> 3) & 1) * 8 + (lane & 7)) * 128;
        const uint32_t st_chunk = (uint32_t)((lane >> 4) ^ (lane & 7)) << 4;
        const float inv[2] = {l[0] == 0.f ? 0.f : 1.f / l[0], l[1] == 0.f ? 0.f : 1.f / l[1]};
        if (mine > 0) {
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            uint32_t r[32];
            tmem_ld_16x256b_x8(tmem_O + h * 64, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = pack_bf16x2(down * __uint_as_float(r[4 * i + 2 * e]) * inv[e & 1], down * __uint_as_float(r[4 * i + 2 * e + 1]) * inv[e & 1]);
              stmatrix_x4(st_row + h * CHALF + (st_chunk ^ (i << 4)), w[0], w[1], w[2], w[3]);
            }
          }
          __syncwarp();
        }
        const uint32_t per = 65536u / G + 1;               // r / G = r per >> 16 for r < 128
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = base + 2 * i + (lane >> 4), c = lane & 15, of = r * per >> 16, token = token0 + t * T + of;
          if (r < T * G && token < q_len && (done >> (r - base) & 1) == 0)
            *reinterpret_cast<uint4*>(args.o + (long long)(q0 + token) * args.ldo + (long long)(kvh * G + r - of * G) * HEAD + c * 8) =
                mine > 0 ? *reinterpret_cast<const uint4*>(sOt + (c >> 3) * CHALF + swz128_offset(r, c & 7)) : make_uint4(0, 0, 0, 0);
        }
      } else {
        const long long at0 = ((long long)item.w + t * T * G + base + (lane >> 2)) * args.heads + kvh;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
          if (mine > 0) {
            tmem_ld_16x256b_x8(tmem_O + h * 64, r);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = 0;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (lim[e] >= 0 && (done >> (lane >> 2) + 8 * e & 1) == 0) {
              float* dst = args.part + (at0 + 8ll * e * args.heads) * HEAD + h * 64 + q2;
#pragma unroll
              for (int i = 0; i < 8; ++i)
                *reinterpret_cast<float2*>(dst + i * 8) = make_float2(down * __uint_as_float(r[4 * i + 2 * e]), down * __uint_as_float(r[4 * i + 2 * e + 1]));
            }
          __syncwarp();
        }
        if ((lane & 3) == 0) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (lim[e] >= 0 && (done >> (lane >> 2) + 8 * e & 1) == 0)        // scores that were all NaN are not to be taken for no keys at all
              args.part_ml[at0 + 8ll * e * args.heads] = make_float2(m[e] == -INFINITY && l[e] != l[e] ? 0.f : FP16 ? m[e] - P_TOP + SUM_DOWN : m[e], l[e]);
        }
      }
    }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    if (*abort_flag) {
      uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 2000000ull) {
      }
    }
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int MODE>
static int launch_chunks(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const Plan& p, const ChunkArgs& a,
                         int items, cudaStream_t st) {
  int dev = 0;
  SNU1_CUDA_CHECK(cudaGetDevice(&dev));
  static std::once_flag once[64];
  cudaError_t err = cudaSuccess;
  std::call_once(once[dev & 63], [&]() {
    err = cudaFuncSetAttribute(paged_chunk_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Chunk<MODE>::SMEM);
  });
  SNU1_CUDA_CHECK(err);
  SNU1_CUDA_CHECK(launch_pdl(paged_chunk_kernel<MODE>, dim3(a.heads * items), dim3(CHUNK_THREADS), Chunk<MODE>::SMEM, st, tm_q, tm_k, tm_v, p, a));
  return kHostOk;
}

int launch_chunks(const Cache& c, const Plan& p, const void* q, long long ldq, void* o, long long ldo, float* part, float2* part_ml,
                  float scale_log2, void* wide, const float4* factors, cudaStream_t st) {
  const int G = p.group, T = 128 / G;
  CUtensorMap tm_q, tm_k, tm_v;
  int rc;
  {
    const uint64_t dims[3] = {128, (uint64_t)c.heads * G, (uint64_t)p.rows}, str[2] = {256, (uint64_t)ldq * 2};
    const uint32_t box[3] = {64, (uint32_t)G, (uint32_t)T};
    if ((rc = encode_tmap(&tm_q, TmapType::kBf16, true, q, 3, dims, str, box)) != kHostOk) return rc;
  }
  ChunkArgs a;
  a.first_page = nullptr;
  a.factors = nullptr;
  a.page = c.page;
  a.pages = c.pages;
  a.q = (const __nv_bfloat16*)q;
  a.ldq = ldq;
  a.data = (const uint8_t*)c.data;
  a.scales = c.scales;
  a.cache_pages = c.pages;
  a.o = (__nv_bfloat16*)o;
  a.ldo = ldo;
  a.part = part;
  a.part_ml = part_ml;
  a.heads = c.heads;
  a.scale_log2 = scale_log2;
  a.status = device_status_word();
  if (p.one_count > 0) {
    a.items = p.one;
    if ((rc = launch_chunks<kRaw>(tm_q, c.k, c.scale, p, a, p.one_count, st)) != kHostOk) return rc;
  }
  if (p.chunk_count == 0) return kHostOk;
  a.items = p.chunk;
  if (!c.fp8) return launch_chunks<kPages>(tm_q, c.k, c.v, p, a, p.chunk_count, st);
  const uint64_t dims[4] = {128, 128, (uint64_t)c.heads, (uint64_t)p.unpack_count};
  const uint64_t str[3] = {256, 256 * 128, 256ull * 128 * c.heads * 2};
  const uint32_t box[4] = {64, 128, 1, 1};
  if ((rc = encode_tmap(&tm_k, TmapType::kBf16, true, wide, 4, dims, str, box)) != kHostOk) return rc;
  if ((rc = encode_tmap(&tm_v, TmapType::kBf16, true, (uint8_t*)wide + 256ull * 128 * c.heads, 4, dims, str, box)) != kHostOk) return rc;
  a.factors = factors;
  a.first_page = p.unpack_first;
  a.page = 128;
  a.pages = p.unpack_count;
  return launch_chunks<kWide>(tm_q, tm_k, tm_v, p, a, p.chunk_count, st);
}

}  // namespace paged
}  // namespace snu1
