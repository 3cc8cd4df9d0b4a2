// Attention of many sequences' few new rows to the tokens that all of them share, over a paged cache: the first part of a row's
// keys, read once for the whole run of sequences.  The rest of the keys is each sequence's own (attn_paged.cu, TAIL); both leave unnormalised results
// (maximum, sum, weighted values, fp32) that paged_share_join_kernel puts together.
//
//   S^T = K q^T,   p = exp2(S^T - m),   o^T = V^T p^T
//
// The rows of a run are its new tokens times the query heads of the group, up to 64 per CTA.  They are the N of both products
// (tcgen05.mma, accumulators in tensor memory), the 128 keys of a tile (the 128 values of a head) the M: eight rows cost an eighth of 64,
// where rows as the M would fill 128 lanes whatever their number.  A thread of the softmax has one key and a column per row, so the
// maximum over keys lies across lanes; it moves only when it is outgrown (by 2^8), and a vote per tile is all that costs.  Sums stay
// with the threads until the end.
//
// e4m3 codes go to the first product as they are; a query is two e4m3 numbers, each row times a power of two: hi has 4 of the 8 bits
// of bf16, lo the others, 16 times as large, as 64 more columns.  A value of less than 2^-14 of its row's largest loses bits below 2^-22 of it.  A key's scale
// is a number of the thread's.  For the second product four warps widen codes to fp16, which is exact; a value's scale goes into its probability, times a
// power of two per row that keeps the largest product at 2^7 to 2^15.  bf16: probabilities are two bf16 numbers, hi and lo as 64 columns each.
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
  static constexpr int TILE = PK * HEAD * (FP8 ? 1 : 2), WIDE = PK * HEAD * 2, Q = 16384, P = FP8 ? PK * PR * 2 : 2 * PK * PR * 2;
  static constexpr int SMEM = Q + (K_STAGES + V_STAGES) * TILE + (FP8 ? W_STAGES * WIDE : 0) + P_STAGES * P + 1024;
  static constexpr int COLS = FP8 ? 512 : 256;  // of tensor memory: scores twice, output
  static constexpr int S_COLS = FP8 ? 2 * PR : PR, O_AT = 2 * S_COLS;
};

struct PrefixArgs {
  const __nv_bfloat16* q;
  long long ldq;
  float* part;
  float2* part_ml;
  const float* scales;
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
// largest of a warp's; -inf if all are NaN
__device__ __forceinline__ float warp_max(float x) {
  const uint32_t b = __float_as_uint(x), k = x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
  const uint32_t m = __reduce_max_sync(0xffffffffu, k);
  return m == 0 ? -INFINITY : __uint_as_float(m & 0x80000000u ? m & 0x7fffffffu : ~m);
}

// What the softmax knows of a row; column n.
struct RowState {
  float m;           // running maximum, log2 units; 0 as long as there is none
  float rs;          // a score's factor
  float move;        // a score relative to m that is larger moves the maximum: 8, or -inf as long as there is none
  float move_value;  // e4m3: one that is larger with log2 of its value's scale added does so too
};

template <bool FP8>
__global__ void __launch_bounds__(Prefix<FP8>::THREADS, 1)
    paged_prefix_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Plan p,
                        const __grid_constant__ PrefixArgs args) {
  using F = Prefix<FP8>;
  constexpr int KS = F::K_STAGES, VS = F::V_STAGES, WS = F::W_STAGES, PS = F::P_STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;                            // e4m3: [hi 64, lo 64][128]; bf16: [half of the values][64][64]
  uint8_t* sK = sQ + F::Q;
  uint8_t* sV = sK + KS * F::TILE;
  uint8_t* sP = sV + VS * F::TILE;               // [key][64 rows] fp16; bf16: hi, then lo
  uint8_t* sW = sP + PS * F::P;                  // e4m3: widened values, [half][key][64]
  __shared__ uint64_t q_ready, k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], w_full[WS], w_empty[WS], s_full[2], s_empty[2], p_full[PS], pv_done[PS];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word, s_poison;
  __shared__ int s_lim[PR], s_most, s_least;
  __shared__ RowState s_row[PR];
  __shared__ float s_by[PR], s_f[PR], s_fo[PR], s_mv[PR];
  __shared__ int s_ec[PR];                       // e4m3: exponent of a row's factor of p times the value's scale
  __shared__ float s_red[8][32], s_red2[8][32], s_sum[8][32];
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
    for (int i = 0; i < PS; ++i) {
      mbar_init(&p_full[i], 4 * sides);
      mbar_init(&pv_done[i], 1);
    }
    abort_word = 0;
    s_poison = 0x7fffffff;
    s_most = 0;
    s_least = 0x7fffffff;
    mbar_fence_init();
    tma_prefetch_desc(&tm_k);
    if (!FP8) tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, F::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  if (!args.beside) pdl_wait();
  pdl_trigger();
  // column of row r: 8 (r / 8 / 2) + r % 8 of the half that its set of warps has
  if (tid < PR) {
    const int col = (tid >> 3 & 1) * 32 + (tid >> 4) * 8 + (tid & 7);
    int lim = 0;
    if (tid < rows) {
      const int t = t0 + (row0 + tid) / G, b = p.row_seq[t], q0 = p.q_start[b];
      lim = min(shared, row_limit(p, q0, p.q_start[b + 1] - q0, seq_len(p, b), t - q0));
      atomicMax(&s_most, lim);
      atomicMin(&s_least, lim);
    }
    s_lim[col] = lim;
  }
  __syncthreads();
  const int most = s_most, least = s_least;
  const int all = (most + PK - 1) / PK;
  const int j0 = (int)((long long)all * part / parts), n_tiles = (int)((long long)all * (part + 1) / parts) - j0;
  const int* table = p.table + (long long)run.z * p.width;

  if (warp == 0) {
    // ------------------------------ pages --------------------------------
    const int page = p.page, per = PK / page, used = (most + page - 1) / page;
    auto page_of = [&](int n) -> int {
      const int i = (j0 + n) * per + lane;
      return n < n_tiles && lane < per && i < used ? table[i] : 0;
    };
    int pg = page_of(0);
    for (int n = 0; n < n_tiles; ++n) {
      const int next = page_of(n + 1), live = min(per, used - (j0 + n) * per);
      if (lane < live && (pg < 0 || pg >= args.pages)) report_status(args.status, kBadPage, 10);     // reads as zeros
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int stages = kv ? VS : KS, s = n % stages;
        uint64_t *const full = kv ? &v_full[s] : &k_full[s], *const empty = kv ? &v_empty[s] : &k_empty[s];
        uint8_t* dst = (kv ? sV : sK) + s * F::TILE + lane * page * 128;
        if (!mbar_wait_warp(empty, ((n / stages) & 1) ^ 1, abort_flag, args.status, 1)) {
          n = n_tiles;
          break;
        }
        if (lane == 0) mbar_expect_tx(full, live * page * (FP8 ? 128 : 256));
        __syncwarp();
        if (lane < live) {
          if (FP8) {
            tma_load_5d(smem_u32(dst), &tm_k, full, 0, 0, head, kv, pg);
          } else {
            tma_load_4d(dst, kv ? &tm_v : &tm_k, full, 0, 0, head, pg);
            tma_load_4d(dst + PK * 128, kv ? &tm_v : &tm_k, full, 64, 0, head, pg);
          }
        }
        __syncwarp();
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
      if (FP8) ok &= mbar_wait(&w_full[n % WS], (n / WS) & 1, abort_flag, args.status, 3);
      else ok &= mbar_wait(&v_full[n % VS], (n / VS) & 1, abort_flag, args.status, 3);
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
  } else if (warp >= 4) {
    // ------------------------------ softmax --------------------------------
    const int w = warp - 4, side = w >> 2, c0 = side * 32, active = (groups + 1 - side) >> 1;      // groups of eight columns from c0 on
    const int in_tile = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    bool ok = true;
    {
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
      float rs = args.scale_log2;
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
        rs = e == 128 ? __int_as_float(0x7fffffff) : rs * __int_as_float((127 - up) << 23);      // not finite: NaN
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
        s_row[col] = RowState{0.f, rs, -INFINITY, -INFINITY};
        s_ec[col] = 0;
        s_mv[col] = -INFINITY;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready);
      named_bar_sync(1, 256);
    }
    if (active > 0 && n_tiles > 0) {
      // e4m3: scales of this thread's key and value, read a tile ahead
      auto scales_of = [&](int n) -> float2 {
        const int key = (j0 + n) * PK + in_tile;
        float2 x = make_float2(0.f, 0.f);
        if (n < n_tiles && key < most) {
          const int pg = table[key / p.page];
          if (pg >= 0 && pg < args.pages) {
            const float* at = args.scales + ((long long)pg * 2 * args.heads + head) * p.page + key % p.page;
            x = make_float2(at[0], at[(long long)args.heads * p.page]);
          }
        }
        return x;
      };
      float x[32], l[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) l[i] = 0.f;
      float2 sc = FP8 ? scales_of(0) : make_float2(1.f, 1.f);
      for (int n = 0; n < n_tiles; ++n) {        // all tiles also after a time-out
        const int k0 = (j0 + n) * PK, key = k0 + in_tile;
        const bool dirty = k0 + PK > least;      // some row may not read all of it
        const float2 next = FP8 ? scales_of(n + 1) : sc;
        const float lv = FP8 ? log2_of(sc.y) : 0.f;
        ok &= mbar_wait(&s_full[n & 1], (n >> 1) & 1, abort_flag, args.status, 5);
        __syncwarp();
        tc_fence_after();
        const uint32_t S = tmem + (n & 1) * F::S_COLS + c0 + lanes;
        bool move = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i >= active) break;
          uint32_t h[8], lo[8];
          tmem_ld_x8(S + 8 * i, h);
          if (FP8) tmem_ld_x8(S + PR + 8 * i, lo);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const RowState r = s_row[c0 + 8 * i + e];
            const float s = FP8 ? fmaf(__uint_as_float(lo[e]), 0.0625f, __uint_as_float(h[e])) : __uint_as_float(h[e]);
            float y = __fmul_rn(s, FP8 ? r.rs * sc.x : r.rs);      // (never fused with the difference)
            if (dirty && key >= s_lim[c0 + 8 * i + e]) y = -INFINITY;
            y -= r.m;
            move |= y > r.move || (FP8 && y + lv > r.move_value);
            x[8 * i + e] = y;
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[n & 1]);
        if (named_bar_any(2 + side, 128, move)) {
          // the maximum moves (the first tile, and seldom after it)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i >= active) break;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float a = warp_max(x[8 * i + e]), b = FP8 ? warp_max(x[8 * i + e] + lv) : 0.f;
              if (lane == 0) {
                s_red[w][8 * i + e] = a;
                s_red2[w][8 * i + e] = b;
              }
            }
          }
          named_bar_sync(2 + side, 128);
          if ((w & 3) == 0 && lane < 8 * active) {
            const int col = c0 + lane;
            RowState r = s_row[col];
            float top = -INFINITY, topv = -INFINITY;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              top = fmaxf(top, s_red[side * 4 + k][lane]);
              topv = fmaxf(topv, s_red2[side * 4 + k][lane]);
            }
            const bool fresh = r.move == -INFINITY, none = fresh && top == -INFINITY;
            const float by = none ? 0.f : fresh ? top : fmaxf(top, 0.f);
            r.m += by;
            if (!none) r.move = 8.f;
            s_by[col] = by;
            s_f[col] = fresh ? 0.f : fast_exp2(-by);
            if (FP8) {
              const float mv = fmaxf(s_mv[col], topv) - by;
              const int was = s_ec[col], ec = mv == -INFINITY ? was : max(-120, min(120, (int)floorf(P_TOP - mv)));
              s_mv[col] = mv;
              s_ec[col] = ec;
              r.move_value = mv == -INFINITY ? -INFINITY : P_TOP + 8.f - (float)ec;
              s_fo[col] = fresh ? 0.f : exp2f(-by + (float)(ec - was));
            }
            s_row[col] = r;
          }
          named_bar_sync(2 + side, 128);
          if (n > 0) {
            ok &= mbar_wait(&pv_done[(n - 1) % PS], ((n - 1) / PS) & 1, abort_flag, args.status, 6);
            __syncwarp();
            tc_fence_after();
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i >= active) break;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              x[8 * i + e] -= s_by[c0 + 8 * i + e];
              l[8 * i + e] *= s_f[c0 + 8 * i + e];
            }
            if (n > 0) {
#pragma unroll
              for (int half = 0; half < (FP8 ? 1 : 2); ++half) {
                const uint32_t at = tmem + F::O_AT + half * PR + c0 + 8 * i + lanes;
                uint32_t o[8];
                tmem_ld_x8(at, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * (FP8 ? s_fo : s_f)[c0 + 8 * i + e]);
                tmem_st_x8(at, o);
              }
            }
          }
          tmem_st_wait();
          tc_fence_before();
        }
        if (!FP8 && dirty) {
          // values that some row may not read: what nobody may and what is not finite is cleared, see attn_paged.cu
          ok &= mbar_wait(&v_full[n % VS], (n / VS) & 1, abort_flag, args.status, 5);
          uint8_t* tile = sV + (n % VS) * F::TILE;
          for (int i = tid - 128; i < PK * 16; i += 128 * sides) {
            const int k = i >> 4;
            uint4* at = reinterpret_cast<uint4*>(tile + ((i & 15) >> 3) * (PK * 128) + swz128_offset(k, i & 7));
            uint4 v = *at;
            uint32_t* u = reinterpret_cast<uint32_t*>(&v);
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool a = (u[e] & 0x7f80u) == 0x7f80u, b = (u[e] & 0x7f800000u) == 0x7f800000u;
              bad |= a || b;
              u[e] &= (a ? 0xffff0000u : 0xffffffffu) & (b ? 0xffffu : 0xffffffffu);
            }
            if (k0 + k >= most) {
              *at = make_uint4(0, 0, 0, 0);
            } else if (bad) {
              *at = v;
              atomicMin(&s_poison, k0 + k);
            }
          }
        }
        if (n >= PS) {
          ok &= mbar_wait(&pv_done[n % PS], ((n - PS) / PS) & 1, abort_flag, args.status, 6);
          __syncwarp();
        }
        uint8_t* P = sP + (n % PS) * F::P;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i >= active) break;
          uint32_t u[4], v[4];
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            float y[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int r = 8 * i + e + k;
              y[k] = fast_exp2(x[r]);
              l[r] += y[k];
              // (the scale of a key that is hidden may be anything)
              if (FP8) y[k] = dirty && x[r] == -INFINITY ? 0.f : y[k] * (sc.y * __int_as_float((127 + s_ec[c0 + r]) << 23));
            }
            if (FP8) {
              u[e >> 1] = pack_f16x2(y[0], y[1]);
            } else {
              u[e >> 1] = pack_bf16x2(y[0], y[1]);
              v[e >> 1] = pack_bf16x2(y[0] - __uint_as_float(u[e >> 1] << 16), y[1] - __uint_as_float(u[e >> 1] & 0xffff0000u));
            }
          }
          const uint32_t at = swz128_offset(in_tile, side * 4 + i);
          *reinterpret_cast<uint4*>(P + at) = make_uint4(u[0], u[1], u[2], u[3]);
          if (!FP8) *reinterpret_cast<uint4*>(P + PK * 128 + at) = make_uint4(v[0], v[1], v[2], v[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[n % PS]);
        sc = next;
      }
      // sums over the keys' threads, then the output
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if (i >= 8 * active) break;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
        if (lane == 0) s_sum[w][i] = l[i];
      }
      ok &= mbar_wait(&pv_done[(n_tiles - 1) % PS], ((n_tiles - 1) / PS) & 1, abort_flag, args.status, 6);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
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
          if (r < rows && ok)
            args.part[((long long)(item.w + r) * args.heads + head) * HEAD + in_tile] =
                FP8 ? __uint_as_float(h[e]) * __int_as_float((127 - s_ec[col]) << 23) : __uint_as_float(h[e]) + __uint_as_float(lo[e]);
        }
      }
    }
    if ((w & 3) == 0 && lane < 8 * active) {
      const int col = c0 + lane, r = (2 * (lane >> 3) + side) * 8 + (lane & 7);
      float m = -INFINITY, l = 0.f;
      if (n_tiles > 0) {
        m = s_row[col].move == -INFINITY ? -INFINITY : s_row[col].m;
#pragma unroll
        for (int k = 0; k < 4; ++k) l += s_sum[side * 4 + k][lane];
        if (!FP8 && s_lim[col] > *reinterpret_cast<volatile int*>(&s_poison)) l = __int_as_float(0x7fffffff);
        if (l != l && m == -INFINITY) m = 0.f;   // all NaN: not to be taken for no keys at all
      }
      if (r < rows) args.part_ml[(long long)(item.w + r) * args.heads + head] = make_float2(m, l);
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
  SNU1_CUDA_CHECK(launch_pdl(paged_prefix_kernel<FP8>, dim3(a.heads * p.prefix_count), dim3(Prefix<FP8>::THREADS), Prefix<FP8>::SMEM, st, c.k, c.v, p, a));
  return kHostOk;
}

int launch_prefix(const Cache& c, const Plan& p, const void* q, long long ldq, float* part, float2* part_ml, float scale_log2, int beside,
                  cudaStream_t st) {
  PrefixArgs a;
  a.q = (const __nv_bfloat16*)q;
  a.ldq = ldq;
  a.part = part;
  a.part_ml = part_ml;
  a.scales = c.scales;
  a.pages = c.pages;
  a.heads = c.heads;
  a.scale_log2 = scale_log2;
  a.beside = beside;
  a.status = device_status_word();
  return c.fp8 ? launch<true>(c, p, a, st) : launch<false>(c, p, a, st);
}

}  // namespace paged
}  // namespace snu1
