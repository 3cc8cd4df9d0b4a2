// Attention of a few new rows per key/value head over a paged cache: decode steps, drafted tokens, and the joining of
// partial results (also those of attn_paged_sm100.cu).
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp(scale q_r k_j - m_r),   j < limit_r
//
// The rows of a (sequence, key/value head) are its new tokens times the query heads of the group, up to 64 per CTA.  What
// bounds it is the stream of keys and values, so the work is split over keys: a work item is one part of a sequence, the
// parts are made as equal as they can be over the whole batch (ops/paged.py), and their unnormalised results (maximum, sum,
// weighted values, fp32) are joined by a second kernel in a fixed order, without atomics.
//
// One warp asks for whole pages through TMA (keys and values of one head in one box), several stages ahead; four warps
// compute with mma.sync m16n8k16: at 16 rows and up to 8 bytes of cache per clock and warp the legacy tensor path is far from
// its limit, and its fragments let e4m3 codes be widened to bf16 in registers (exactly, see e4m3x2_to_bf16x2): the scale
// of a key goes into its score, that of a value into its probability, both in fp32.  Up to 16 rows every warp takes other
// keys, up to 32 rows two warps share them, up to 64 rows all four do.
//
// Masked places: scores of keys at or beyond a row's limit are -inf whatever the cache holds.  A probability of zero does
// not hide an infinite or NaN value from the matrix product, so in a tile that some row may not read whole, bf16 values
// that are not finite are cleared in shared memory and the first key that held one is kept: rows that may read it give
// NaN, the others are as if it were not there.  (e4m3 codes are finite; what is not finite there is the row's scale, and that
// is only used where the mask allows.)
#include <string.h>

#include <mutex>

#include "host_common.h"
#include "paged.cuh"

namespace snu1 {
namespace paged {

constexpr int KT = 64;                       // keys of a stage
constexpr int FEW_THREADS = 160;             // four warps that compute, one that asks for pages

template <bool FP8>
struct Few {
  static constexpr int HALVES = FP8 ? 1 : 2;                    // boxes of 128 bytes per row
  static constexpr int DATA = KT * 2 * 128 * HALVES;            // keys and values of a stage
  static constexpr int STAGE = DATA + (FP8 ? KT * 2 * 4 : 0);
  static constexpr int STAGES = FP8 ? 5 : 3;
  static constexpr int DATA_ALL = STAGES * DATA;
  static constexpr int SCALES_ALL = STAGES * (STAGE - DATA);
  static constexpr int SMEM = DATA_ALL + SCALES_ALL + 1024;
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
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct FewArgs {
  const __nv_bfloat16* q;
  __nv_bfloat16* o;
  long long ldq, ldo;
  float* part;        // [partial rows][heads][128]
  float2* part_ml;    // [partial rows][heads] maximum (log2 units), sum
  int pages, heads;   // of the cache
  float scale_log2;
  int* status;
};

// WR: warps along the rows (16 each); the others take other keys.
template <bool FP8, int WR>
__global__ void __launch_bounds__(FEW_THREADS)
    paged_few_kernel(const __grid_constant__ CUtensorMap tm_kv, const __grid_constant__ CUtensorMap tm_scale, const Plan p,
                     const FewArgs a) {
  using F = Few<FP8>;
  constexpr int WK = 4 / WR, M = 16 * WR, NB = KT / 16 / WK;     // warps along the keys, rows, blocks of 16 keys per warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* s_scales = reinterpret_cast<float*>(smem + F::DATA_ALL);   // [stage][page box][keys, values][box rows]
  __shared__ uint64_t full[F::STAGES], empty[F::STAGES];
  __shared__ int abort_word, s_poison;
  __shared__ float s_m[4][16], s_l[4][16];
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < F::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    abort_word = 0;
    s_poison = 0x7fffffff;
    mbar_fence_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  const int4 item = p.few[blockIdx.x];
  const int b = item.x, row0 = item.y, part = item.z & 0xffff, parts = item.z >> 16;
  const int head = blockIdx.y, G = p.group;
  const int q0 = p.q_start[b], q_len = p.q_start[b + 1] - q0;
  const int kv_len = seq_len(p, b);
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
  const int tiles = (max_lim + KT - 1) / KT;
  const int j0 = (int)((long long)tiles * part / parts), j1 = (int)((long long)tiles * (part + 1) / parts);
  const int bx = min(p.page, KT), boxes = KT / bx;               // rows of a box, boxes of a stage
  const int box_bytes = 2 * bx * 128;

  if (warp == 4) {
    if (lane == 0) {
      bool gave_up = false;
      const int* table = p.table + (long long)b * p.width;
      const int pages_used = (max_lim + p.page - 1) / p.page;
      for (int j = j0; j < j1; ++j) {
        const int n = j - j0, s = n % F::STAGES;
        if (!mbar_wait(&empty[s], ((n / F::STAGES) & 1) ^ 1, abort_flag, a.status, 10)) {
          gave_up = true;
          break;
        }
        const int k0 = j * KT;
        int live = 0;
        for (int i = 0; i < boxes; ++i) live += (k0 + i * bx) / p.page < pages_used;
        mbar_expect_tx(&full[s], live * (box_bytes * F::HALVES + (FP8 ? bx * 8 : 0)));
        for (int i = 0; i < live; ++i) {
          const int k = k0 + i * bx;
          const int pg = table[k / p.page];
          if (pg < 0 || pg >= a.pages) report_status(a.status, kBadPage, 10);     // reads as zeros
#pragma unroll
          for (int h = 0; h < F::HALVES; ++h)
            tma_load_5d(smem_u32(smem + s * F::DATA + (i * F::HALVES + h) * box_bytes), &tm_kv, &full[s], h * 64, k % p.page, head,
                        0, pg);
          if (FP8)
            tma_load_4d(s_scales + (s * KT + i * bx) * 2, &tm_scale, &full[s], k % p.page, head, 0, pg);
        }
      }
      if (gave_up) {                       // copies may be on their way into this CTA's memory
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) {
        }
      }
    }
  } else {
    const int wr = warp / WK, wk = warp % WK;
    const int g = lane >> 2, c = lane & 3;
    // query fragments of rows g and g + 8 of this warp
    uint32_t qf[8][4];
    int lim[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = wr * 16 + g + r * 8;
      const bool on = row < rows;
      const int t = (row0 + row) / G;
      lim[r] = on ? row_limit(p, q0, q_len, kv_len, t) : 0;
      const __nv_bfloat16* qp = a.q + (long long)(q0 + t) * a.ldq + (long long)(head * G + (row0 + row) % G) * HEAD;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        // e4m3: a thread's four codes of a 16-value piece stand side by side, and so do its query values
        uint32_t lo = 0, hi = 0;
        if (on) {
          if (FP8) {
            const uint2 u = *reinterpret_cast<const uint2*>(qp + k * 16 + c * 4);
            lo = u.x;
            hi = u.y;
          } else {
            lo = *reinterpret_cast<const uint32_t*>(qp + k * 16 + c * 2);
            hi = *reinterpret_cast<const uint32_t*>(qp + k * 16 + c * 2 + 8);
          }
        }
        qf[k][r] = lo;
        qf[k][2 + r] = hi;
      }
    }
    float acc[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    bool ok = true;
    for (int j = j0; j < j1; ++j) {
      const int n = j - j0, s = n % F::STAGES, k0 = j * KT;
      ok &= mbar_wait(&full[s], (n / F::STAGES) & 1, abort_flag, a.status, 10);
      const uint32_t data = smem_u32(smem + s * F::DATA);
      const float* sc = s_scales + s * KT * 2;
      const bool partial = k0 + KT > min_lim;
      if (!FP8 && partial) {
        // values that are not finite, and rows that no box has filled
        for (int i = threadIdx.x; i < KT * 16; i += 128) {
          const int key = i >> 4, ch = i & 15;
          const int box = key / bx, row = key % bx;
          uint4* at = reinterpret_cast<uint4*>(smem + s * F::DATA + (box * 2 + (ch >> 3)) * box_bytes + bx * 128 +
                                               swz128_offset(row, ch & 7));
          if (k0 + key >= kv_len) {
            *at = make_uint4(0, 0, 0, 0);
          } else {
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
        named_bar_sync(1, 128);
      }
      float sv[NB][2][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int key0 = (wk * NB + nb) * 16, box = key0 / bx, brow = key0 % bx;
        const uint32_t kb = data + box * F::HALVES * box_bytes + brow * 128;
#pragma unroll
        for (int e = 0; e < 4; ++e) sv[nb][0][e] = sv[nb][1][e] = 0.f;
        if (FP8) {
          // matrices: keys 0-7 and 8-15 of a 16-byte piece, then of the next piece
          const int row = (lane & 7) + ((lane >> 3) & 1) * 8, pc = lane >> 4;
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            uint32_t r[4];
            ldsm_x4(kb + swz128_offset(row, k + pc), r);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                const uint32_t w = r[i * 2 + t];
                mma_bf16(sv[nb][t], qf[k + i], e4m3x2_to_bf16x2(__byte_perm(w, 0, 0x1404)), e4m3x2_to_bf16x2(__byte_perm(w, 0, 0x3424)));
              }
          }
        } else {
          // matrices: two pieces of keys 0-7, two of keys 8-15
          const int row = (lane & 7) + (lane >> 4) * 8, pc = (lane >> 3) & 1;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            uint32_t r[4];
            ldsm_x4(kb + (k >> 2) * box_bytes + swz128_offset(row, (k & 3) * 2 + pc), r);
            mma_bf16(sv[nb][0], qf[k], r[0], r[1]);
            mma_bf16(sv[nb][1], qf[k], r[2], r[3]);
          }
        }
      }
      // scores in log2 units, masked; the largest of a row
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int key = (wk * NB + nb) * 16 + t * 8 + c * 2;
          float f[2] = {a.scale_log2, a.scale_log2};
          if (FP8) {
            const float2 u = *reinterpret_cast<const float2*>(sc + (key / bx) * 2 * bx + key % bx);
            f[0] *= u.x;
            f[1] *= u.y;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = sv[nb][t][e] * f[e & 1];
            if (partial && k0 + key + (e & 1) >= lim[e >> 1]) x = -INFINITY;
            sv[nb][t][e] = x;
            mx[e >> 1] = fmaxf(mx[e >> 1], x);
          }
        }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      }
      // the running maximum moves only when it is outgrown by more than 2^8, see attn_infer_sm100.cu
      if (__any_sync(0xffffffffu, mx[0] > m[0] + 8.f || mx[1] > m[1] + 8.f)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float mn = fmaxf(m[r], mx[r]);
          const float f = m[r] == -INFINITY ? 0.f : fast_exp2(m[r] - mn);
          m[r] = mn;
          l[r] *= f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            acc[i][2 * r] *= f;
            acc[i][2 * r + 1] *= f;
          }
        }
      }
      const float mu[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        uint32_t pf[4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = fast_exp2(sv[nb][t][e] - mu[e >> 1]);
            l[e >> 1] += x[e];
          }
          if (FP8) {
            const int key = (wk * NB + nb) * 16 + t * 8 + c * 2;
            const float2 u = *reinterpret_cast<const float2*>(sc + (key / bx) * 2 * bx + bx + key % bx);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[e] *= (e & 1) ? u.y : u.x;
              if (partial && k0 + key + (e & 1) >= lim[e >> 1]) x[e] = 0.f;
            }
          }
          pf[t * 2] = pack_bf16x2(x[0], x[1]);
          pf[t * 2 + 1] = pack_bf16x2(x[2], x[3]);
        }
        const int key0 = (wk * NB + nb) * 16, box = key0 / bx, brow = key0 % bx;
        const uint32_t vb = data + box * F::HALVES * box_bytes + bx * 128 + brow * 128;
        const int row = (lane & 7) + ((lane >> 3) & 1) * 8, pc = lane >> 4;   // keys 0-7, 8-15 of a piece, then of the next
        if (FP8) {
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            uint32_t r[4];
            ldsm_x4_t(vb + swz128_offset(row, k + pc), r);
            // a thread has two values side by side of two keys: the even and the odd columns of a piece are two tiles
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t w0 = r[2 * i], w1 = r[2 * i + 1];
              mma_bf16(acc[2 * (k + i)], pf, e4m3x2_to_bf16x2((w0 << 8) & 0xff00ff00u), e4m3x2_to_bf16x2((w1 << 8) & 0xff00ff00u));
              mma_bf16(acc[2 * (k + i) + 1], pf, e4m3x2_to_bf16x2(w0 & 0xff00ff00u), e4m3x2_to_bf16x2(w1 & 0xff00ff00u));
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            uint32_t r[4];
            ldsm_x4_t(vb + (k >> 2) * box_bytes + swz128_offset(row, (k & 3) * 2 + pc), r);
            mma_bf16(acc[2 * k], pf, r[0], r[1]);
            mma_bf16(acc[2 * k + 1], pf, r[2], r[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
    ok = __all_sync(0xffffffffu, ok);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (l[r] != l[r] && m[r] == -INFINITY) m[r] = 0.f;         // scores that were all NaN: not to be taken for no keys at all
    }
    // Warps of the same rows meet in the ring: every stage has been read (a barrier below), and TMA asks for nothing more.
    named_bar_sync(1, 128);
    if (!FP8) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (lim[r] > s_poison) {
          l[r] = __int_as_float(0x7fffffff);
          m[r] = fmaxf(m[r], 0.f);
        }
    }
    float* ring = reinterpret_cast<float*>(smem);                // [warp][16][132]
    constexpr int LD = 132;
    if (c == 0) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        s_m[warp][g + 8 * r] = m[r];
        s_l[warp][g + 8 * r] = l[r];
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float* at = ring + (warp * 16 + g + 8 * r) * LD;
        if (FP8) {                         // columns 2 c, 2 c + 1 of an even / odd tile: values 4 c + {0, 2} / {1, 3} of a piece
          at[(i >> 1) * 16 + c * 4 + (i & 1)] = acc[i][2 * r];
          at[(i >> 1) * 16 + c * 4 + 2 + (i & 1)] = acc[i][2 * r + 1];
        } else {
          *reinterpret_cast<float2*>(at + i * 8 + c * 2) = make_float2(acc[i][2 * r], acc[i][2 * r + 1]);
        }
      }
    named_bar_sync(1, 128);
    const bool direct = item.w < 0;
    // a warp finishes one row at a time, four values per lane
    for (int row = warp; row < rows; row += 4) {
      const int w0 = row / 16 * WK, rr = row % 16;
      float mt = s_m[w0][rr];
#pragma unroll
      for (int w = 1; w < WK; ++w) mt = fmaxf(mt, s_m[w0 + w][rr]);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      float lt = 0.f;
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const float mw = s_m[w0 + w][rr];
        const float f = mw == -INFINITY ? 0.f : fast_exp2(mw - mt);
        const float4 y = *reinterpret_cast<const float4*>(ring + ((w0 + w) * 16 + rr) * LD + lane * 4);
        x.x += f * y.x;
        x.y += f * y.y;
        x.z += f * y.z;
        x.w += f * y.w;
        lt += mw == -INFINITY ? 0.f : f * s_l[w0 + w][rr];
      }
      if (!ok) continue;
      if (direct) {
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
  }
}

// Joins the parts of a row: one warp per (row, key/value head), four values per lane.
constexpr int MERGE_THREADS = 128;

__global__ void __launch_bounds__(MERGE_THREADS) paged_merge_kernel(const Plan p, const FewArgs a) {
  pdl_wait();
  pdl_trigger();
  const int4 e = p.merge[blockIdx.x];
  const int b = e.x, row0 = e.y, parts = e.z & 0xffff, rows = e.z >> 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.group;
  const int q0 = p.q_start[b], q_len = p.q_start[b + 1] - q0;
  const int w = blockIdx.y * (MERGE_THREADS / 32) + warp;
  const int row = w / a.heads, head = w % a.heads;
  if (row >= rows || row0 + row >= q_len * G) return;
  const long long step = (long long)rows * a.heads;
  const long long at = (long long)(e.w + row) * a.heads + head;
  float mt = -INFINITY;
  for (int s = lane; s < parts; s += 32) mt = fmaxf(mt, a.part_ml[at + s * step].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  float lt = 0.f;
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const float2 ml = a.part_ml[at + s * step];
    const float4 y = *reinterpret_cast<const float4*>(a.part + (at + s * step) * HEAD + lane * 4);
    const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - mt);
    x.x += f * y.x;
    x.y += f * y.y;
    x.z += f * y.z;
    x.w += f * y.w;
    lt += ml.x == -INFINITY ? 0.f : f * ml.y;
  }
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
  const int t = (row0 + row) / G;
  uint2 u;
  u.x = pack_bf16x2(x.x * inv, x.y * inv);
  u.y = pack_bf16x2(x.z * inv, x.w * inv);
  *reinterpret_cast<uint2*>(a.o + (long long)(q0 + t) * a.ldo + (long long)(head * G + (row0 + row) % G) * HEAD + lane * 4) = u;
}

template <bool FP8, int WR>
static int launch_few(const Cache& c, const Plan& p, const FewArgs& a, cudaStream_t st) {
  auto kernel = paged_few_kernel<FP8, WR>;
  int dev = 0;
  SNU1_CUDA_CHECK(cudaGetDevice(&dev));
  static std::once_flag once[64];
  cudaError_t err = cudaSuccess;
  std::call_once(once[dev & 63], [&]() {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<FP8>::SMEM);
  });
  SNU1_CUDA_CHECK(err);
  SNU1_CUDA_CHECK(launch_pdl(kernel, dim3(p.few_count, c.heads), dim3(FEW_THREADS), Few<FP8>::SMEM, st, c.kv, c.scale, p, a));
  return kHostOk;
}

}  // namespace paged
}  // namespace snu1

using namespace snu1;

// o_r = attention of row r over its sequence's first keys, rows [rows][heads of queries][128] bf16, ldq / ldo apart.
// scratch: partial results (partial_rows x heads x (128 values, maximum, sum) in fp32), then unpack_pages bf16 pages of 128 tokens.
SNU1_API int snu1_paged_attention(const void* cache, const void* plan, const void* q, long long ldq, void* o, long long ldo,
                                  float scale, void* scratch, void* stream) {
  using namespace paged;
  Cache c;
  Plan p;
  memcpy(&c, cache, sizeof(c));
  memcpy(&p, plan, sizeof(p));
  if (p.rows <= 0) return kHostOk;
  if (p.page != c.page || ldq % 8 || ldo % 8 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(scratch)) & 15) != 0) {
    set_last_error("paged_attention: rows must be 16-byte aligned, and the plan made for this page size");
    return kHostBadArg;
  }
  FewArgs a;
  a.q = (const __nv_bfloat16*)q;
  a.o = (__nv_bfloat16*)o;
  a.ldq = ldq;
  a.ldo = ldo;
  a.part = (float*)scratch;
  a.part_ml = (float2*)(a.part + (long long)p.partial_rows * c.heads * HEAD);
  a.pages = c.pages;
  a.heads = c.heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = device_status_word();
  cudaStream_t st = (cudaStream_t)stream;
  int rc = kHostOk;
  if (p.chunk_count > 0) {
    void* wide = a.part_ml + (((long long)p.partial_rows * c.heads + 15) & ~15ll);      // 128-byte aligned
    if (c.fp8 && (rc = launch_widen(c, p, wide, st)) != kHostOk) return rc;
    if ((rc = launch_chunks(c, p, q, ldq, p.rows, o, ldo, a.part, a.part_ml, a.scale_log2, wide, st)) != kHostOk) return rc;
  }
  if (p.few_count > 0) {
    if (c.fp8)
      rc = p.few_rows <= 16 ? launch_few<true, 1>(c, p, a, st) : p.few_rows <= 32 ? launch_few<true, 2>(c, p, a, st) : launch_few<true, 4>(c, p, a, st);
    else
      rc = p.few_rows <= 16 ? launch_few<false, 1>(c, p, a, st) : p.few_rows <= 32 ? launch_few<false, 2>(c, p, a, st) : launch_few<false, 4>(c, p, a, st);
    if (rc != kHostOk) return rc;
  }
  if (p.merge_count > 0)
    SNU1_CUDA_CHECK(launch_pdl(paged_merge_kernel, dim3(p.merge_count, (p.merge_rows * c.heads + 3) / 4), dim3(MERGE_THREADS), 0, st, p, a));
  return kHostOk;
}
