// Paged key/value cache: what the kernels that write, read and attend to it share.
//
// A cache holds one layer.  Page p keeps ``page`` tokens of all key/value heads, head by head:
//   data   [pages][2 (key, value)][heads][page][128]   bf16, or e4m3 codes
//   scales [pages][2][heads][page]                     fp32, e4m3 only: value = code * scale
// so the rows of one head are contiguous inside a page, which is the unit that an attention CTA asks for (one TMA box for
// keys and values together).  Sequences own pages through a table in any order; pages of 16 to 128 tokens.
#pragma once
#include <cuda_fp16.h>

#include "attn_common.cuh"
#include "host_common.h"

namespace snu1 {
namespace paged {

constexpr int HEAD = 128;                  // width of a head
constexpr float E4M3_MAX = 448.f;
constexpr float TINY = 7.70371977754894342e-34f;   // 2^-110, least row maximum that a scale is made of: 448 / TINY is finite

constexpr float P_TOP = 7.f;               // fp16 probabilities: the largest is 2^7, or up to 2^15 while the running maximum is old

// One layer's cache, filled by snu1_paged_cache_init.
struct alignas(64) Cache {
  CUtensorMap kv;          // box: up to 128 tokens of one head, keys and values, of bf16 up to 64 and 64 values wide
  CUtensorMap scale;       // box: the scales of the same
  CUtensorMap k, v;        // boxes of up to 128 tokens of one head, 64 values wide; e4m3: k takes keys or values, 128 wide
  void* data;
  float* scales;
  int pages, heads, page, fp8;
};

constexpr int PLAN_LAYOUT = 0x70670002;

// Device arrays and counts of a plan (ops/paged.py builds it).
struct Plan {
  const int* q_start;      // [seqs + 1] first query row of a sequence
  const int* kv_len;       // [seqs] cached tokens, the new ones among them; may be advanced in place ...
  const int* cap;          // [seqs] ... up to this
  const int* table;        // [seqs][width] pages
  const int* behind;       // [rows] a row reads its sequence's first kv_len - behind keys; null: up to itself
  const int* row_seq;      // [rows] sequence of a row
  const int* k_start;      // [seqs + 1] first packed row of a sequence, by the planned lengths
  const int2* read_pages;  // [read_count] (sequence, page of it) of all planned pages
  const int2* unpack;      // [unpack_count] (sequence, tile of 128 tokens) of the e4m3 sequences that the chunk kernel handles
  const int* unpack_first; // [seqs] first page of such a sequence in the scratch for unpacked rows
  const int4* few;         // [few_count] work of the kernel for few rows: sequence, first row, part | parts << 16, partial row (-1: none)
  const int4* chunk;       // [chunk_count] the same for chunks
  const int4* one;         // [one_count] the same for e4m3 chunks of one row tile per CTA
  const int4* merge;       // [merge_count] up to four rows to join: sequence, first row, parts | rows << 12 | rows of a part << 16, first partial row
  int seqs, rows, width, page, group;
  int read_count, few_count, few_rows, few_parts, few_cluster, chunk_count, one_count, merge_count;
  int partial_rows;        // rows of the scratch for partial results (x heads)
  int unpack_count;        // also the 128-token pages of the scratch for unpacked rows
  int layout;              // PLAN_LAYOUT; changes with the fields
};

// A tile whose largest scale is ``top`` is divided by a power of two for fp16: 2^tile_exponent would make its values at most 1 (codes are
// up to 448), and they are taken 2^WIDEN_UP times larger, up to 2^15 if the exponent is at its upper limit.
constexpr int WIDEN_UP = 13;
__device__ __forceinline__ int tile_exponent(float top) {
  return max(-80, min(126, (int)(__float_as_uint(E4M3_MAX * top) >> 23) - 126));
}

__device__ __forceinline__ int seq_len(const Plan& p, int b) { return max(0, min(p.kv_len[b], p.cap[b])); }

// A sequence with new rows that has grown past what the plan has pages for: its rows are not those that the caller means.
__device__ __forceinline__ void report_grown(const Plan& p, int b, int* status) {
  if (p.kv_len[b] > p.cap[b]) report_status(status, kBadShape, 10);
}

// Keys that row ``token`` of a sequence may read.
__device__ __forceinline__ int row_limit(const Plan& p, int q0, int q_len, int kv_len, int token) {
  const int behind = p.behind != nullptr ? p.behind[q0 + token] : q_len - 1 - token;
  return max(0, min(kv_len, kv_len - behind));
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// A factor as two fp16 numbers, hi + lo.
__device__ __forceinline__ uint32_t split_f16(float f) {
  const __half hi = __float2half_rn(f), lo = __float2half_rn(f - __half2float(hi));
  return (uint32_t)__half_as_ushort(hi) | (uint32_t)__half_as_ushort(lo) << 16;
}

// The four codes in ``w`` times a factor as fp16, ``hi`` and ``lo`` twice each: the product with hi has 15 bits and is rounded once,
// together with the product with lo.
__device__ __forceinline__ uint2 widen_scaled(uint32_t w, uint32_t hi, uint32_t lo) {
  uint2 r;
  asm("{\n.reg .b16 l, u;\n.reg .b32 h, t;\nmov.b32 {l, u}, %2;\n"
      "cvt.rn.f16x2.e4m3x2 h, l;\nmul.rn.f16x2 t, h, %4;\nfma.rn.f16x2 %0, h, %3, t;\n"
      "cvt.rn.f16x2.e4m3x2 h, u;\nmul.rn.f16x2 t, h, %4;\nfma.rn.f16x2 %1, h, %3, t;\n}"
      : "=r"(r.x), "=r"(r.y)
      : "r"(w), "r"(hi), "r"(lo));
  return r;
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z, int w, int u) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(u)
      : "memory");
}

// paged_cache.cu: a plan's ``unpack`` tiles of an e4m3 cache as fp16 pages at ``wide``
int launch_widen(const Cache& c, const Plan& p, void* wide, float4* factors, cudaStream_t st);
// attn_paged_sm100.cu: a plan's ``one`` and ``chunk`` items
int launch_chunks(const Cache& c, const Plan& p, const void* q, long long ldq, void* o, long long ldo, float* part,
                  float2* part_ml, float scale_log2, void* wide, const float4* factors, cudaStream_t st);

}  // namespace paged
}  // namespace snu1
