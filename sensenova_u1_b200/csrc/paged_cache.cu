// Paged key/value cache: descriptors, writing (with quantisation) and reading back.
//
// Quantising a row x of 128 values (one token, one head, keys or values): a = max(max |x|, 2^-110), scale = a / 448,
// code = e4m3(x * (448 / a)), all in fp32 with one rounding to e4m3 at the end; e4m3 because a code is a bf16 value
// exactly, so attention can take codes straight to the tensor cores and apply the scales in fp32.  One scale per row: rows
// of one head differ in size from token to token, and a row is written once, by itself.  A row that holds a value that is
// not finite gets NaN as its scale: it reads back as NaN, and attention to it is NaN.
//
// Both directions are bound by memory: 16 lanes own a row (16 bytes of bf16, 8 codes each), four rows are in flight per
// lane.  Where a token or a page lives takes three dependent loads, so a block looks that up once for many rows: up to 16
// tokens of all heads when writing, 256 rows of a page when reading.  Measured, e4m3: 32001 tokens of 8 heads written in 38 us, 5.2 TB/s
// or 0.80 of what a long copy reaches; 32001 of 4 heads read back in 20 us, 4.9 TB/s.  A plain copy of as many bytes takes as long:
// 100 MB read and written 38 us, 53 MB 22 to 25.
#include <cuda_fp8.h>
#include <string.h>

#include "host_common.h"
#include "paged.cuh"

namespace snu1 {
namespace paged {

// eight codes as numbers
__device__ __forceinline__ void decode8(uint2 u, float (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __half2 h(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((j < 2 ? u.x : u.y) >> (16 * (j & 1))), __NV_E4M3));
    const float2 g = __half22float2(h);
    f[2 * j] = g.x;
    f[2 * j + 1] = g.y;
  }
}

// two numbers as codes, the first in the low byte
__device__ __forceinline__ uint32_t e4m3x2(uint64_t x) {
  float lo, hi;
  unpack_f32x2(x, lo, hi);
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

constexpr int WRITE_THREADS = 256;
constexpr int WRITE_TOKENS = 16;     // most tokens of a block
constexpr int WRITE_DEEP = 4;        // heads of a token that a warp has in flight

// A block writes ``tokens`` rows of all heads; a warp four heads of a token at a time, 16 lanes the keys, 16 the values.
template <bool FP8>
__global__ void __launch_bounds__(WRITE_THREADS)
    paged_write_kernel(const __nv_bfloat16* __restrict__ k, long long ldk, const __nv_bfloat16* __restrict__ v, long long ldv,
                       uint8_t* __restrict__ data, float* __restrict__ scales, int pages, int heads, int tokens, Plan p, int* status) {
  __shared__ long long place[WRITE_TOKENS];          // the token's row for head 0's keys, -1: none
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kv = lane >> 4, c = lane & 15;
  const int row0 = blockIdx.x * tokens, count = min(tokens, p.rows - row0);
  if (threadIdx.x < count) {
    const int row = row0 + threadIdx.x, b = p.row_seq[row];
    const int pos = seq_len(p, b) - (p.q_start[b + 1] - row);
    long long at = -1;
    if (p.kv_len[b] > p.cap[b]) {                    // grown past what the plan has pages for
      report_status(status, kBadShape, 9);
    } else if (pos >= 0) {
      const int pg = p.table[(long long)b * p.width + pos / p.page];
      if (pg >= 0 && pg < pages) at = (long long)pg * 2 * heads * p.page + pos % p.page;
      else report_status(status, kBadPage, 9);
    }
    place[threadIdx.x] = at;
  }
  const __nv_bfloat16* src = (kv ? v : k) + (long long)row0 * (kv ? ldv : ldk) + c * 8;
  const long long ld = kv ? ldv : ldk;
  const int fours = (heads + WRITE_DEEP - 1) / WRITE_DEEP, tasks = count * fours;
  bool known = false;
  for (int task = warp; task < tasks; task += WRITE_THREADS / 32) {
    const int token = task / fours, head = (task - token * fours) * WRITE_DEEP;
    const __nv_bfloat16* from = src + token * ld + head * HEAD;
    uint4 x[WRITE_DEEP];
#pragma unroll
    for (int i = 0; i < WRITE_DEEP; ++i)
      x[i] = head + i < heads ? *reinterpret_cast<const uint4*>(from + i * HEAD) : make_uint4(0, 0, 0, 0);
    if (!known) {
      __syncthreads();
      known = true;
    }
    const long long base = place[token];
    if (base < 0) continue;                          // (the whole warp)
    const long long at = base + (long long)(kv * heads + head) * p.page;      // of the first head; the next is a page's rows on
    uint8_t* to = data + at * (FP8 ? HEAD : 2 * HEAD) + c * (FP8 ? 8 : 16);
    const int step = p.page * (FP8 ? HEAD : 2 * HEAD);
    if (!FP8) {
#pragma unroll
      for (int i = 0; i < WRITE_DEEP; ++i)
        if (head + i < heads) *reinterpret_cast<uint4*>(to + i * step) = x[i];
      continue;
    }
    // The instructions bound this (144 per warp and head took 44 us for 32001 tokens of 8 heads, the bytes take 31), so a warp has
    // four heads of one token, the largest value is found two 16-bit words at a time, and a lane divides for one of the
    // four rows.  As whole numbers a NaN is larger than infinity, which is larger than every finite value.
    uint32_t tops[WRITE_DEEP];
#pragma unroll
    for (int i = 0; i < WRITE_DEEP; ++i) {
      uint32_t t = max_u16x2(max_u16x2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu), max_u16x2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu));
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) t = max_u16x2(t, __shfl_xor_sync(0xffffffffu, t, o));
      tops[i] = t;
    }
    // (picked by hand: an index would put the array in local memory)
    const uint32_t t = c & 2 ? (c & 1 ? tops[3] : tops[2]) : (c & 1 ? tops[1] : tops[0]);
    const uint32_t top = max(t << 16, t & 0xffff0000u);
    const bool finite = top < 0x7f800000u;           // otherwise NaN is the scale, and the codes are zeros
    const float a = fmaxf(__uint_as_float(top), TINY), inv = finite ? __fdiv_rn(E4M3_MAX, a) : 0.f;
    if (c < WRITE_DEEP && head + c < heads) scales[at + c * p.page] = finite ? __fdiv_rn(a, E4M3_MAX) : __int_as_float(0x7fffffff);
#pragma unroll
    for (int i = 0; i < WRITE_DEEP; ++i) {
      const float f = __shfl_sync(0xffffffffu, inv, (lane & 16) + i);
      const uint64_t f2 = pack_f32x2(f, f);
      const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      uint32_t q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = e4m3x2(mul_f32x2(bf16x2_to_f32x2(u[j]), f2));
      if (head + i < heads)
        *reinterpret_cast<uint2*>(to + i * step) =
            f != 0.f ? make_uint2(__byte_perm(q[0], q[1], 0x5410), __byte_perm(q[2], q[3], 0x5410)) : make_uint2(0, 0);
    }
  }
  if (!known) __syncthreads();
}

constexpr int READ_THREADS = 256;
constexpr int READ_DEEP = 4;                                         // rows that a lane has in flight
constexpr int READ_BLOCK = 256;                                      // rows of a block

// Rows of the planned pages, in order: keys to ``out``, values to ``out2``, [rows][heads][128].
template <bool FP8>
__global__ void __launch_bounds__(READ_THREADS)
    paged_read_kernel(const uint8_t* __restrict__ data, const float* __restrict__ scales, int pages, int heads, int page, Plan p,
                      __nv_bfloat16* __restrict__ out, __nv_bfloat16* __restrict__ out2, int* status) {
  const int2 e = p.read_pages[blockIdx.x];                           // set by the host, as is k_start
  const int page_log = __ffs(page) - 1;
  const int b = e.x, pos0 = e.y * page, c = threadIdx.x & 15;
  const int k0 = p.k_start[b], len = p.k_start[b + 1] - k0;
  pdl_wait();
  pdl_trigger();
  const int pg = p.table[(long long)b * p.width + e.y];
  const bool there = pg >= 0 && pg < pages;
  if (!there && threadIdx.x == 0) report_status(status, kBadPage, 9);
  const int total = 2 * heads * page, end = min(total, (int)(blockIdx.y + 1) * READ_BLOCK);
  for (int first = blockIdx.y * READ_BLOCK + (threadIdx.x >> 4); first < end; first += READ_THREADS / 16 * READ_DEEP) {
    uint4 x[READ_DEEP];
    float s[READ_DEEP];
#pragma unroll
    for (int i = 0; i < READ_DEEP; ++i) {
      const int r = first + i * (READ_THREADS / 16);                 // row of the page: (kv, head, token)
      x[i] = make_uint4(0, 0, 0, 0);
      s[i] = 0.f;
      if (there && r < end && pos0 + (r & (page - 1)) < len) {
        const long long at = (long long)pg * total + r;
        if (FP8) {
          const uint2 u = *reinterpret_cast<const uint2*>(data + at * HEAD + c * 8);
          x[i].x = u.x;
          x[i].y = u.y;
          s[i] = scales[at];
        } else {
          x[i] = *reinterpret_cast<const uint4*>(data + at * (HEAD * 2) + c * 16);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < READ_DEEP; ++i) {
      const int r = first + i * (READ_THREADS / 16);
      const int pos = pos0 + (r & (page - 1)), kvh = r >> page_log, kv = kvh >= heads, head = kvh - kv * heads;
      if (r >= end || pos >= len) continue;
      uint4 y = x[i];
      if (FP8) {
        float f[8];
        decode8(make_uint2(x[i].x, x[i].y), f);
        y = make_uint4(pack_bf16x2(f[0] * s[i], f[1] * s[i]), pack_bf16x2(f[2] * s[i], f[3] * s[i]),
                       pack_bf16x2(f[4] * s[i], f[5] * s[i]), pack_bf16x2(f[6] * s[i], f[7] * s[i]));
      }
      *reinterpret_cast<uint4*>((kv ? out2 : out) + ((long long)(k0 + pos) * heads + head) * HEAD + c * 8) = y;
    }
  }
}

// Tiles of 128 tokens of an e4m3 cache for attn_paged_sm100.cu: fp16 pages of 128 tokens in a cache's own layout, every
// sequence from a page of its own on, rows behind its last token cleared.  A tile of one head is divided by a power of two,
// so that its largest value is at most 2^13 (2^-93 to 2^113; that factor goes into the scores, or into the probabilities): code times
// scale is rounded to 11 bits, and what falls below fp16's normal range is 2^27 times smaller than the tile's largest value.
// factors [page][heads]: the keys' power of two, the exponent of the values' (log2), and, as a whole number, the first
// key of the sequence in this tile whose value is not finite (its scale is not); that value is cleared.
constexpr int WIDEN_THREADS = 256;

__global__ void __launch_bounds__(WIDEN_THREADS)
    paged_widen_kernel(const uint8_t* __restrict__ data, const float* __restrict__ scales, int pages, int heads, Plan p,
                       uint8_t* __restrict__ wide, float4* __restrict__ factors, int* status) {
  __shared__ long long s_at[128];          // the token's row of the cache, -1: none
  __shared__ uint32_t s_mult[128];         // the row's factor, see split_f16
  __shared__ float s_top[4];
  __shared__ int s_bad[4];
  const int2 e = p.unpack[blockIdx.x];     // set by the host
  pdl_wait();
  pdl_trigger();
  const int kv = blockIdx.y >= heads, head = blockIdx.y - kv * heads, b = e.x, t = threadIdx.x;
  const int len = seq_len(p, b);
  float s = 0.f;
  if (t < 128) {
    const int pos = e.y * 128 + t;
    long long at = -1;
    if (pos < len) {
      const int pg = p.table[(long long)b * p.width + pos / p.page];
      if (pg >= 0 && pg < pages) {
        at = (((long long)pg * 2 + kv) * heads + head) * p.page + pos % p.page;
        s = scales[at];
      } else {
        report_status(status, kBadPage, 9);
      }
    }
    const bool finite = fabsf(s) < INFINITY;
    const uint32_t top = __reduce_max_sync(0xffffffffu, finite ? __float_as_uint(fabsf(s)) : 0u);
    const int bad = __reduce_min_sync(0xffffffffu, finite ? 0x7fffffff : pos);
    if (kv && !finite) {
      at = -1;
      s = 0.f;
    }
    s_at[t] = at;
    if ((t & 31) == 0) {
      s_top[t >> 5] = __uint_as_float(top);
      s_bad[t >> 5] = bad;
    }
  }
  __syncthreads();
  const int ex = tile_exponent(fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]))) - WIDEN_UP;
  const float down = __int_as_float((127 - ex) << 23);
  const long long page = p.unpack_first[b] + e.y;
  if (t == 0) {
    float* f = reinterpret_cast<float*>(factors + page * heads + head);
    f[kv] = kv ? (float)ex : __int_as_float((127 + ex) << 23);
    if (kv) f[2] = __int_as_float(min(min(s_bad[0], s_bad[1]), min(s_bad[2], s_bad[3])));
  }
  if (t < 128) s_mult[t] = split_f16(s * down);
  const int c = t & 15;
  uint2 x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long long at = s_at[(t >> 4) + 16 * i];
    x[i] = at >= 0 ? *reinterpret_cast<const uint2*>(data + at * HEAD + c * 8) : make_uint2(0, 0);
  }
  __syncthreads();
  uint8_t* to = wide + ((page * 2 + kv) * heads + head) * 128 * 256 + c * 16;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = (t >> 4) + 16 * i;
    const uint32_t f = s_mult[row], hi = __byte_perm(f, f, 0x1010), lo = __byte_perm(f, f, 0x3232);
    const uint2 y = widen_scaled(x[i].x, hi, lo), z = widen_scaled(x[i].y, hi, lo);
    *reinterpret_cast<uint4*>(to + row * 256) = make_uint4(y.x, y.y, z.x, z.y);
  }
}

int launch_widen(const Cache& c, const Plan& p, void* wide, float4* factors, cudaStream_t st) {
  SNU1_CUDA_CHECK(launch_pdl(paged_widen_kernel, dim3(p.unpack_count, 2 * c.heads), dim3(WIDEN_THREADS), 0, st, (const uint8_t*)c.data,
                             (const float*)c.scales, c.pages, c.heads, p, (uint8_t*)wide, factors, device_status_word()));
  return kHostOk;
}

}  // namespace paged
}  // namespace snu1

using namespace snu1;

SNU1_API int snu1_paged_cache_bytes() { return (int)sizeof(paged::Cache); }
SNU1_API int snu1_paged_plan_bytes() { return (int)sizeof(paged::Plan); }

// Fills ``out`` (snu1_paged_cache_bytes) for the cache at data / scales.
SNU1_API int snu1_paged_cache_init(void* out, void* data, void* scales, int pages, int heads, int page, int fp8) {
  if (pages <= 0 || heads <= 0 || (page != 16 && page != 32 && page != 64 && page != 128) || (fp8 != 0) != (scales != nullptr) ||
      ((reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(scales)) & 15) != 0) {
    set_last_error("paged_cache: pages of 16, 32, 64 or 128 tokens in 16-byte aligned memory, scales for e4m3 only");
    return kHostBadArg;
  }
  paged::Cache c;
  memset(&c, 0, sizeof(c));
  c.data = data;
  c.scales = (float*)scales;
  c.pages = pages;
  c.heads = heads;
  c.page = page;
  c.fp8 = fp8;
  const uint64_t row = fp8 ? 128 : 256, P = page, H = heads;
  const uint32_t bx = fp8 || page < 64 ? page : 64;      // a stage of attn_paged.cu: 128 tokens of e4m3, 64 of bf16
  int rc;
  {
    const uint64_t dims[5] = {128, P, H, 2, (uint64_t)pages}, str[4] = {row, row * P, row * P * H, row * P * H * 2};
    const uint32_t box[5] = {fp8 ? 128u : 64u, bx, 1, 2, 1};
    if ((rc = encode_tmap(&c.kv, fp8 ? TmapType::kU8 : TmapType::kBf16, true, data, 5, dims, str, box)) != kHostOk) return rc;
  }
  if (fp8) {
    const uint64_t dims[4] = {P, H, 2, (uint64_t)pages}, str[3] = {P * 4, P * H * 4, P * H * 8};
    const uint32_t box[4] = {bx, 1, 2, 1};
    const uint64_t kdims[5] = {128, P, H, 2, (uint64_t)pages}, kstr[4] = {row, row * P, row * P * H, row * P * H * 2};
    const uint32_t kbox[5] = {128, (uint32_t)page, 1, 1, 1};
    if ((rc = encode_tmap(&c.k, TmapType::kU8, true, data, 5, kdims, kstr, kbox)) != kHostOk) return rc;
    if ((rc = encode_tmap(&c.scale, TmapType::kF32, false, scales, 4, dims, str, box)) != kHostOk) return rc;
  } else {
    const uint64_t dims[4] = {128, P, H, (uint64_t)pages}, str[3] = {row, row * P, row * P * H * 2};
    const uint32_t box[4] = {64, (uint32_t)page, 1, 1};
    if ((rc = encode_tmap(&c.k, TmapType::kBf16, true, data, 4, dims, str, box)) != kHostOk) return rc;
    if ((rc = encode_tmap(&c.v, TmapType::kBf16, true, (uint8_t*)data + row * P * H, 4, dims, str, box)) != kHostOk) return rc;
  }
  if (device_status_word() == nullptr) {          // here and not in a first call that may be captured
    set_last_error("paged_cache: no status word (cudaMalloc failed?)");
    return kHostCuda;
  }
  memcpy(out, &c, sizeof(c));
  return kHostOk;
}

// Keys and values of a plan's new rows ([rows][heads][128] bf16, rows ldk / ldv apart) into their sequences' pages.
SNU1_API int snu1_paged_write(const void* cache, const void* plan, const void* k, long long ldk, const void* v, long long ldv,
                              void* stream) {
  paged::Cache c;
  paged::Plan p;
  memcpy(&c, cache, sizeof(c));
  memcpy(&p, plan, sizeof(p));
  if (p.layout != paged::PLAN_LAYOUT) {
    set_last_error("paged: this plan was made for another version of the library");
    return kHostBadArg;
  }
  if (p.rows <= 0) return kHostOk;
  if (p.page != c.page || ldk % 8 || ldv % 8 || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) != 0) {
    set_last_error("paged_write: rows must be 16-byte aligned, and the plan made for this page size");
    return kHostBadArg;
  }
  // many tokens share a block's look-up, as long as there are blocks for every SM
  const int tokens = max(1, min(paged::WRITE_TOKENS, p.rows / (4 * num_sms())));
  auto kernel = c.fp8 ? paged::paged_write_kernel<true> : paged::paged_write_kernel<false>;
  SNU1_CUDA_CHECK(launch_pdl(kernel, dim3((p.rows + tokens - 1) / tokens), dim3(paged::WRITE_THREADS), 0, (cudaStream_t)stream,
                             (const __nv_bfloat16*)k, ldk, (const __nv_bfloat16*)v, ldv, (uint8_t*)c.data, c.scales, c.pages, c.heads,
                             tokens, p, device_status_word()));
  return kHostOk;
}

// Cached rows of a plan's sequences, packed: k, v [planned keys][heads][128] bf16.
SNU1_API int snu1_paged_read(const void* cache, const void* plan, void* k, void* v, void* stream) {
  paged::Cache c;
  paged::Plan p;
  memcpy(&c, cache, sizeof(c));
  memcpy(&p, plan, sizeof(p));
  if (p.layout != paged::PLAN_LAYOUT) {
    set_last_error("paged: this plan was made for another version of the library");
    return kHostBadArg;
  }
  if (p.read_count <= 0) return kHostOk;
  if (p.page != c.page || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) != 0) {
    set_last_error("paged_read: outputs must be 16-byte aligned, and the plan made for this page size");
    return kHostBadArg;
  }
  const int total = 2 * c.heads * c.page;
  auto kernel = c.fp8 ? paged::paged_read_kernel<true> : paged::paged_read_kernel<false>;
  SNU1_CUDA_CHECK(launch_pdl(kernel, dim3(p.read_count, (total + paged::READ_BLOCK - 1) / paged::READ_BLOCK),
                             dim3(paged::READ_THREADS), 0, (cudaStream_t)stream, (const uint8_t*)c.data, c.scales, c.pages, c.heads,
                             c.page, p, (__nv_bfloat16*)k, (__nv_bfloat16*)v, device_status_word()));
  return kHostOk;
}
