// Block tables of the paged cache, kept on the device: every sequence goes on from the tokens of its parent.
//
//   kept_s = min(length of parent_s, keep_s) (0 without a parent),  length_s = kept_s + new_s
//   whole pages of the kept tokens are shared; rows of a page that is not full are the first sequence's that has them and that nobody
//   holds whole, the others get a page of their own and copies of the rows; then pages for the new tokens.  Pages that nobody holds
//   are free, and the free ones are taken lowest number first, sequence after sequence.
//
// No page that is not full has two holders, so new tokens never meet another sequence's.
//
// First kernel: a block has a few columns of all tables, which are independent of one another, so rows are moved in place; where an
// entry changes, the use counts of the old and the new page do.  The block that is last does what needs all of them: which partial pages
// stay, a scan over the use counts for free pages, lengths, and the list of copies.  Second kernel: the copies, in all layers at once.
// What bounds it: latency (launch, dependent look-ups, the scan), and for the copies memory.  So table entries are on their way before lengths and parents are
// known, and use counts before it is known which pages stay.  In a graph, both kernels: 4 beams over 864 tokens, 12 layers 7.6 us; 16 x 8
// beams over 1570 e4m3 tokens in pages of 16 15.1 (17.0 with all look-ups one after another), 4.5 of them the bytes; 32 beams over 32301 tokens 10.8.
#include <string.h>

#include <mutex>

#include "host_common.h"
#include "paged.cuh"

namespace snu1 {
namespace pages {

constexpr int THREADS = 512;
constexpr int MAX_SEQS = 1024;
constexpr int COLUMNS = 16;          // of a block
constexpr int MAX_LAYERS = 256;
constexpr int AHEAD = 4;             // table entries of a thread that are on their way before anything else is known
constexpr int FREE_CHUNKS = 4;       // the use counts of as many times 2048 pages are looked at early

// Device arrays of ops/page_tables.py's PageTables.
struct Tables {
  int* table;          // [seqs][width], -1: no page
  int* lens;           // [seqs]
  int* refs;           // [pages] sequences that hold a page
  int* claim;          // [pages] scratch: MAX_SEQS between steps
  int4* copies;        // [seqs] source, destination, rows (0: none)
  int* count;          // blocks that are done; 0 between steps
  int seqs, width, pages, page;
  int layout;
};
constexpr int LAYOUT = 0x70670003;

struct StepArgs {
  Tables t;
  const int* parents;  // null: every sequence goes on from itself
  const int* keep;     // null: all
  const int* more;     // [seqs] new tokens; null: ``each``
  int each;
  int* status;
};

__device__ __forceinline__ int kept_of(const StepArgs& a, int s, int* parent) {
  const int p = a.parents != nullptr ? a.parents[s] : s;
  *parent = p;
  if (p < 0 || p >= a.t.seqs) {
    if (p != -1) report_status(a.status, kBadShape, 12);
    return 0;
  }
  const int len = max(0, min(a.t.lens[p], a.t.width * a.t.page));
  return a.keep != nullptr ? max(0, min(len, a.keep[s])) : len;
}

// sum over the block of what the threads before have, and of all
__device__ __forceinline__ int2 scan_block(int x, int* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int y = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = y;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    before += w < warp ? s_warp[w] : 0;
    all += s_warp[w];
  }
  return make_int2(before + y - x, all);
}

__global__ void __launch_bounds__(THREADS) step_kernel(const StepArgs a) {
  extern __shared__ int s_col[];                 // [seqs][COLUMNS] the columns before the step
  __shared__ int s_warp[THREADS / 32];
  __shared__ int s_vote;
  __shared__ int s_parent[MAX_SEQS], s_kept[MAX_SEQS], s_from[MAX_SEQS], s_need[MAX_SEQS], s_src[MAX_SEQS], s_used[MAX_SEQS];
  __shared__ uint32_t s_stays[FREE_CHUNKS * THREADS * 4 / 32];       // pages that stay with one sequence, by bit
  const Tables& t = a.t;
  const int tid = threadIdx.x, S = t.seqs, W = t.width, page = t.page, page_log = __ffs(page) - 1;
  const int c0 = blockIdx.x * COLUMNS, cn = min(COLUMNS, W - c0);
  for (int i = tid; i < FREE_CHUNKS * THREADS * 4 / 32; i += THREADS) s_stays[i] = 0;
  pdl_wait();
  pdl_trigger();
  int ahead[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = tid + k * THREADS, s = i / COLUMNS, c = i % COLUMNS;
    ahead[k] = s < S && c < cn ? t.table[(long long)s * W + c0 + c] : -1;
  }
  for (int s = tid; s < S; s += THREADS) {
    const int len = max(0, t.lens[s]);
    int p;
    s_kept[s] = kept_of(a, s, &p);
    s_parent[s] = p;
    s_from[s] = min(W, (len + page - 1) >> page_log);     // pages before
    s_src[s] = s_used[s] = -1;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = tid + k * THREADS;
    if (i < S * COLUMNS) s_col[i] = c0 + i % COLUMNS < s_from[i / COLUMNS] ? ahead[k] : -1;
  }
  for (int i = tid + AHEAD * THREADS; i < S * COLUMNS; i += THREADS) {
    const int s = i / COLUMNS, c = i % COLUMNS;
    s_col[i] = c < cn && c0 + c < s_from[s] ? t.table[(long long)s * W + c0 + c] : -1;
  }
  __syncthreads();
  for (int i = tid; i < S * COLUMNS; i += THREADS) {
    const int s = i / COLUMNS, c = i % COLUMNS, j = c0 + c;
    if (c >= cn) continue;
    const int kept = s_kept[s], full = kept >> page_log, part = kept & (page - 1), old = s_col[i];
    const int src = j < full + (part != 0) ? s_col[s_parent[s] * COLUMNS + c] : -1;             // (kept > 0: there is a parent)
    const int now = j < full ? src : -1;
    if (j >= full || now != old) t.table[(long long)s * W + j] = now;
    if (now != old) {
      if (old >= 0 && old < t.pages) atomicSub(&t.refs[old], 1);
      if (now >= 0 && now < t.pages) atomicAdd(&t.refs[now], 1);
    }
    if (j == full && part != 0) {                                                                // the page that is not full
      t.copies[s] = make_int4(src, -1, part, 0);
      if (src >= 0 && src < t.pages) atomicMin(&t.claim[src], s);
    }
  }
  // the last block goes on
  if (gridDim.x > 1) {
    __threadfence();
    __syncthreads();
    if (tid == 0) s_vote = atomicAdd(t.count, 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (!s_vote) return;
    __threadfence();
    if (tid == 0) *t.count = 0;
  } else {
    __syncthreads();
  }
  int4 uses[FREE_CHUNKS];                        // as they are now: a page that stays is told by its bit
#pragma unroll
  for (int k = 0; k < FREE_CHUNKS; ++k) {
    const int p = (k * THREADS + tid) * 4;
    uses[k] = make_int4(1, 1, 1, 1);
    if (p + 3 < t.pages) {
      uses[k] = __ldcg(reinterpret_cast<const int4*>(t.refs + p));
    } else if (p < t.pages) {
      uses[k].x = __ldcg(t.refs + p);
      if (p + 1 < t.pages) uses[k].y = __ldcg(t.refs + p + 1);
      if (p + 2 < t.pages) uses[k].z = __ldcg(t.refs + p + 2);
    }
  }
  // partial pages: stay or are copied; how many pages every sequence needs
  int total = 0;
  for (int s0 = 0; s0 < S; s0 += THREADS) {
    const int s = s0 + tid;
    int need = 0, begin = 0, src = -1, part = 0;
    bool stays = false;
    if (s < S) {
      const int kept = s_kept[s], full = kept >> page_log;
      const long long more = a.more != nullptr ? max(0, a.more[s]) : a.each;
      const long long want = min((long long)kept + more, (long long)W * page);
      if (want < kept + more) report_status(a.status, kBadShape, 12);
      part = kept & (page - 1);
      if (part != 0) {
        src = __ldcg(&t.copies[s].x);
        stays = src >= 0 && src < t.pages && __ldcg(&t.refs[src]) == 0 && __ldcg(&t.claim[src]) == s;
      }
      begin = full + (stays ? 1 : 0);
      need = max(0, (int)((want + page - 1) >> page_log) - begin);
      s_src[s] = stays ? src : -1;
      s_used[s] = src;
      if (stays && src < FREE_CHUNKS * THREADS * 4) atomicOr(&s_stays[src >> 5], 1u << (src & 31));
      t.copies[s] = part != 0 && !stays ? make_int4(src, -1, part, 0) : make_int4(-1, -1, 0, 0);
      if (stays) t.table[(long long)s * W + full] = src;
      t.lens[s] = (int)want;
    }
    const int2 sc = scan_block(need, s_warp);
    if (s < S) {
      s_need[s] = total + sc.x;                  // free pages that go to the sequences before
      s_from[s] = begin;
    }
    total += sc.y;
  }
  __syncthreads();
  for (int s = tid; s < S; s += THREADS) {       // after everybody has looked at the counts
    if (s_src[s] >= 0) t.refs[s_src[s]] = 1;
    if (s_used[s] >= 0 && s_used[s] < t.pages) t.claim[s_used[s]] = MAX_SEQS;
  }
  __syncthreads();
  // the first ``total`` free pages, in order
  int found = 0;
  auto deal = [&](int p, const bool (&free)[4]) {
    const int2 sc = scan_block(free[0] + free[1] + free[2] + free[3], s_warp);
    int n = found + sc.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!free[i]) continue;
      if (n < total) {
        // whose it is: the last sequence that has at most n pages before its own
        int lo = 0, hi = S - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) / 2;
          if (s_need[mid] <= n) lo = mid;
          else hi = mid - 1;
        }
        const int j = s_from[lo] + n - s_need[lo], kept = s_kept[lo];
        t.table[(long long)lo * W + j] = p + i;
        t.refs[p + i] = 1;
        if (j == kept >> page_log && (kept & (page - 1)) != 0) t.copies[lo].y = p + i;
      }
      ++n;
    }
    found += sc.y;
  };
#pragma unroll
  for (int k = 0; k < FREE_CHUNKS; ++k) {
    const int p = (k * THREADS + tid) * 4;
    if (k * THREADS * 4 >= t.pages || found >= total) break;
    const uint32_t stays = s_stays[p >> 5] >> (p & 31);
    const bool free[4] = {uses[k].x == 0 && !(stays & 1), uses[k].y == 0 && !(stays & 2), uses[k].z == 0 && !(stays & 4), uses[k].w == 0 && !(stays & 8)};
    deal(p, free);
  }
  for (int p0 = FREE_CHUNKS * THREADS * 4; p0 < t.pages && found < total; p0 += THREADS * 4) {
    const int p = p0 + tid * 4;
    bool free[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) free[i] = p + i < t.pages && __ldcg(&t.refs[p + i]) == 0;
    deal(p, free);
  }
  if (found < total && tid == 0) report_status(a.status, kBadPage, 12);       // fewer free pages than are needed: -1 stays in their places
}

struct CopyArgs {
  const long long* layers;   // [2][layers] data and scales
  const int4* copies;
  int heads, page, pages, row_bytes, sides;       // row_bytes: of a token's values of one head; sides: of a block
};

constexpr int COPY_THREADS = 256;

// A block copies the rows of one sequence and layer, of ``sides`` sides (a side: keys or values of one head, whose rows are contiguous in a
// page): as many as a full page of them is 32 KB.  (16 x 8 sequences, 12 layers, pages of 16 tokens: the whole step 37 us with a
// block per side, so 17.)
__global__ void __launch_bounds__(COPY_THREADS) copy_kernel(const CopyArgs a) {
  pdl_wait();
  pdl_trigger();
  const int4 c = a.copies[blockIdx.x];
  if (c.z <= 0 || c.x < 0 || c.x >= a.pages || c.y < 0 || c.y >= a.pages) return;
  const int layer = blockIdx.z, first = blockIdx.y * a.sides, sides = min(a.sides, 2 * a.heads - first);
  uint8_t* data = reinterpret_cast<uint8_t*>(a.layers[layer]);
  float* scales = reinterpret_cast<float*>(a.layers[gridDim.z + layer]);
  const long long from = (long long)c.x * 2 * a.heads + first, to = (long long)c.y * 2 * a.heads + first;
  const int n = c.z * (a.row_bytes / 16), step = a.page * (a.row_bytes / 16);        // 16 bytes at a time: of a side, and from side to side
  const uint4* x = reinterpret_cast<const uint4*>(data) + from * step;
  uint4* y = reinterpret_cast<uint4*>(data) + to * step;
  for (int i0 = 0; i0 < n * sides; i0 += COPY_THREADS * 4) {
    uint4 v[4];
    int at[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * COPY_THREADS + threadIdx.x;
      at[k] = i < n * sides ? i / n * step + i % n : -1;
      if (at[k] >= 0) v[k] = x[at[k]];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at[k] >= 0) y[at[k]] = v[k];
  }
  if (scales != nullptr)
    for (int i = threadIdx.x; i < c.z * sides; i += COPY_THREADS) {
      const int at = i / c.z * a.page + i % c.z;
      scales[to * a.page + at] = scales[from * a.page + at];
    }
}

}  // namespace pages
}  // namespace snu1

using namespace snu1;

SNU1_API int snu1_page_tables_bytes() { return (int)sizeof(pages::Tables); }

// One step of ``tables`` (a pages::Tables); parents / keep / more: int32 [seqs] on the device or null.
SNU1_API int snu1_page_tables_step(const void* tables, const void* parents, const void* keep, const void* more, int each, void* stream) {
  using namespace pages;
  StepArgs a;
  memcpy(&a.t, tables, sizeof(Tables));
  if (a.t.layout != LAYOUT || a.t.seqs < 1 || a.t.seqs > MAX_SEQS || a.t.width < 1 || a.t.pages < 1 || each < 0) {
    set_last_error("page_tables_step: tables of another version, or more than %d sequences", MAX_SEQS);
    return kHostBadArg;
  }
  a.parents = (const int*)parents;
  a.keep = (const int*)keep;
  a.more = (const int*)more;
  a.each = each;
  a.status = device_status_word();
  const int smem = a.t.seqs * COLUMNS * 4;
  int dev = 0;
  SNU1_CUDA_CHECK(cudaGetDevice(&dev));
  static std::once_flag once[64];
  cudaError_t err = cudaSuccess;
  std::call_once(once[dev & 63], [&]() {
    err = cudaFuncSetAttribute(step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SEQS * COLUMNS * 4);
  });
  SNU1_CUDA_CHECK(err);
  SNU1_CUDA_CHECK(launch_pdl(step_kernel, dim3((a.t.width + COLUMNS - 1) / COLUMNS), dim3(THREADS), smem, (cudaStream_t)stream, a));
  return kHostOk;
}

// The copies that a step asks for, in ``count`` caches of one geometry; ``layers``: their data's addresses, then their scales' (0: none), int64 on the device.
SNU1_API int snu1_page_tables_copy(const void* tables, const void* layers, int count, int heads, int fp8, void* stream) {
  using namespace pages;
  Tables t;
  memcpy(&t, tables, sizeof(t));
  if (t.layout != LAYOUT || count < 1 || count > MAX_LAYERS || heads < 1) {
    set_last_error("page_tables_copy: tables of another version, or more than %d caches", MAX_LAYERS);
    return kHostBadArg;
  }
  CopyArgs a;
  a.layers = (const long long*)layers;
  a.copies = t.copies;
  a.heads = heads;
  a.page = t.page;
  a.pages = t.pages;
  a.row_bytes = fp8 ? paged::HEAD : 2 * paged::HEAD;
  a.sides = max(1, min(2 * heads, 32768 / (t.page * a.row_bytes)));
  SNU1_CUDA_CHECK(launch_pdl(copy_kernel, dim3(t.seqs, (2 * heads + a.sides - 1) / a.sides, count), dim3(COPY_THREADS), 0, (cudaStream_t)stream, a));
  return kHostOk;
}
