// layout.cu -- where the rows of one step go: the block tables are extended
// with pages from a free list and every new row gets its cache slot, position,
// request and visible length, all from the request lengths on the device.
//
// With s_b rows of request b in the cache and q_b new ones,
//   pages before / after   have_b = ceil(s_b / 64), need_b = ceil((s_b + q_b) / 64)
//   first new page         P_b = sum_{a<b} (need_a - have_a) of the free list
//   first new row          R_b = sum_{a<b} q_a of the outputs
//   table[b][have_b + i]   = free[P_b + i]
//   row R_b + j: position prefix + s_b + j, visible s_b + j + 1 own rows, slot
//   table[b][(s_b + j) / 64] * 64 + (s_b + j) % 64.
//
// One launch and no workspace: every CTA scans the two sums of a chunk of
// requests into shared memory (the lengths are a few KB and stay in L2), then
// the rows and pages of the chunk are dealt out over the grid and each finds
// its request by a binary search there.  A second launch behind a scan kernel
// would cost more than the repeated scan.  Bound by latency: the call moves
// 16 bytes a row and 8 a request.
#include "../../../include/dsa_b200.h"
#include <climits>

#include "../common.cuh"

namespace dsa {
namespace {

// Small CTAs: the scan's depth is what a call waits for (64 requests / 32768 rows of
// 509: 3.0 / 3.7 us; with 512 threads 3.6 / 4.4, with 8 requests a thread 3.5 / 4.4).
constexpr int kLayThreads = 128;
constexpr int kLayItems = 4;                         // requests per thread and chunk
constexpr int kLayChunk = kLayThreads * kLayItems;

struct LayoutParams {
  const int32_t *seq, *query, *free_pages, *prefix_len;
  int32_t *table, *slots, *positions, *request, *lens, *pages_used;
  int64_t batch, bt_stride, max_pages, num_free, rows;
  int* err;
};

// Exclusive sums of a thread's (rows, pages) over the CTA; *total gets both sums.
__device__ __forceinline__ longlong2 cta_scan(longlong2 v, longlong2* warp_sums, longlong2* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  longlong2 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, x.x, o), b = __shfl_up_sync(0xffffffffu, x.y, o);
    if (lane >= o) {
      x.x += a;
      x.y += b;
    }
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  longlong2 before = make_longlong2(0, 0), all = make_longlong2(0, 0);
  for (int w = 0; w < kLayThreads / 32; ++w) {
    const longlong2 s = warp_sums[w];
    if (w < warp) {
      before.x += s.x;
      before.y += s.y;
    }
    all.x += s.x;
    all.y += s.y;
  }
  *total = all;
  return make_longlong2(before.x + x.x - v.x, before.y + x.y - v.y);
}

// Largest i in [0, n) with first[i] <= at (first[0] <= at, ascending).
__device__ __forceinline__ int last_not_above(const long long* first, int n, long long at) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= at)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kLayThreads) dsa_step_layout_kernel(const LayoutParams p) {
  __shared__ long long row0[kLayChunk], page0[kLayChunk];
  __shared__ int32_t seq[kLayChunk];
  __shared__ longlong2 warp_sums[kLayThreads / 32];
  const int64_t at0 = (int64_t)blockIdx.x * kLayThreads + threadIdx.x;
  const int64_t step = (int64_t)gridDim.x * kLayThreads;
  const int64_t prefix = p.prefix_len ? max(*p.prefix_len, 0) : 0;
  long long rows_base = 0, pages_base = 0;
  int bits = 0;
  for (int64_t b0 = 0; b0 < p.batch; b0 += kLayChunk) {
    const int n = (int)min((int64_t)kLayChunk, p.batch - b0);
    int32_t s[kLayItems], q[kLayItems];
    longlong2 mine = make_longlong2(0, 0);
#pragma unroll
    for (int i = 0; i < kLayItems; ++i) {
      const int at = threadIdx.x * kLayItems + i;
      s[i] = at < n ? max(p.seq[b0 + at], 0) : 0;  // negative lengths count as none
      q[i] = at < n ? max(p.query[b0 + at], 0) : 0;
      mine.x += q[i];
      mine.y += (((long long)s[i] + q[i] + 63) >> 6) - (((long long)s[i] + 63) >> 6);
    }
    longlong2 total;
    longlong2 first = cta_scan(mine, warp_sums, &total);
#pragma unroll
    for (int i = 0; i < kLayItems; ++i) {
      const int at = threadIdx.x * kLayItems + i;
      if (at < n) {
        row0[at] = first.x;
        page0[at] = first.y;
        seq[at] = s[i];
      }
      first.x += q[i];
      first.y += (((long long)s[i] + q[i] + 63) >> 6) - (((long long)s[i] + 63) >> 6);
    }
    __syncthreads();
    // new pages of the chunk
    for (long long j = at0; j < total.y; j += step) {
      const int b = last_not_above(page0, n, j);
      const long long col = (((long long)seq[b] + 63) >> 6) + (j - page0[b]);
      const long long src = pages_base + j;
      if (col < p.max_pages)
        p.table[(b0 + b) * p.bt_stride + col] = src < p.num_free ? p.free_pages[src] : -1;
      if (col >= p.max_pages || src >= p.num_free) bits |= kErrCapacity;
    }
    // rows of the chunk
    const long long rows = min(total.x, p.rows - rows_base);
    if (total.x > p.rows - rows_base) bits |= kErrCapacity;
    for (long long i = at0; i < rows; i += step) {
      const int b = last_not_above(row0, n, i);
      const long long pos = (long long)seq[b] + (i - row0[b]);
      const long long col = pos >> 6, have = ((long long)seq[b] + 63) >> 6;
      int32_t page = -1;
      if (col < p.max_pages) {
        const long long src = pages_base + page0[b] + (col - have);
        const bool have_it = col < have || src < p.num_free;
        if (have_it) page = col < have ? p.table[(b0 + b) * p.bt_stride + col] : p.free_pages[src];
        // a slot past 2^31 rows has no 32-bit id: no cache of this library is that long
        if (have_it && (page < 0 || page >= (1 << 25))) bits |= kErrBadIndex;
      } else {
        bits |= kErrCapacity;  // of a page that the request had before too, though none is handed out for it
      }
      const long long out = rows_base + i;
      const bool ok = page >= 0 && page < (1 << 25);
      p.slots[out] = ok ? page * 64 + (int)(pos & 63) : -1;
      p.positions[out] = (int32_t)min(prefix + pos, (long long)INT32_MAX);
      p.request[out] = (int32_t)(b0 + b);
      p.lens[out] = (int32_t)min(pos + 1, (long long)INT32_MAX);
    }
    rows_base = min(rows_base + total.x, (long long)p.rows);
    pages_base += total.y;
    __syncthreads();  // the chunk's sums are read before the next chunk's are written
  }
  // rows behind the last request: no slot, nothing visible
  for (int64_t i = rows_base + at0; i < p.rows; i += step) {
    p.slots[i] = -1;
    p.positions[i] = 0;
    p.request[i] = 0;
    p.lens[i] = 0;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0)
    *p.pages_used = (int32_t)min(pages_base, (long long)p.num_free);
  if (bits) set_error(p.err, bits);
}

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_step_layout(const int32_t* seq_lens, const int32_t* query_lens, int64_t batch,
                               int32_t* block_table, int64_t block_table_stride, int64_t max_pages,
                               const int32_t* free_pages, int64_t num_free, const int32_t* prefix_len,
                               int64_t num_tokens, int32_t* slots, int32_t* positions,
                               int32_t* token_request, int32_t* token_lens, int32_t* pages_used,
                               int* device_error, void* stream) {
  if (batch < 0 || max_pages < 0 || num_free < 0 || num_tokens < 0)
    return report_error(DSA_ERR_INVALID_ARG, "negative size");
  if (batch > INT32_MAX || num_tokens > INT32_MAX || num_free > INT32_MAX)
    return report_error(DSA_ERR_UNSUPPORTED, "requests, rows and free pages are counted in 32 bits");
  if (!pages_used || (batch > 0 && (!seq_lens || !query_lens)) ||
      (batch > 0 && max_pages > 0 && !block_table) || (num_free > 0 && !free_pages) ||
      (num_tokens > 0 && (!slots || !positions || !token_request || !token_lens)))
    return report_error(DSA_ERR_INVALID_ARG, "NULL pointer argument");
  if (batch > 1 && block_table_stride < max_pages)
    return report_error(DSA_ERR_INVALID_ARG, "block table rows overlap");
  LayoutParams p;
  p.seq = seq_lens;
  p.query = query_lens;
  p.free_pages = free_pages;
  p.prefix_len = prefix_len;
  p.table = block_table;
  p.slots = slots;
  p.positions = positions;
  p.request = token_request;
  p.lens = token_lens;
  p.pages_used = pages_used;
  p.batch = batch;
  p.bt_stride = block_table_stride;
  p.max_pages = max_pages;
  p.num_free = num_free;
  p.rows = num_tokens;
  p.err = device_error;
  const int64_t ctas = (num_tokens + kLayThreads - 1) / kLayThreads;
  dsa_step_layout_kernel<<<(unsigned)(ctas < 1 ? 1 : ctas > 148 ? 148 : ctas), kLayThreads, 0,
                           static_cast<cudaStream_t>(stream)>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return report_error(DSA_ERR_CUDA, cudaGetErrorString(e));
  return DSA_OK;
}
