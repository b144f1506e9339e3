// Block tables of the HiF8 paged KV cache, kept on the GPU, for gfx950: pages for
// a step's new tokens are taken from a stack of free page ids and the tokens'
// slots worked out (hif8_extend_block_tables), and pages that no later token
// needs go back onto it (hif8_release_blocks).
//
// The state is the table and the stack alone: an entry below zero holds no page.
// Ids are taken from the top of the stack, and put there, in the order (request,
// table column), so both calls are prefix sums and repeat themselves exactly.
#include <stddef.h>

#include <algorithm>

#include "hif8_common.h"

namespace hif8 {
namespace {

constexpr int kScan = 1024;  // threads of a workgroup that ranks entries: sixteen wavefronts
constexpr int kScanWaves = kScan / kWave;
constexpr int kRowThreads = 256;

// A request's new query rows, clipped to the call's rows (start_loc is caller data).
__device__ __forceinline__ void new_rows(const int32_t *start_loc, int b, int total, int &begin, int &count) {
  begin = max(start_loc[b], 0);
  count = max(min(start_loc[b + 1], total) - begin, 0);
}

// Exclusive sum over the workgroup of what each thread counts; `all` gets the total.
// sums: kScanWaves + 1 ints of LDS, free again after the next barrier.
__device__ __forceinline__ int block_exclusive(int mine, int *sums, int &all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int left = __shfl_up(upto, o, kWave);
    if (lane >= o) upto += left;
  }
  if (lane == kWave - 1) sums[wave] = upto;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kScanWaves; ++w) {
    const int s = sums[w];
    before += w < wave ? s : 0;
    all += s;
  }
  __syncthreads();
  return before + upto - mine;
}

struct ExtendParams {
  void *table;               // [batch, width]
  const int32_t *free_ids;   // [capacity]
  int32_t *free_count;       // [1]
  const int32_t *lens;       // [batch]
  const int32_t *start_loc;  // [batch + 1]
  int64_t *slots, *positions;
  int32_t *new_lens, *missing;
  int64_t width, capacity;
  int batch, total, block_size;
};

// Ids for the table columns that the new tokens reach.  One workgroup: the rank of
// a column among those without a page runs over all requests.
template <typename BtT>
__global__ __launch_bounds__(kScan) void extend_kernel(const ExtendParams p) {
  __shared__ int first[kScan + 1];  // columns of the chunk's requests before each
  __shared__ int low[kScan];        // a request's first column
  __shared__ int lack[kScan];       // pages that it did not get
  __shared__ int sums[kScanWaves];
  const int tid = threadIdx.x;
  const int have = int(min(int64_t(max(*p.free_count, 0)), p.capacity));
  int64_t taken = 0;  // columns without a page so far
  for (int base = 0; base < p.batch; base += kScan) {
    const int b = base + tid;
    int columns = 0, lo = 0, beyond = 0;
    if (b < p.batch) {
      int begin, n;
      new_rows(p.start_loc, b, p.total, begin, n);
      const int64_t ctx = max(p.lens[b], 0), end = ctx + n;
      p.new_lens[b] = int32_t(min(end, int64_t(0x7FFFFFFF)));
      if (n > 0) {
        const int64_t l = ctx / p.block_size, h = (end + p.block_size - 1) / p.block_size;
        lo = int(min(l, p.width));
        columns = int(min(h, p.width)) - lo;
        beyond = int(h - max(l, min(h, p.width)));
      }
    }
    int total;
    first[tid] = block_exclusive(columns, sums, total);
    low[tid] = lo;
    lack[tid] = beyond;
    __syncthreads();
    for (int c0 = 0; c0 < total; c0 += kScan) {
      const int c = c0 + tid;
      int r = 0;
      BtT *entry = nullptr;
      bool wants = false;
      if (c < total) {
        // The last request of the chunk that starts at or before column c.
        int hi = kScan - 1;
        while (r < hi) {
          const int mid = (r + hi + 1) / 2;
          if (first[mid] <= c) r = mid;
          else hi = mid - 1;
        }
        entry = static_cast<BtT *>(p.table) + int64_t(base + r) * p.width + (low[r] + c - first[r]);
        wants = *entry < 0;
      }
      int here;
      const int64_t rank = taken + block_exclusive(wants ? 1 : 0, sums, here);
      if (wants) {
        if (rank < have) *entry = BtT(p.free_ids[have - 1 - rank]);
        else atomicAdd(&lack[r], 1);
      }
      taken += here;
    }
    __syncthreads();
    if (b < p.batch) p.missing[b] = lack[tid];
    __syncthreads();
  }
  if (tid == 0) *p.free_count = int32_t(have - min(taken, int64_t(have)));
}

// Slot and position of every row, from the table as extend_kernel has left it.
template <typename BtT>
__global__ __launch_bounds__(kRowThreads) void slots_kernel(const ExtendParams p) {
  const int row = int(blockIdx.x) * kRowThreads + threadIdx.x;
  if (row >= p.total) return;
  int lo = 0, hi = p.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (p.start_loc[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  int begin, n;
  new_rows(p.start_loc, lo, p.total, begin, n);
  int64_t slot = -1, at = -1;  // a row of no request: padding
  if (row >= begin && row - begin < n) {
    at = int64_t(max(p.lens[lo], 0)) + (row - begin);
    const int64_t col = at / p.block_size;
    const int64_t page = col < p.width ? int64_t(static_cast<const BtT *>(p.table)[int64_t(lo) * p.width + col]) : -1;
    if (page >= 0) slot = page * p.block_size + (at - col * p.block_size);
  }
  p.slots[row] = slot;
  p.positions[row] = at;
}

struct ReleaseParams {
  void *table;
  int32_t *free_ids;
  int32_t *free_count;
  const int32_t *lens;
  int32_t *counts;  // [chunks] pages that go, then the stack's count before the call
  int64_t width, capacity, entries;
  int64_t window;   // 0: none
  int64_t sinks;
  int block_size, chunks;
};

constexpr int kPer = 4;                   // consecutive entries per thread
constexpr int kChunk = kScan * kPer;

// Whether request b goes on needing the page of its column `col`.
__device__ __forceinline__ bool stays(const ReleaseParams &p, int64_t b, int64_t col) {
  const int64_t len = max(p.lens[b], 0), from = col * p.block_size;
  if (from >= len) return false;
  return p.window == 0 || from < p.sinks || from + p.block_size > len + 1 - p.window;
}

// Bit i: entry first + i holds a page that goes.
template <typename BtT>
__device__ __forceinline__ uint32_t goers(const ReleaseParams &p, int64_t first, BtT (&ids)[kPer]) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t e = first + i;
    ids[i] = -1;
    if (e >= p.entries) continue;
    ids[i] = static_cast<const BtT *>(p.table)[e];
    const int64_t b = e / p.width;
    if (ids[i] >= 0 && !stays(p, b, e - b * p.width)) bits |= 1u << i;
  }
  return bits;
}

template <typename BtT>
__global__ __launch_bounds__(kScan) void release_count_kernel(const ReleaseParams p) {
  __shared__ int sums[kScanWaves];
  BtT ids[kPer];
  const uint32_t bits = goers(p, int64_t(blockIdx.x) * kChunk + int64_t(threadIdx.x) * kPer, ids);
  int all;
  block_exclusive(__popc(bits), sums, all);
  if (threadIdx.x == 0) {
    p.counts[blockIdx.x] = all;
    if (blockIdx.x == 0) p.counts[p.chunks] = *p.free_count;
  }
}

template <typename BtT>
__global__ __launch_bounds__(kScan) void release_kernel(const ReleaseParams p) {
  __shared__ int sums[kScanWaves];
  const int have = int(min(int64_t(max(p.counts[p.chunks], 0)), p.capacity));
  int mine = 0;
  for (int i = threadIdx.x; i < int(blockIdx.x); i += kScan) mine += p.counts[i];
  int before;
  block_exclusive(mine, sums, before);
  BtT ids[kPer];
  const int64_t first = int64_t(blockIdx.x) * kChunk + int64_t(threadIdx.x) * kPer;
  const uint32_t bits = goers(p, first, ids);
  int here;
  int64_t place = int64_t(have) + before + block_exclusive(__popc(bits), sums, here);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (!((bits >> i) & 1u)) continue;
    if (place < p.capacity) {  // a stack that is full leaves the page where it is
      p.free_ids[place] = int32_t(ids[i]);
      static_cast<BtT *>(p.table)[first + i] = BtT(-1);
    }
    ++place;
  }
  if (int(blockIdx.x) == p.chunks - 1 && threadIdx.x == 0)
    *p.free_count = int32_t(min(int64_t(have) + before + here, p.capacity));
}

int64_t chunks_of(int64_t batch, int64_t width) { return (batch * width + kChunk - 1) / kChunk; }

}  // namespace
}  // namespace hif8

using namespace hif8;

extern "C" int hif8_extend_block_tables(void *block_table, int block_table_dtype, int64_t max_blocks_per_seq,
                                        const int32_t *free_blocks, int64_t free_capacity, int32_t *free_count,
                                        const int32_t *context_lens, const int32_t *query_start_loc, int64_t batch,
                                        int64_t total_query_tokens, int64_t block_size, int64_t *slot_mapping,
                                        int64_t *positions, int32_t *seq_lens, int32_t *missing,
                                        hif8_stream_t stream) {
  static const char *kName = "hif8_extend_block_tables";
  clear_error();
  if (max_blocks_per_seq <= 0 || free_capacity < 0 || batch < 0 || total_query_tokens < 0 || block_size <= 0)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions must be positive", kName);
  if (block_table_dtype != HIF8_INDEX_INT32 && block_table_dtype != HIF8_INDEX_INT64)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: block_table must be int32 or int64", kName);
  if (max_blocks_per_seq > 0x3FFFFFll || block_size > 0x7FFFFFFFll || free_capacity > 0x7FFFFFFFll ||
      batch > 0xFFFFFFll || total_query_tokens > 0x7FFFFF00ll)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", kName);
  if (batch == 0 && total_query_tokens == 0) return HIF8_OK;
  if (!query_start_loc || (total_query_tokens && (!slot_mapping || !positions)) ||
      (batch && (!block_table || !free_count || !context_lens || !seq_lens || !missing)) ||
      (free_capacity && !free_blocks))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: null pointer argument", kName);
  ExtendParams p{block_table, free_blocks, free_count, context_lens, query_start_loc, slot_mapping, positions,
                 seq_lens, missing, max_blocks_per_seq, free_capacity, int(batch), int(total_query_tokens),
                 int(block_size)};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool i64 = block_table_dtype == HIF8_INDEX_INT64;
  if (batch > 0) {
    if (i64) extend_kernel<int64_t><<<1, kScan, 0, s>>>(p);
    else extend_kernel<int32_t><<<1, kScan, 0, s>>>(p);
  }
  if (total_query_tokens > 0) {
    const unsigned blocks = unsigned((total_query_tokens + kRowThreads - 1) / kRowThreads);
    if (i64) slots_kernel<int64_t><<<blocks, kRowThreads, 0, s>>>(p);
    else slots_kernel<int32_t><<<blocks, kRowThreads, 0, s>>>(p);
  }
  return check_launch(kName);
}

extern "C" size_t hif8_release_blocks_workspace_size(int64_t batch, int64_t max_blocks_per_seq) {
  if (batch <= 0 || max_blocks_per_seq <= 0) return 0;
  return size_t(chunks_of(batch, max_blocks_per_seq) + 1) * sizeof(int32_t);
}

extern "C" int hif8_release_blocks(void *block_table, int block_table_dtype, int64_t max_blocks_per_seq,
                                   int32_t *free_blocks, int64_t free_capacity, int32_t *free_count,
                                   const int32_t *seq_lens, int64_t batch, int64_t block_size, int64_t window,
                                   int64_t sinks, void *workspace, size_t workspace_bytes, hif8_stream_t stream) {
  static const char *kName = "hif8_release_blocks";
  clear_error();
  if (max_blocks_per_seq <= 0 || free_capacity < 0 || batch < 0 || block_size <= 0)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions must be positive", kName);
  if (window < 0 || sinks < 0) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: window and sinks must not be negative", kName);
  if (block_table_dtype != HIF8_INDEX_INT32 && block_table_dtype != HIF8_INDEX_INT64)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: block_table must be int32 or int64", kName);
  if (max_blocks_per_seq > 0x3FFFFFll || block_size > 0x7FFFFFFFll || free_capacity > 0x7FFFFFFFll ||
      batch > 0xFFFFFFll || batch * max_blocks_per_seq > 0x7FFFFFFFll)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", kName);
  if (batch == 0) return HIF8_OK;
  if (!block_table || !free_count || !seq_lens || (free_capacity && !free_blocks))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: null pointer argument", kName);
  const size_t need = hif8_release_blocks_workspace_size(batch, max_blocks_per_seq);
  if (!workspace || workspace_bytes < need)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes required (got %zu)", kName, need,
                workspace_bytes);
  if (!aligned(workspace, 4)) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace must be 4-byte aligned", kName);
  ReleaseParams p{block_table, free_blocks, free_count, seq_lens, static_cast<int32_t *>(workspace),
                  max_blocks_per_seq, free_capacity, batch * max_blocks_per_seq,
                  window, std::min<int64_t>(sinks, 0x7FFFFFFFll), int(block_size),
                  int(chunks_of(batch, max_blocks_per_seq))};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (block_table_dtype == HIF8_INDEX_INT64) {
    release_count_kernel<int64_t><<<unsigned(p.chunks), kScan, 0, s>>>(p);
    release_kernel<int64_t><<<unsigned(p.chunks), kScan, 0, s>>>(p);
  } else {
    release_count_kernel<int32_t><<<unsigned(p.chunks), kScan, 0, s>>>(p);
    release_kernel<int32_t><<<unsigned(p.chunks), kScan, 0, s>>>(p);
  }
  return check_launch(kName);
}
