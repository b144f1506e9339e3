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
#include <type_traits>

#include "mfma_lookup.h"  // wave_prefix

namespace hif8 {
namespace {

constexpr int kScan = 1024;  // threads of a workgroup that ranks entries: sixteen wavefronts
constexpr int kScanWaves = kScan / kWave;
constexpr int kRowThreads = 256;

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
  int with_slots;            // the workgroup that takes the ids works out the slots too
};

constexpr int kPerThread = 8;  // columns of a thread where there are more than threads
// Rows up to which one workgroup does all of a call.  Against a kernel of its own for the
// slots, 8 requests in a graph: 8 rows 4.4 and 5.3 us, 1024 4.8 and 5.7, 2048 5.7 and 5.7,
// 4096 7.4 and 5.7; outside a graph the second launch is also 4 us of the host's.
constexpr int kFewRows = 2048;

// Slot and position of a row, from the table as it stands; of a row of no request -1.
template <typename BtT>
__device__ __forceinline__ void put_slot(const ExtendParams &p, int row, int b, int begin, int n) {
  int64_t slot = -1, at = -1;
  if (row >= begin && row - begin < n) {
    at = int64_t(max(p.lens[b], 0)) + (row - begin);
    const int64_t col = uint64_t(at) >> 32 ? at / p.block_size : int64_t(uint32_t(at) / uint32_t(p.block_size));
    const int64_t page = col < p.width ? int64_t(static_cast<const BtT *>(p.table)[int64_t(b) * p.width + col]) : -1;
    if (page >= 0) slot = page * p.block_size + (at - col * p.block_size);
  }
  p.slots[row] = slot;
  p.positions[row] = at;
}

// Ids for the table columns that the new tokens reach.  One workgroup: the rank of
// a column among those without a page runs over all requests.  Bound by the dependent
// reads of lengths, table and stack (four round trips, 4.3 us with a new token each).  48
// prompts of 4k tokens on 16-token pages, 9200 columns: 12.9 us; with one column a thread
// and pass 19.
template <typename BtT>
__global__ __launch_bounds__(kScan) void extend_kernel(const ExtendParams p) {
  __shared__ int first[kScan];      // columns of the chunk's requests before each
  __shared__ int low[kScan];        // a request's first column
  __shared__ int lack[kScan];       // pages that it did not get
  __shared__ int sums[kScanWaves], counts[kPerThread * kScanWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int have = int(min(int64_t(max(*p.free_count, 0)), p.capacity));
  int64_t taken = 0;  // columns without a page so far
  for (int base = 0; base < p.batch; base += kScan) {
    const int b = base + tid;
    int columns = 0, lo = 0, beyond = 0;
    if (b < p.batch) {
      int begin, n;
      clipped_rows(p.start_loc, b, p.total, begin, n);
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
    auto columns_of = [&](auto per) {
      constexpr int kPer = decltype(per)::value;
      for (uint32_t c0 = 0; c0 < uint32_t(total); c0 += kScan * kPer) {  // unsigned: total may come near 2^31
        // Column c0 + kScan j + tid: its request is the last of the chunk that starts at or before it.
        int owner[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) owner[j] = 0;
#pragma unroll
        for (int step = kScan / 2; step > 0; step /= 2)
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (uint32_t(first[owner[j] + step]) <= c0 + kScan * j + tid) owner[j] += step;
        BtT *entry[kPer], id[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const uint32_t c = c0 + kScan * j + tid;
          const int r = owner[j];
          // `first` wraps past 2^31 as c does (starts that go back and forth give every request many rows).
          entry[j] = static_cast<BtT *>(p.table) + int64_t(base + r) * p.width + low[r] + int64_t(c - uint32_t(first[r]));
          id[j] = c < uint32_t(total) ? *entry[j] : BtT(0);
        }
        uint64_t wants[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          wants[j] = __ballot(id[j] < 0);
          if (lane == 0) counts[j * kScanWaves + wave] = __popcll(wants[j]);
        }
        __syncthreads();
        // Those of the 16 wavefronts, one j after the other: before[i] of count i.
        constexpr int kCounts = kPer * kScanWaves;
        int upto[(kCounts + kWave - 1) / kWave], all = 0;
#pragma unroll
        for (int i = 0; i < (kCounts + kWave - 1) / kWave; ++i) {
          const int mine = kWave * i + lane < kCounts ? counts[kWave * i + lane] : 0;
          upto[i] = all + wave_prefix(mine);
          all = __builtin_amdgcn_readlane(upto[i], kWave - 1);
          upto[i] -= mine;
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int i = j * kScanWaves + wave;
          const int64_t rank = taken + __builtin_amdgcn_readlane(upto[j * kScanWaves / kWave], i % kWave) +
                               __popcll(wants[j] & ((uint64_t(1) << lane) - 1));
          if (id[j] >= 0) continue;
          if (rank < have) *entry[j] = BtT(p.free_ids[have - 1 - rank]);
          else atomicAdd(&lack[owner[j]], 1);
        }
        taken += all;
        __syncthreads();
      }
    };
    if (total <= kScan) columns_of(std::integral_constant<int, 1>{});
    else columns_of(std::integral_constant<int, kPerThread>{});
    __syncthreads();
    if (b < p.batch) p.missing[b] = lack[tid];
    __syncthreads();
  }
  if (tid == 0) *p.free_count = int32_t(have - min(taken, int64_t(have)));
  if (!p.with_slots) return;  // uniform; here the batch is one chunk
  for (int i = tid; i < p.batch; i += kScan) first[i] = p.start_loc[i];
  __syncthreads();
  for (int row = tid; row < p.total; row += kScan) {
    int b = 0, hi = p.batch - 1;
    while (b < hi) {
      const int mid = (b + hi + 1) / 2;
      if (first[mid] <= row) b = mid;
      else hi = mid - 1;
    }
    int begin, n;
    clipped_rows(p.start_loc, b, p.total, begin, n);
    put_slot<BtT>(p, row, b, begin, n);
  }
}

// Slots and positions of many rows, from the table as extend_kernel has left it.
template <typename BtT>
__global__ __launch_bounds__(kRowThreads) void slots_kernel(const ExtendParams p) {
  const int row = int(blockIdx.x) * kRowThreads + threadIdx.x;
  if (row >= p.total) return;
  int b = 0, hi = p.batch - 1;
  while (b < hi) {
    const int mid = (b + hi + 1) / 2;
    if (p.start_loc[mid] <= row) b = mid;
    else hi = mid - 1;
  }
  int begin = 0, n = 0;
  if (p.batch > 0) clipped_rows(p.start_loc, b, p.total, begin, n);
  put_slot<BtT>(p, row, b, begin, n);
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

// Whether a request of len rows goes on needing the page of its column `col`.
__device__ __forceinline__ bool stays(const ReleaseParams &p, int64_t len, int64_t col) {
  const int64_t from = col * p.block_size;
  if (from >= len) return false;
  return p.window == 0 || from < p.sinks || from + p.block_size > len + 1 - p.window;
}

// Bit i: entry first + i holds a page that goes.
template <typename BtT>
__device__ __forceinline__ uint32_t goers(const ReleaseParams &p, int64_t first, BtT (&ids)[kPer]) {
  const BtT *table = static_cast<const BtT *>(p.table);
  if (first + kPer <= p.entries) {
    typedef BtT vec __attribute__((ext_vector_type(kPer), aligned(sizeof(BtT))));
    const vec v = *reinterpret_cast<const vec *>(table + first);
#pragma unroll
    for (int i = 0; i < kPer; ++i) ids[i] = v[i];
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) ids[i] = first + i < p.entries ? table[first + i] : BtT(-1);
  }
  uint32_t held = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) held |= ids[i] >= 0 ? 1u << i : 0u;
  if (!held) return 0;  // most of a table is empty
  uint32_t b = uint32_t(first) / uint32_t(p.width), col = uint32_t(first) - b * uint32_t(p.width), bits = 0;
  int64_t len = max(p.lens[b], 0);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if ((held >> i) & 1u) bits |= stays(p, len, col) ? 0u : 1u << i;
    if (++col == uint32_t(p.width) && first + i + 1 < p.entries) {
      col = 0;
      len = max(p.lens[++b], 0);
    }
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

// A workgroup per kChunk entries; what the earlier ones release has been counted, unless
// one workgroup has them all (8 requests of 25 columns 3.0 us).  256 requests of 2049 columns,
// 2.1 MB of table: 4.2 + 6.2 us, two reads of the table and a launch's latency each.
template <typename BtT>
__global__ __launch_bounds__(kScan) void release_kernel(const ReleaseParams p) {
  __shared__ int sums[kScanWaves];
  const int stack = p.chunks > 1 ? p.counts[p.chunks] : *p.free_count;
  const int have = int(min(int64_t(max(stack, 0)), p.capacity));
  int before = 0;
  if (p.chunks > 1) {
    int mine = 0;
    for (int i = threadIdx.x; i < int(blockIdx.x); i += kScan) mine += p.counts[i];
    block_exclusive(mine, sums, before);
  }
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
  if (batch && share(context_lens, seq_lens, batch))  // the slots are worked out from the lengths before
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: seq_lens must not overlap context_lens", kName);
  ExtendParams p{block_table, free_blocks, free_count, context_lens, query_start_loc, slot_mapping, positions,
                 seq_lens, missing, max_blocks_per_seq, free_capacity, int(batch), int(total_query_tokens),
                 int(block_size), batch <= kScan && total_query_tokens <= kFewRows ? 1 : 0};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool i64 = block_table_dtype == HIF8_INDEX_INT64;
  if (batch > 0) {
    if (i64) extend_kernel<int64_t><<<1, kScan, 0, s>>>(p);
    else extend_kernel<int32_t><<<1, kScan, 0, s>>>(p);
  }
  if (total_query_tokens > 0 && (batch == 0 || !p.with_slots)) {
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
    if (p.chunks > 1) release_count_kernel<int64_t><<<unsigned(p.chunks), kScan, 0, s>>>(p);
    release_kernel<int64_t><<<unsigned(p.chunks), kScan, 0, s>>>(p);
  } else {
    if (p.chunks > 1) release_count_kernel<int32_t><<<unsigned(p.chunks), kScan, 0, s>>>(p);
    release_kernel<int32_t><<<unsigned(p.chunks), kScan, 0, s>>>(p);
  }
  return check_launch(kName);
}
