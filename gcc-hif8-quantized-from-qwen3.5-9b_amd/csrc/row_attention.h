// Shared by the two operators that run a few query rows per request over the
// whole HiF8 paged cache: attention of drafted tokens under a tree mask, and
// decode attention that also accumulates every cached row's softmax weight.
#pragma once

#include "hif8_common.h"

namespace hif8 {

// Request b owns query rows start_loc[b] .. start_loc[b + 1] - 1 (start_loc
// null: row b alone).  It has lens[b] rows that every query row sees; under a
// tree mask the rows behind them, one per query row of the request, are its
// drafts, and query row i sees draft j where mask[row of i][j] is not zero.
struct RowAttnParams {
  const void *query;           // [total_q, Hq, D]
  const uint8_t *key_cache;    // [num_blocks, block_size, Hkv, D + 4]
  const uint8_t *value_cache;  // [num_blocks, block_size, Hkv, Dv + 4]
  const void *block_table;     // [batch, bt_stride] int32 or int64
  const int32_t *start_loc;    // [batch + 1] or null
  const int32_t *lens;         // [batch]
  const uint8_t *mask;         // [total_q, mask_stride] or null
  void *out;                   // [total_q, Hq, Dv]
  // Partial outputs and (maximum, sum): any-shape kernel [total_q * Hq, num_splits] (outputs: two splits or more),
  // matrix cores [2 workers, Hkv, rows_cap] and [workers + batch, Hkv, rows_cap].
  float *part_o;
  float *part_ml;
  int32_t *plan;               // matrix cores: [batch + 1] tiles before each request
  float *x;                    // [total_q * Hq, x_stride] base-2 logits, or null
  float *weights;              // [batch, Hkv, w_stride], or null
  int64_t bt_stride, num_blocks, mask_stride, x_stride, w_stride;
  int block_size, hkv, hq, group, d, dv, batch, total_q, max_len, num_splits, split_tokens, accumulate;
  int zero_rest;               // query rows of no request get zeros (else they are left as they were)
  // Matrix cores: workers that share the tiles, row tiles of the longest request,
  // query rows of all of them (a KV head's), ceil(2^31 / group).
  int workers, row_tiles, rows_cap, heads_together;
  uint32_t group_magic;
  float scale_log2;            // softmax scale * log2(e)
};

__device__ __forceinline__ int clamp_rows(int n, int most) { return n < 0 ? 0 : (n > most ? most : n); }

// Cache rows that some query row of a request may see: its context, and as many
// drafts as it has query rows (and the mask columns).
__device__ __forceinline__ int rows_seen(const RowAttnParams &p, int ctx, int count) {
  return p.mask ? clamp_rows(ctx + int(min(int64_t(count), p.mask_stride)), p.max_len) : ctx;
}

// Query rows of request b, clipped to the query tensor (start_loc is caller data).
__device__ __forceinline__ void request_rows(const RowAttnParams &p, int b, int &begin, int &count) {
  if (!p.start_loc) {
    begin = b;
    count = 1;
    return;
  }
  begin = max(p.start_loc[b], 0);
  count = max(min(p.start_loc[b + 1], p.total_q) - begin, 0);
}

// The request of a query row, or -1: the last b with start_loc[b] <= row.
__device__ __forceinline__ int request_of_row(const RowAttnParams &p, int row) {
  if (!p.start_loc) return row;
  int lo = 0, hi = p.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (p.start_loc[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  int begin, count;
  request_rows(p, lo, begin, count);
  return row >= begin && row - begin < count ? lo : -1;
}

}  // namespace hif8
