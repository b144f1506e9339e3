// Shared by the operators that run a few query rows per request over the HiF8
// paged cache: attention of drafted tokens under a tree mask, decode attention
// that also accumulates every cached row's softmax weight, and attention within a
// sliding window.
#pragma once

#include <stddef.h>

#include "hif8_common.h"

namespace hif8 {

// Request b owns query rows start_loc[b] .. start_loc[b + 1] - 1 (start_loc
// null: row b alone).  It has lens[b] rows that every query row sees; under a
// tree mask the rows behind them, one per query row of the request, are its
// drafts, and query row i sees draft j where mask[row of i][j] is not zero.
// With a window (no mask) lens[b] counts the request's query rows too: they are its
// last positions, and the one at position P sees the rows t <= P with t > P - window
// or t < sinks.
struct RowAttnParams {
  const void *query;           // [total_q, Hq, D]
  const uint8_t *key_cache;    // [num_blocks, block_size, Hkv, D + 4]
  const uint8_t *value_cache;  // [num_blocks, block_size, Hkv, Dv + 4]
  const void *block_table;     // [batch, bt_stride] int32 or int64
  const int32_t *start_loc;    // [batch + 1] or null
  const int32_t *lens;         // [batch]
  const uint8_t *mask;         // [total_q, mask_stride] or null
  void *out;                   // [total_q, Hq, Dv]
  // Partial outputs and (maximum, sum): any-shape kernel [total_q * Hq, num_splits] (two splits or more; with weights
  // (maximum, sum) of one too),
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
  int window, sinks;           // window 0: none
  int most_rows;               // window: bound of WindowRows::rows
  int long_rows;               // window: requests of more (token, head) rows per KV head are not these kernels'
  float scale_log2;            // softmax scale * log2(e)
};

__device__ __forceinline__ int clamp_rows(int n, int most) { return n < 0 ? 0 : (n > most ? most : n); }

// Cache rows that some query row of a request may see: its context, and as many
// drafts as it has query rows (and the mask columns).
__device__ __forceinline__ int rows_seen(const RowAttnParams &p, int ctx, int count) {
  return p.mask ? clamp_rows(ctx + int(min(int64_t(count), p.mask_stride)), p.max_len) : ctx;
}

// The cache rows that the query rows of a request see under a window, pushed
// together in groups of 16: `head` rows from the first on, then those behind the
// `skip` rows that no query row sees.  `rows` of them.
struct WindowRows {
  int head, skip, rows;
  // The cache row of pushed-together row t (of its group of 16, where t starts one).
  __device__ int real(int t) const { return t < head ? t : t + skip; }
};

__device__ __forceinline__ WindowRows window_rows(const RowAttnParams &p, int len, int count) {
  const int low = int(max(int64_t(len) - count + 1 - p.window, int64_t(0))) & ~15;  // of the first query row
  const int head = int(min((int64_t(p.sinks) + 15) & ~int64_t(15), int64_t(low)));
  return WindowRows{head, low - head, min(len - (low - head), p.most_rows)};
}

// Whether the query row at position `at` sees cache row t.
__device__ __forceinline__ bool window_sees(const RowAttnParams &p, int at, int t) {
  return t <= at && (int64_t(t) > int64_t(at) - p.window || t < p.sinks);
}

// Query rows that another kernel takes.
__device__ __forceinline__ bool left_out(const RowAttnParams &p, int count) {
  return p.window && int64_t(count) * p.group > p.long_rows;
}

// Query rows of request b, clipped to the query tensor (start_loc is caller data).
__device__ __forceinline__ void request_rows(const RowAttnParams &p, int b, int &begin, int &count) {
  if (!p.start_loc) {
    begin = b;
    count = 1;
    return;
  }
  clipped_rows(p.start_loc, b, p.total_q, begin, count);
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

// Host side: a call's arguments, and the call (row_attention.hip).  long_rows: requests
// of more (token, head) rows per KV head are left to another kernel (window; 0: none).
struct RowArgs {
  const void *query;
  int q_dtype;
  const uint8_t *key_cache, *value_cache;
  int64_t num_blocks, block_size, hkv, d, dv;
  const void *block_table;
  int bt_dtype;
  int64_t max_blocks;
  const int32_t *start_loc, *lens;
  const uint8_t *mask;
  int64_t mask_stride, batch, heads, total_q, max_query, max_len;
  float scale;
  void *out;
  float *weights;
  int64_t w_stride;
  int accumulate;
  int zero_rest;
  void *workspace;
  size_t workspace_bytes;
  hif8_stream_t stream;
  int64_t window, sinks, long_rows;
};

int check_row_args(const char *name, const RowArgs &a);  // the arguments alone, without the workspace
int row_attention(const char *name, const RowArgs &a);
// Its workspace; max_len as rows_bound gives it.
size_t row_workspace(int64_t batch, int64_t total_q, int64_t heads, int64_t hkv, int64_t d, int64_t dv,
                     int64_t block_size, int64_t max_query, int64_t max_len, bool weights);
// Cache rows of a request that its query rows can see: all of them, or the window's
// (WindowRows: whole groups of 16).
int64_t rows_bound(int64_t max_len, int64_t max_query, int64_t window, int64_t sinks);

}  // namespace hif8
