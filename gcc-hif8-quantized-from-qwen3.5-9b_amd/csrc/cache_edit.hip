// Edits of the HiF8 paged KV cache in place, for gfx950: the rows of an accepted
// draft path move to the end of the context, and the rows of least accumulated
// attention weight are dropped.  Both move whole rows (codes and scale), byte
// for byte, and are bound by the bytes of the rows that move.
#include <stddef.h>

#include <algorithm>

#include "hif8_common.h"

namespace hif8 {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int clamp_rows(int n, int most) { return n < 0 ? 0 : (n > most ? most : n); }

// First flat slot of the page of a request's row, or -1.
template <typename BtT>
__device__ __forceinline__ int64_t slot_of(const BtT *bt, int64_t row, int64_t width, int block_size,
                                           int64_t num_blocks) {
  const int64_t col = row / block_size;
  if (row < 0 || col >= width) return -1;
  const int64_t blk = int64_t(bt[col]);
  return blk < 0 || blk >= num_blocks ? int64_t(-1) : blk * block_size + row % block_size;
}

// --------------------------------------------------------------- acceptance

constexpr int kMaxCaches = 128;  // caches (K and V of every layer) of one launch

struct AcceptParams {
  uint32_t *cache[kMaxCaches];  // [num_blocks, block_size, words]
  int words[kMaxCaches];        // 4-byte words of one token's rows, all KV heads
  const void *block_table;
  const int32_t *lens;          // [batch] rows before the drafts
  const int32_t *path;          // [batch, path_width] draft indices, rising
  const int32_t *counts;        // [batch]
  int32_t *new_lens;            // [batch]
  int64_t bt_stride, num_blocks;
  int block_size, path_width, caches;
};

// Row lens[b] + path[b][i] -> row lens[b] + i for i < counts[b], in every cache.
// A thread owns one 4-byte column of the rows and moves them in order, eight
// loads ahead of eight stores.  path rises, so path[j] >= j and a row that is
// written is never read later: the move is in place and needs no barrier.
template <typename BtT>
__global__ __launch_bounds__(kThreads) void accept_kernel(const AcceptParams p) {
  constexpr int kAhead = 8;
  const int b = blockIdx.x, c = blockIdx.y;
  const int col = int(blockIdx.z) * kThreads + threadIdx.x;
  const int ctx = max(p.lens[b], 0), count = clamp_rows(p.counts[b], p.path_width);
  if (c == 0 && blockIdx.z == 0 && threadIdx.x == 0 && p.new_lens) p.new_lens[b] = ctx + count;
  const int words = p.words[c];
  if (col >= words) return;
  const BtT *bt = static_cast<const BtT *>(p.block_table) + size_t(b) * p.bt_stride;
  const int32_t *path = p.path + size_t(b) * p.path_width;
  uint32_t *cache = p.cache[c] + col;
  for (int i0 = 0; i0 < count; i0 += kAhead) {
    uint32_t w[kAhead];
    int64_t to[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j;
      to[j] = -1;
      w[j] = 0;
      if (i < count) {
        const int a = path[i];
        const int64_t from =
            a < 0 || a == i ? int64_t(-1) : slot_of(bt, int64_t(ctx) + a, p.bt_stride, p.block_size, p.num_blocks);
        if (from >= 0) {
          to[j] = slot_of(bt, int64_t(ctx) + i, p.bt_stride, p.block_size, p.num_blocks);
          w[j] = cache[from * words];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (to[j] >= 0) cache[to[j] * words] = w[j];
  }
}

// ----------------------------------------------------------------- eviction

struct EvictParams {
  uint32_t *key_cache, *value_cache;  // rows of key_words / value_words 4-byte words
  const void *block_table;
  const int32_t *lens, *keep, *protect_from;  // [batch]; keep, protect_from may be null
  float *weights;                      // [batch, Hkv, w_stride]
  int32_t *positions;                  // [batch, Hkv, w_stride] or null
  int32_t *new_lens;                   // [batch]
  int32_t *moves;                      // [batch * Hkv, 2, move_stride]: to, from
  int32_t *move_counts;                // [batch * Hkv]
  int64_t bt_stride, num_blocks, w_stride, move_stride;
  int block_size, hkv, key_words, value_words, max_len, keep_all, sinks;
};

// Larger is kept first: protected rows, then weights in falling order, NaN last.
__device__ __forceinline__ uint32_t rank_of(float w, bool safe) {
  if (safe) return 0xFFFFFFFFu;
  if (__builtin_isnan(w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 counts as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;

// Exclusive prefix of a flag over the workgroup, and the total.
__device__ __forceinline__ int block_rank(bool flag, int *red, int &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t ball = __ballot(flag);
  const int before = __popcll(ball & ((uint64_t(1) << lane) - 1));
  __syncthreads();
  if (lane == 0) red[wave] = __popcll(ball);
  __syncthreads();
  int base = 0;
  total = 0;
  for (int w = 0; w < kSelWaves; ++w) {
    if (w < wave) base += red[w];
    total += red[w];
  }
  return base + before;
}

// One workgroup per (request, KV head): the rank of the last kept row by radix
// selection (four 8-bit digits from the top), then in row order the dropped
// rows before the new length and the kept rows behind it, paired one to one.
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(const EvictParams p) {
  __shared__ int hist[256];
  __shared__ int red[kSelWaves];
  __shared__ int pick[2];
  const int tid = threadIdx.x;
  const int bh = blockIdx.x, b = bh / p.hkv;
  const int len = clamp_rows(p.lens[b], p.max_len);
  const int keep = min(max(p.keep ? p.keep[b] : p.keep_all, 0), len);
  if (tid == 0 && bh % p.hkv == 0) p.new_lens[b] = keep;
  if (tid == 0) p.move_counts[bh] = 0;
  if (keep == len) return;  // uniform: nothing to drop
  float *w = p.weights + int64_t(bh) * p.w_stride;
  int32_t *pos = p.positions ? p.positions + int64_t(bh) * p.w_stride : nullptr;
  const int from = p.protect_from ? p.protect_from[b] : 0x7FFFFFFF;
  auto rank_at = [&](int t) {
    const int at = pos ? pos[t] : t;
    return rank_of(w[t], at < p.sinks || (p.protect_from && at >= from));
  };
  uint32_t limit = 0;  // the rank of the keep-th row, digit by digit
  int need = keep;     // rows of the digits still open that are kept
  if (keep > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int t = tid; t < len; t += kSelThreads) {
        const uint32_t k = rank_at(t);
        if (shift == 24 || (k >> (shift + 8)) == (limit >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255u], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int left = need, d = 255;
        while (d > 0 && hist[d] < left) left -= hist[d--];
        pick[0] = d;
        pick[1] = left;
      }
      __syncthreads();
      limit |= uint32_t(pick[0]) << shift;
      need = pick[1];
      __syncthreads();
    }
  }
  int32_t *to = p.moves + int64_t(bh) * 2 * p.move_stride, *src = to + p.move_stride;
  int equal = 0, holes = 0, movers = 0;
  for (int t0 = 0; t0 < len; t0 += kSelThreads) {
    const int t = t0 + tid;
    const bool in = t < len;
    const uint32_t k = in ? rank_at(t) : 0u;
    int total;
    const int eq = equal + block_rank(in && k == limit, red, total);
    equal += total;
    const bool kept = in && keep > 0 && (k > limit || (k == limit && eq < need));
    const int hole = holes + block_rank(in && t < keep && !kept, red, total);
    if (in && t < keep && !kept) to[hole] = t;
    holes += total;
    const int mover = movers + block_rank(kept && t >= keep, red, total);
    if (kept && t >= keep) src[mover] = t;
    movers += total;
  }
  if (tid == 0) p.move_counts[bh] = holes;
  __threadfence_block();
  __syncthreads();
  for (int i = tid; i < holes; i += kSelThreads) {
    w[to[i]] = w[src[i]];
    if (pos) pos[to[i]] = pos[src[i]];
  }
  __syncthreads();
  for (int t = keep + tid; t < len; t += kSelThreads) w[t] = 0.f;
}

// Copies the paired rows, a wavefront per row (K, then V).
template <typename BtT>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(const EvictParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int bh = blockIdx.y, b = bh / p.hkv, h = bh % p.hkv;
  const int count = p.move_counts[bh];
  const int32_t *to = p.moves + int64_t(bh) * 2 * p.move_stride, *src = to + p.move_stride;
  const BtT *bt = static_cast<const BtT *>(p.block_table) + size_t(b) * p.bt_stride;
  for (int i = int(blockIdx.x) * (kThreads / kWave) + wave; i < count; i += int(gridDim.x) * (kThreads / kWave)) {
    const int64_t d = slot_of(bt, to[i], p.bt_stride, p.block_size, p.num_blocks);
    const int64_t s = slot_of(bt, src[i], p.bt_stride, p.block_size, p.num_blocks);
    if (d < 0 || s < 0) continue;
    const uint32_t *ks = p.key_cache + (s * p.hkv + h) * p.key_words, *vs = p.value_cache + (s * p.hkv + h) * p.value_words;
    uint32_t *kd = p.key_cache + (d * p.hkv + h) * p.key_words, *vd = p.value_cache + (d * p.hkv + h) * p.value_words;
    for (int j = lane; j < p.key_words; j += kWave) kd[j] = ks[j];
    for (int j = lane; j < p.value_words; j += kWave) vd[j] = vs[j];
  }
}

size_t evict_list_stride(int64_t max_len) { return size_t(std::max<int64_t>(max_len, 2) / 2 + 1); }

}  // namespace
}  // namespace hif8

using namespace hif8;

extern "C" int hif8_accept_drafts(void *const *caches, const int64_t *row_bytes, int64_t num_caches,
                                  int64_t num_blocks, int64_t block_size, const void *block_table,
                                  int block_table_dtype, int64_t max_blocks_per_seq, const int32_t *context_lens,
                                  const int32_t *accepted, int64_t accepted_width, const int32_t *accepted_counts,
                                  int64_t batch, int32_t *new_lens, hif8_stream_t stream) {
  static const char *kName = "hif8_accept_drafts";
  clear_error();
  if (num_caches < 0 || num_blocks <= 0 || block_size <= 0 || max_blocks_per_seq <= 0 || accepted_width < 0 || batch < 0)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions must be positive", kName);
  if (block_table_dtype != HIF8_INDEX_INT32 && block_table_dtype != HIF8_INDEX_INT64)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: block_table must be int32 or int64", kName);
  if (block_size > 0x7FFFFFFFll || accepted_width > 0x7FFFFFFFll || batch > 0xFFFFFFll)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", kName);
  if (batch == 0 || num_caches == 0) return HIF8_OK;
  if (!caches || !row_bytes || !block_table || !context_lens || !accepted_counts || (accepted_width && !accepted))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: null pointer argument", kName);
  int64_t widest = 0;
  for (int64_t i = 0; i < num_caches; ++i) {
    if (!caches[i]) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: null pointer argument", kName);
    if (!aligned(caches[i], 4)) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: caches must be 4-byte aligned", kName);
    if (row_bytes[i] <= 0 || row_bytes[i] % 4 || row_bytes[i] > (int64_t(kThreads) * 0xFFFF) * 4)
      return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: a token's rows must be a multiple of four bytes", kName);
    widest = std::max(widest, row_bytes[i] / 4);
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  for (int64_t c0 = 0; c0 < num_caches; c0 += kMaxCaches) {
    AcceptParams p{};
    p.caches = int(std::min<int64_t>(num_caches - c0, kMaxCaches));
    for (int i = 0; i < p.caches; ++i) {
      p.cache[i] = static_cast<uint32_t *>(caches[c0 + i]);
      p.words[i] = int(row_bytes[c0 + i] / 4);
    }
    p.block_table = block_table;
    p.lens = context_lens;
    p.path = accepted;
    p.counts = accepted_counts;
    p.new_lens = c0 == 0 ? new_lens : nullptr;
    p.bt_stride = max_blocks_per_seq;
    p.num_blocks = num_blocks;
    p.block_size = int(block_size);
    p.path_width = int(accepted_width);
    const dim3 grid(unsigned(batch), unsigned(p.caches), unsigned((widest + kThreads - 1) / kThreads));
    if (block_table_dtype == HIF8_INDEX_INT64) accept_kernel<int64_t><<<grid, kThreads, 0, s>>>(p);
    else accept_kernel<int32_t><<<grid, kThreads, 0, s>>>(p);
  }
  return check_launch(kName);
}

extern "C" size_t hif8_kv_evict_workspace_size(int64_t batch, int64_t num_kv_heads, int64_t max_seq_len) {
  if (batch <= 0 || num_kv_heads <= 0 || max_seq_len <= 0) return 0;
  return size_t(batch) * num_kv_heads * (2 * evict_list_stride(max_seq_len) + 1) * sizeof(int32_t);
}

extern "C" int hif8_kv_evict(uint8_t *key_cache, uint8_t *value_cache, int64_t num_blocks, int64_t block_size,
                             int64_t num_kv_heads, int64_t head_size, int64_t head_size_v, const void *block_table,
                             int block_table_dtype, int64_t max_blocks_per_seq, const int32_t *seq_lens,
                             int64_t batch, int64_t max_seq_len, float *key_weights, int32_t *positions,
                             int64_t weights_stride, const int32_t *keep, int64_t keep_all, int64_t sinks,
                             const int32_t *protect_from, int32_t *new_lens, void *workspace, size_t workspace_bytes,
                             hif8_stream_t stream) {
  static const char *kName = "hif8_kv_evict";
  clear_error();
  if (num_blocks <= 0 || block_size <= 0 || num_kv_heads <= 0 || head_size <= 0 || head_size_v <= 0 ||
      max_blocks_per_seq <= 0 || batch < 0 || max_seq_len < 0)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions must be positive", kName);
  if (head_size % 4 || head_size_v % 4)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: head sizes must be divisible by four", kName);
  if (block_table_dtype != HIF8_INDEX_INT32 && block_table_dtype != HIF8_INDEX_INT64)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: block_table must be int32 or int64", kName);
  if ((!keep && keep_all < 0) || sinks < 0)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: keep and sinks must not be negative", kName);
  if (block_size > 0x7FFFFFFFll || max_seq_len > 0x7FFFFFFFll - 4096 || head_size > 0x7FFFFFFll ||
      head_size_v > 0x7FFFFFFll || num_kv_heads > 0xFFFF || batch * num_kv_heads > 0xFFFF)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", kName);
  if (max_seq_len > max_blocks_per_seq * block_size)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: max_seq_len exceeds the block table capacity", kName);
  if (weights_stride < max_seq_len)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: key_weights rows are shorter than max_seq_len", kName);
  if (batch == 0) return HIF8_OK;
  if (!key_cache || !value_cache || !block_table || !seq_lens || !new_lens || (max_seq_len && !key_weights))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: null pointer argument", kName);
  if (!aligned(key_cache, 4) || !aligned(value_cache, 4))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: caches must be 4-byte aligned", kName);
  const size_t lists = evict_list_stride(std::max<int64_t>(max_seq_len, 1));
  const size_t need = hif8_kv_evict_workspace_size(batch, num_kv_heads, std::max<int64_t>(max_seq_len, 1));
  if (!workspace || workspace_bytes < need)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes required (got %zu)", kName, need,
                workspace_bytes);
  if (!aligned(workspace, 16))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned", kName);
  EvictParams p{};
  p.key_cache = reinterpret_cast<uint32_t *>(key_cache);
  p.value_cache = reinterpret_cast<uint32_t *>(value_cache);
  p.block_table = block_table;
  p.lens = seq_lens;
  p.keep = keep;
  p.protect_from = protect_from;
  p.weights = key_weights;
  p.positions = positions;
  p.new_lens = new_lens;
  p.move_counts = static_cast<int32_t *>(workspace);
  p.moves = p.move_counts + batch * num_kv_heads;
  p.bt_stride = max_blocks_per_seq;
  p.num_blocks = num_blocks;
  p.w_stride = weights_stride;
  p.move_stride = int64_t(lists);
  p.block_size = int(block_size);
  p.hkv = int(num_kv_heads);
  p.key_words = int((head_size + 4) / 4);
  p.value_words = int((head_size_v + 4) / 4);
  p.max_len = int(max_seq_len);
  p.keep_all = int(std::min<int64_t>(keep_all, 0x7FFFFFFF));
  p.sinks = int(std::min<int64_t>(sinks, 0x7FFFFFFF));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const unsigned bh = unsigned(batch * num_kv_heads);
  evict_select_kernel<<<bh, kSelThreads, 0, s>>>(p);
  const unsigned movers = unsigned(std::min<size_t>((lists + 3) / 4, std::max<size_t>(1, 2048 / bh)));
  if (block_table_dtype == HIF8_INDEX_INT64) evict_move_kernel<int64_t><<<dim3(movers, bh), kThreads, 0, s>>>(p);
  else evict_move_kernel<int32_t><<<dim3(movers, bh), kThreads, 0, s>>>(p);
  return check_launch(kName);
}
