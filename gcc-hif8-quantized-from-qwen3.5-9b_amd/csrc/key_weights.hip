// Accumulated attention weight of every cached row under many query rows, from
// the HiF8 key cache alone, for gfx950.
//
//   weights[b, h, t] (+)= sum over request b's query rows i and the query heads
//                         of KV head h of softmax_t(scale * q_i . K_t)
//
// over the rows t that query row i sees: all of the request's, or with `causal`
// rows 0 .. seq_len - q_len + i.  K_t is dec(code) * row scale.
#include <stddef.h>

#include <algorithm>

#include "hif8_common.h"

namespace hif8 {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

struct WeightParams {
  const void *query;           // [total_q, Hq, D]
  const uint8_t *key_cache;    // [num_blocks, block_size, Hkv, D + 4]
  const void *block_table;     // [batch, bt_stride]
  const int32_t *start_loc;    // [batch + 1]
  const int32_t *lens;         // [batch]
  float *weights;              // [batch, Hkv, w_stride]
  float *stat;                 // [total_q * Hq, 2]: maximum, 1 / sum
  int64_t bt_stride, num_blocks, w_stride;
  int block_size, hkv, hq, group, d, batch, total_q, max_len, causal, accumulate;
  float scale_log2;
};

__device__ __forceinline__ int clamp_rows(int n, int most) { return n < 0 ? 0 : (n > most ? most : n); }

__device__ __forceinline__ void request_rows(const WeightParams &p, int b, int &begin, int &count) {
  begin = max(p.start_loc[b], 0);
  count = max(min(p.start_loc[b + 1], p.total_q) - begin, 0);
}

// Rows that query row i of a request with `len` cached rows sees.
__device__ __forceinline__ int rows_of(const WeightParams &p, int len, int count, int i) {
  return p.causal ? clamp_rows(len - count + i + 1, len) : len;
}

// Any head size up to 512: (maximum, 1 / sum) of a (query row, head) by a
// workgroup whose wavefronts take every fourth cache row.
template <bool kBf16, typename BtT>
__global__ __launch_bounds__(kThreads) void key_stats_any(const WeightParams p) {
  constexpr int kPerLane = 8;
  __shared__ float red[kWaves][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = int(blockIdx.x) / p.hq, head = int(blockIdx.x) % p.hq, h = head / p.group;
  int lo = 0, hi = p.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (p.start_loc[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  int begin, count;
  request_rows(p, lo, begin, count);
  if (row < begin || row - begin >= count) return;  // a row behind the last request
  const int end = rows_of(p, clamp_rows(p.lens[lo], p.max_len), count, row - begin);
  const uint16_t *q = static_cast<const uint16_t *>(p.query) + (size_t(row) * p.hq + head) * p.d;
  const BtT *bt = static_cast<const BtT *>(p.block_table) + size_t(lo) * p.bt_stride;
  float qv[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int dim = lane + kWave * i;
    qv[i] = dim < p.d ? half_bits_to_float<kBf16>(q[dim]) : 0.f;
  }
  float m = -__builtin_inff(), l = 0.f;
  for (int t = wave; t < end; t += kWaves) {
    const int64_t blk = int64_t(bt[t / p.block_size]);
    if (blk < 0 || blk >= p.num_blocks) continue;
    const uint8_t *kr = p.key_cache + ((blk * p.block_size + t % p.block_size) * p.hkv + h) * (p.d + 4);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int dim = lane + kWave * i;
      if (dim < p.d) dot = fmaf(qv[i], __uint_as_float(kDeviceTables.decode_f32[kr[dim]]), dot);
    }
    const float x = wave_sum(dot) * *reinterpret_cast<const float *>(kr + p.d) * p.scale_log2;
    const float m_new = fmaxf(m, x);
    const float m_use = m_new == -__builtin_inff() ? 0.f : m_new;
    l = l * __builtin_amdgcn_exp2f(m - m_use) + __builtin_amdgcn_exp2f(x - m_use);
    m = m_new;
  }
  if (lane == 0) {
    red[wave][0] = m;
    red[wave][1] = l;
  }
  __syncthreads();
  if (threadIdx.x) return;
  float mx = red[0][0];
  for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, red[w][0]);
  float total = 0.f;
  for (int w = 0; w < kWaves; ++w)
    if (red[w][1] != 0.f) total += __builtin_amdgcn_exp2f(red[w][0] - mx) * red[w][1];
  p.stat[2 * size_t(blockIdx.x)] = mx == -__builtin_inff() ? 0.f : mx;
  p.stat[2 * size_t(blockIdx.x) + 1] = total != 0.f ? 1.f / total : 0.f;
}

// The weights of 64 cached rows of a (request, KV head), 16 per wavefront: the
// row's values stay in the lanes while the query rows go by.
template <bool kBf16, typename BtT>
__global__ __launch_bounds__(kThreads) void key_sums_any(const WeightParams p, int tiles) {
  constexpr int kPerLane = 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tile = int(blockIdx.x) % tiles, bh = int(blockIdx.x) / tiles, h = bh % p.hkv, b = bh / p.hkv;
  const int len = clamp_rows(p.lens[b], p.max_len);
  int begin, count;
  request_rows(p, b, begin, count);
  const BtT *bt = static_cast<const BtT *>(p.block_table) + size_t(b) * p.bt_stride;
  float *w = p.weights + (int64_t(b) * p.hkv + h) * p.w_stride;
  for (int t = 64 * tile + 16 * wave; t < min(64 * tile + 16 * wave + 16, len); ++t) {
    const int64_t blk = int64_t(bt[t / p.block_size]);
    float sum = 0.f;
    if (blk >= 0 && blk < p.num_blocks) {
      const uint8_t *kr = p.key_cache + ((blk * p.block_size + t % p.block_size) * p.hkv + h) * (p.d + 4);
      const float ksc = *reinterpret_cast<const float *>(kr + p.d) * p.scale_log2;
      float kv[kPerLane];
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int dim = lane + kWave * i;
        kv[i] = dim < p.d ? __uint_as_float(kDeviceTables.decode_f32[kr[dim]]) : 0.f;
      }
      // The first query row that sees row t.
      const int first = p.causal ? max(0, t - (len - count)) : 0;
      for (int i = first; i < count; ++i)
        for (int g = 0; g < p.group; ++g) {
          const size_t r = size_t(begin + i) * p.hq + h * p.group + g;
          const uint16_t *q = static_cast<const uint16_t *>(p.query) + r * p.d;
          float dot = 0.f;
#pragma unroll
          for (int j = 0; j < kPerLane; ++j) {
            const int dim = lane + kWave * j;
            if (dim < p.d) dot = fmaf(half_bits_to_float<kBf16>(q[dim]), kv[j], dot);
          }
          sum += __builtin_amdgcn_exp2f(wave_sum(dot) * ksc - p.stat[2 * r]) * p.stat[2 * r + 1];
        }
    }
    if (lane == 0) w[t] = p.accumulate ? w[t] + sum : sum;
  }
}

}  // namespace
}  // namespace hif8

using namespace hif8;

extern "C" size_t hif8_key_weights_workspace_size(int64_t batch, int64_t num_heads, int64_t num_kv_heads,
                                                  int64_t head_size, int64_t total_query_tokens,
                                                  int64_t max_query_len, int64_t max_seq_len) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_size <= 0 || total_query_tokens <= 0 ||
      max_query_len <= 0 || max_seq_len <= 0 || num_heads % num_kv_heads)
    return 0;
  return size_t(total_query_tokens) * num_heads * 2 * sizeof(float);
}

extern "C" int hif8_key_weights(const void *query, int q_dtype, const uint8_t *key_cache, int64_t num_blocks,
                                int64_t block_size, int64_t num_kv_heads, int64_t head_size,
                                const void *block_table, int block_table_dtype, int64_t max_blocks_per_seq,
                                const int32_t *query_start_loc, const int32_t *seq_lens, int64_t batch,
                                int64_t num_heads, int64_t total_query_tokens, int64_t max_query_len,
                                int64_t max_seq_len, float scale, int causal, float *key_weights,
                                int64_t weights_stride, int accumulate, void *workspace, size_t workspace_bytes,
                                hif8_stream_t stream) {
  static const char *kName = "hif8_key_weights";
  clear_error();
  if (batch < 0 || num_heads <= 0 || num_kv_heads <= 0 || head_size <= 0 || num_blocks <= 0 || block_size <= 0 ||
      max_blocks_per_seq <= 0 || max_seq_len < 0 || total_query_tokens < 0 || max_query_len < 0)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions must be positive", kName);
  if (num_heads % num_kv_heads)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: num_heads must be divisible by num_kv_heads", kName);
  if (head_size % 4) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: head sizes must be divisible by four", kName);
  if (head_size > 512)
    return fail(HIF8_ERR_UNSUPPORTED, "%s: head sizes above 512 are not supported", kName);
  if (!is_io_dtype(q_dtype))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: query must be float16 or bfloat16", kName);
  if (block_table_dtype != HIF8_INDEX_INT32 && block_table_dtype != HIF8_INDEX_INT64)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: block_table must be int32 or int64", kName);
  if (block_size > 0x7FFFFFFFll || max_seq_len > 0x7FFFFFFFll - 4096 || batch > 0x7FFFFFFFll || num_heads > 0xFFFF ||
      total_query_tokens > 0x7FFFFFFFll)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", kName);
  if (max_seq_len > max_blocks_per_seq * block_size)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: max_seq_len exceeds the block table capacity", kName);
  if (weights_stride < max_seq_len)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: key_weights rows are shorter than max_seq_len", kName);
  if (batch == 0 || max_seq_len == 0) return HIF8_OK;
  if (!key_cache || !block_table || !query_start_loc || !seq_lens || !key_weights || (total_query_tokens && !query))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: null pointer argument", kName);
  if (total_query_tokens > 0 && max_query_len == 0)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: max_query_len must cover the query rows", kName);
  if (!aligned(key_cache, 4)) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: caches must be 4-byte aligned", kName);
  if (!aligned(query, 2)) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: query must be 2-byte aligned", kName);
  if (!aligned(key_weights, 4))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: key_weights must be 4-byte aligned", kName);
  const size_t need = hif8_key_weights_workspace_size(batch, num_heads, num_kv_heads, head_size, total_query_tokens,
                                                      max_query_len, max_seq_len);
  if (need && (!workspace || workspace_bytes < need))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes required (got %zu)", kName, need,
                workspace_bytes);
  if (!aligned(workspace, 16))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned", kName);
  const int64_t tiles = (max_seq_len + 63) / 64;
  const int64_t most = 0xFFFFFFFFll / kThreads;  // workgroups of one launch
  if (total_query_tokens * num_heads > most || batch * num_kv_heads * tiles > most)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", kName);

  WeightParams p{};
  p.query = query;
  p.key_cache = key_cache;
  p.block_table = block_table;
  p.start_loc = query_start_loc;
  p.lens = seq_lens;
  p.weights = key_weights;
  p.stat = static_cast<float *>(workspace);
  p.bt_stride = max_blocks_per_seq;
  p.num_blocks = num_blocks;
  p.w_stride = weights_stride;
  p.block_size = int(block_size);
  p.hkv = int(num_kv_heads);
  p.hq = int(num_heads);
  p.group = int(num_heads / num_kv_heads);
  p.d = int(head_size);
  p.batch = int(batch);
  p.total_q = int(total_query_tokens);
  p.max_len = int(max_seq_len);
  p.causal = causal ? 1 : 0;
  p.accumulate = accumulate ? 1 : 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool bf16 = q_dtype == HIF8_DTYPE_BF16, i64 = block_table_dtype == HIF8_INDEX_INT64;
  const unsigned rows = unsigned(total_query_tokens * num_heads), sums = unsigned(batch * num_kv_heads * tiles);
#define HIF8_KEY_WEIGHTS(BF16, BT)                                                         \
  do {                                                                                     \
    if (rows) key_stats_any<BF16, BT><<<rows, kThreads, 0, s>>>(p);                        \
    key_sums_any<BF16, BT><<<sums, kThreads, 0, s>>>(p, int(tiles));                       \
  } while (0)
  if (bf16 && i64) HIF8_KEY_WEIGHTS(true, int64_t);
  else if (bf16) HIF8_KEY_WEIGHTS(true, int32_t);
  else if (i64) HIF8_KEY_WEIGHTS(false, int64_t);
  else HIF8_KEY_WEIGHTS(false, int32_t);
#undef HIF8_KEY_WEIGHTS
  return check_launch(kName);
}
