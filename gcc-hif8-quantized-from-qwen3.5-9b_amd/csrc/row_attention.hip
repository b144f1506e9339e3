// A few query rows per request over the whole HiF8 paged cache, for gfx950.
//
//   hif8_tree_attention                  drafted tokens under a tree mask
//   hif8_paged_decode_attention_weights  one token per request, and the sum of
//                                        its heads' softmax weights per cached row
//
// o_i = sum_t p_it V_t with p_i = softmax over the rows t that query row i sees
// of scale * q_i . K_t; a query row that sees nothing gets zeros.  K_t and V_t
// are dec(code) * row scale, in FP32 without a rounding in between.
#include <stddef.h>

#include <algorithm>

#include "row_attention.h"

namespace hif8 {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxSplits = 256;

// Any head size up to 512, group, block size and alignment: a workgroup per
// (query row, head, split), its wavefronts taking every fourth cache row with a
// running maximum and sum each, joined through LDS.
template <bool kBf16, typename BtT>
__global__ __launch_bounds__(kThreads) void row_attention_any(const RowAttnParams p) {
  constexpr int kPerLane = 8;  // head sizes up to 512
  __shared__ float red_ml[kWaves][2];
  __shared__ float red_o[kWaves][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = int(blockIdx.x) / p.hq, head = int(blockIdx.x) % p.hq, split = int(blockIdx.y);
  const int b = request_of_row(p, row);
  if (b < 0) return;  // a row behind the last request (uniform)
  int begin, count;
  request_rows(p, b, begin, count);
  const int ctx = clamp_rows(p.lens[b], p.max_len);
  const int len = rows_seen(p, ctx, count);
  const int t0 = split * p.split_tokens, t1 = min(t0 + p.split_tokens, len);
  const int h = head / p.group;
  const uint16_t *q = static_cast<const uint16_t *>(p.query) + (size_t(row) * p.hq + head) * p.d;
  const BtT *bt = static_cast<const BtT *>(p.block_table) + size_t(b) * p.bt_stride;
  const uint8_t *mask = p.mask ? p.mask + size_t(row) * p.mask_stride : nullptr;
  const size_t part = size_t(blockIdx.x) * p.num_splits + split;
  float qv[kPerLane], acc[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int dim = lane + kWave * i;
    qv[i] = dim < p.d ? half_bits_to_float<kBf16>(q[dim]) : 0.f;
    acc[i] = 0.f;
  }
  float m = -__builtin_inff(), l = 0.f;
  for (int t = t0 + wave; t < t1; t += kWaves) {
    const int64_t blk = int64_t(bt[t / p.block_size]);
    const bool seen = blk >= 0 && blk < p.num_blocks && (t < ctx || mask[t - ctx] != 0);
    float x = -__builtin_inff();
    if (seen) {
      const int64_t slot = blk * p.block_size + t % p.block_size;
      const uint8_t *kr = p.key_cache + (slot * p.hkv + h) * (p.d + 4);
      const uint8_t *vr = p.value_cache + (slot * p.hkv + h) * (p.dv + 4);
      const float ksc = *reinterpret_cast<const float *>(kr + p.d);
      const float vsc = *reinterpret_cast<const float *>(vr + p.dv);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int dim = lane + kWave * i;
        if (dim < p.d) dot = fmaf(qv[i], __uint_as_float(kDeviceTables.decode_f32[kr[dim]]), dot);
      }
      x = wave_sum(dot) * ksc * p.scale_log2;
      const float m_new = fmaxf(m, x);
      const float m_use = m_new == -__builtin_inff() ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m - m_use), w = __builtin_amdgcn_exp2f(x - m_use);
      l = l * alpha + w;
      m = m_new;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int dim = lane + kWave * i;
        if (dim < p.dv) acc[i] = fmaf(w * vsc, __uint_as_float(kDeviceTables.decode_f32[vr[dim]]), acc[i] * alpha);
      }
    }
    if (p.x && lane == 0) p.x[size_t(blockIdx.x) * p.x_stride + t] = x;
  }
  if (lane == 0) {
    red_ml[wave][0] = m;
    red_ml[wave][1] = l;
  }
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) red_o[wave][lane + kWave * i] = acc[i];
  __syncthreads();
  float mx = red_ml[0][0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, red_ml[w][0]);
  float f[kWaves], total = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    f[w] = red_ml[w][1] != 0.f ? __builtin_amdgcn_exp2f(red_ml[w][0] - mx) : 0.f;
    total += f[w] * red_ml[w][1];
  }
  if (threadIdx.x == 0) {
    p.part_ml[2 * part] = mx;
    p.part_ml[2 * part + 1] = total;
  }
  if (!(total != 0.f)) return;  // nothing seen: this split's outputs are not read
  for (int dim = threadIdx.x; dim < p.dv; dim += kThreads) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      if (f[w] != 0.f) y += f[w] * red_o[w][dim];
    p.part_o[part * p.dv + dim] = y;
  }
}

// Joins the splits of every query row and, where the call asks for them, adds
// the heads' weights onto the cached rows:
//   M = max_s m_s, L = sum_s 2^(m_s - M) l_s, out = sum_s 2^(m_s - M) O_s / L,
//   weights[b, h, t] (+)= sum over the heads of h of 2^(x_t - M) / L.
// Blocks below p.total_q * Hq * dim_slices take a (row, head, 64 dims) each:
// 16 threads of four dims by 16 groups of splits; the rest take 1024 cached
// rows of a (request, KV head) each.  Every sum has one order.
constexpr int kSliceDims = 64;
constexpr int kWeightKeys = 4 * kThreads;

// (M, 1 / L) of (row, head) `r` over the splits that hold keys; every lane of
// the calling wavefront gets them.
__device__ __forceinline__ void join_stats(const RowAttnParams &p, size_t r, int ns, float &m, float &inv) {
  const int lane = threadIdx.x & 63;
  const float *ml = p.part_ml + 2 * r * p.num_splits;
  float mx = -__builtin_inff();
  for (int s = lane; s < ns; s += kWave) mx = fmaxf(mx, ml[2 * s]);
  mx = wave_max(mx);
  float total = 0.f;
  for (int s = lane; s < ns; s += kWave) {
    // A split that saw nothing has l = 0; one with a NaN logit has l = NaN, whatever its maximum.
    const float ls = ml[2 * s + 1];
    if (ls != 0.f) total += __builtin_amdgcn_exp2f(ml[2 * s] - mx) * ls;
  }
  total = wave_sum(total);
  m = mx == -__builtin_inff() ? 0.f : mx;
  inv = total != 0.f ? 1.f / total : 0.f;
}

template <bool kBf16>
__global__ __launch_bounds__(kThreads) void row_attention_join(const RowAttnParams p, int dim_slices) {
  __shared__ float red[kThreads / 16][kSliceDims + 4];
  __shared__ float fac[kMaxSplits];
  __shared__ float stat[kWave][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t out_blocks = int64_t(p.total_q) * p.hq * dim_slices;
  if (int64_t(blockIdx.x) < out_blocks) {
    const int slice = int(blockIdx.x) % dim_slices;
    const int r = int(blockIdx.x) / dim_slices;
    const int b = request_of_row(p, r / p.hq);
    if (b < 0) return;
    int begin, count;
    request_rows(p, b, begin, count);
    const int ctx = clamp_rows(p.lens[b], p.max_len);
    const int len = rows_seen(p, ctx, count);
    const int ns = (len + p.split_tokens - 1) / p.split_tokens;
    float m, inv;
    join_stats(p, r, ns, m, inv);
    if (wave == 0)
      for (int s = lane; s < ns; s += kWave) {
        const float *ml = p.part_ml + 2 * (size_t(r) * p.num_splits + s);
        fac[s] = ml[1] != 0.f ? __builtin_amdgcn_exp2f(ml[0] - m) : 0.f;
      }
    __syncthreads();
    const int d4 = slice * kSliceDims + 4 * (tid & 15), g = tid >> 4;
    f32x4_t acc{0.f, 0.f, 0.f, 0.f};
    if (d4 < p.dv) {
      const float *po = p.part_o + size_t(r) * p.num_splits * p.dv + d4;
      for (int s = g; s < ns; s += kThreads / 16)
        if (fac[s] != 0.f) acc += fac[s] * *reinterpret_cast<const f32x4_t *>(po + size_t(s) * p.dv);
    }
    *reinterpret_cast<f32x4_t *>(&red[g][4 * (tid & 15)]) = acc;
    __syncthreads();
    const int dim = slice * kSliceDims + tid;
    if (tid >= kSliceDims || dim >= p.dv) return;
    float y = 0.f;
#pragma unroll
    for (int j = 0; j < kThreads / 16; ++j) y += red[j][tid];
    static_cast<uint16_t *>(p.out)[size_t(r) * p.dv + dim] = float_to_half_bits<kBf16>(y * inv);
    return;
  }
  // Weights: one query row per request (row b), so (row, head) index b * Hq + head.
  const int chunks = (p.max_len + kWeightKeys - 1) / kWeightKeys;
  const int64_t item = int64_t(blockIdx.x) - out_blocks;
  const int chunk = int(item % chunks);
  const int h = int(item / chunks) % p.hkv, b = int(item / chunks / p.hkv);
  const int len = clamp_rows(p.lens[b], p.max_len);
  const int t = chunk * kWeightKeys + 4 * tid;
  if (chunk * kWeightKeys >= len) return;  // uniform
  const int ns = (len + p.split_tokens - 1) / p.split_tokens;
  const size_t r0 = size_t(b) * p.hq + size_t(h) * p.group;
  f32x4_t acc{0.f, 0.f, 0.f, 0.f};
  for (int g0 = 0; g0 < p.group; g0 += kWave) {
    const int here = min(kWave, p.group - g0);
    __syncthreads();
    for (int j = wave; j < here; j += kWaves) {
      float m, inv;
      join_stats(p, r0 + g0 + j, ns, m, inv);
      if (lane == 0) {
        stat[j][0] = m;
        stat[j][1] = inv;
      }
    }
    __syncthreads();
    if (t >= len) continue;
    for (int j = 0; j < here; ++j) {
      // x_stride is a multiple of four and covers max_len: the vector stays inside its row.
      const f32x4_t x = *reinterpret_cast<const f32x4_t *>(p.x + (r0 + g0 + j) * p.x_stride + t);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += __builtin_amdgcn_exp2f(x[e] - stat[j][0]) * stat[j][1];
    }
  }
  float *w = p.weights + (int64_t(b) * p.hkv + h) * p.w_stride + t;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (t + e < len) w[e] = p.accumulate ? w[e] + acc[e] : acc[e];
}

// ------------------------------------------------------------- host side

struct RowPlan {
  int split_tokens, num_splits;
};

RowPlan plan_rows(int64_t total_q, int64_t heads, int64_t max_len) {
  RowPlan pl{};
  const int64_t len = std::max<int64_t>(max_len, 1);
  // About 2048 workgroups, at least 64 cache rows each.
  int64_t splits = std::max<int64_t>(1, 2048 / std::max<int64_t>(total_q * heads, 1));
  splits = std::min<int64_t>(splits, (len + 63) / 64);
  splits = std::min<int64_t>(splits, kMaxSplits);
  pl.split_tokens = int((len + splits - 1) / splits);
  pl.num_splits = int((len + pl.split_tokens - 1) / pl.split_tokens);
  return pl;
}

int64_t x_stride_of(int64_t max_len) { return (std::max<int64_t>(max_len, 1) + 63) / 64 * 64; }

size_t row_workspace(int64_t total_q, int64_t heads, int64_t dv, int64_t max_len, bool weights) {
  const RowPlan pl = plan_rows(total_q, heads, max_len);
  size_t floats = size_t(total_q) * heads * pl.num_splits * size_t(dv + 2);
  floats = (floats + 3) / 4 * 4;
  if (weights) floats += size_t(total_q) * heads * size_t(x_stride_of(max_len));
  return floats * sizeof(float);
}

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
  int64_t mask_stride, batch, heads, total_q, max_len;
  float scale;
  void *out;
  float *weights;
  int64_t w_stride;
  int accumulate;
  void *workspace;
  size_t workspace_bytes;
  hif8_stream_t stream;
};

int row_attention(const char *name, const RowArgs &a) {
  if (a.batch < 0 || a.heads <= 0 || a.hkv <= 0 || a.d <= 0 || a.dv <= 0 || a.num_blocks <= 0 || a.block_size <= 0 ||
      a.max_blocks <= 0 || a.max_len < 0 || a.total_q < 0)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions must be positive", name);
  if (a.heads % a.hkv) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: num_heads must be divisible by num_kv_heads", name);
  if (a.d % 4 || a.dv % 4) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: head sizes must be divisible by four", name);
  if (a.d > 512 || a.dv > 512)
    return fail(HIF8_ERR_UNSUPPORTED, "%s: head sizes above 512 are not supported", name);
  if (!is_io_dtype(a.q_dtype)) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: query must be float16 or bfloat16", name);
  if (a.bt_dtype != HIF8_INDEX_INT32 && a.bt_dtype != HIF8_INDEX_INT64)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: block_table must be int32 or int64", name);
  if (a.block_size > 0x7FFFFFFFll || a.max_len > 0x7FFFFFFFll - 4096 || a.batch > 0x7FFFFFFFll || a.heads > 0xFFFF ||
      a.total_q > 0x7FFFFFFFll)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", name);
  if (a.max_len > a.max_blocks * a.block_size)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: max_seq_len exceeds the block table capacity", name);
  if (a.weights && a.w_stride < a.max_len)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: key_weights rows are shorter than max_seq_len", name);
  if (a.batch == 0 || a.total_q == 0) return HIF8_OK;
  if (!a.query || !a.key_cache || !a.value_cache || !a.block_table || !a.lens || !a.out)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: null pointer argument", name);
  if (!aligned(a.key_cache, 4) || !aligned(a.value_cache, 4))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: caches must be 4-byte aligned", name);
  if (!aligned(a.query, 2) || !aligned(a.out, 2))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: query/out must be 2-byte aligned", name);
  const size_t need = row_workspace(a.total_q, a.heads, a.dv, a.max_len, a.weights != nullptr);
  if (!a.workspace || a.workspace_bytes < need)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes required (got %zu)", name, need,
                a.workspace_bytes);
  if (!aligned(a.workspace, 16))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned", name);

  const RowPlan pl = plan_rows(a.total_q, a.heads, a.max_len);
  RowAttnParams p{};
  p.query = a.query;
  p.key_cache = a.key_cache;
  p.value_cache = a.value_cache;
  p.block_table = a.block_table;
  p.start_loc = a.start_loc;
  p.lens = a.lens;
  p.mask = a.mask;
  p.out = a.out;
  p.bt_stride = a.max_blocks;
  p.num_blocks = a.num_blocks;
  p.mask_stride = a.mask_stride;
  p.block_size = int(a.block_size);
  p.hkv = int(a.hkv);
  p.hq = int(a.heads);
  p.group = int(a.heads / a.hkv);
  p.d = int(a.d);
  p.dv = int(a.dv);
  p.batch = int(a.batch);
  p.total_q = int(a.total_q);
  p.max_len = int(a.max_len);
  p.num_splits = pl.num_splits;
  p.split_tokens = pl.split_tokens;
  p.accumulate = a.accumulate ? 1 : 0;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  const size_t rows = size_t(a.total_q) * a.heads;
  p.part_o = static_cast<float *>(a.workspace);
  p.part_ml = p.part_o + rows * pl.num_splits * a.dv;
  if (a.weights) {
    p.x = p.part_o + (rows * pl.num_splits * size_t(a.dv + 2) + 3) / 4 * 4;
    p.x_stride = x_stride_of(a.max_len);
    p.weights = a.weights;
    p.w_stride = a.w_stride;
  }
  const int dim_slices = int((a.dv + kSliceDims - 1) / kSliceDims);
  const int64_t out_blocks = int64_t(rows) * dim_slices;
  const int64_t weight_blocks = a.weights ? a.batch * a.hkv * ((a.max_len + kWeightKeys - 1) / kWeightKeys) : 0;
  if (out_blocks + weight_blocks > 0xFFFFFFFFll / kThreads)  // threads of one launch
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", name);
  hipStream_t s = reinterpret_cast<hipStream_t>(a.stream);
  const bool bf16 = a.q_dtype == HIF8_DTYPE_BF16, i64 = a.bt_dtype == HIF8_INDEX_INT64;
  const dim3 grid(unsigned(rows), unsigned(pl.num_splits));
  if (bf16 && i64) row_attention_any<true, int64_t><<<grid, kThreads, 0, s>>>(p);
  else if (bf16) row_attention_any<true, int32_t><<<grid, kThreads, 0, s>>>(p);
  else if (i64) row_attention_any<false, int64_t><<<grid, kThreads, 0, s>>>(p);
  else row_attention_any<false, int32_t><<<grid, kThreads, 0, s>>>(p);
  const unsigned blocks = unsigned(out_blocks + weight_blocks);
  if (bf16) row_attention_join<true><<<blocks, kThreads, 0, s>>>(p, dim_slices);
  else row_attention_join<false><<<blocks, kThreads, 0, s>>>(p, dim_slices);
  return check_launch(name);
}

}  // namespace
}  // namespace hif8

using namespace hif8;

extern "C" size_t hif8_tree_attention_workspace_size(int64_t batch, int64_t num_heads, int64_t num_kv_heads,
                                                     int64_t head_size, int64_t head_size_v,
                                                     int64_t total_query_tokens, int64_t max_query_len,
                                                     int64_t max_seq_len) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_size <= 0 || head_size_v <= 0 ||
      total_query_tokens <= 0 || max_query_len <= 0 || max_seq_len < 0 || num_heads % num_kv_heads)
    return 0;
  return row_workspace(total_query_tokens, num_heads, head_size_v, max_seq_len, false);
}

extern "C" int hif8_tree_attention(const void *query, int q_dtype, const uint8_t *key_cache,
                                   const uint8_t *value_cache, int64_t num_blocks, int64_t block_size,
                                   int64_t num_kv_heads, int64_t head_size, int64_t head_size_v,
                                   const void *block_table, int block_table_dtype, int64_t max_blocks_per_seq,
                                   const int32_t *query_start_loc, const int32_t *context_lens,
                                   const uint8_t *tree_mask, int64_t mask_width, int64_t batch, int64_t num_heads,
                                   int64_t total_query_tokens, int64_t max_query_len, int64_t max_seq_len,
                                   float scale, void *out, void *workspace, size_t workspace_bytes,
                                   hif8_stream_t stream) {
  static const char *kName = "hif8_tree_attention";
  clear_error();
  if (max_query_len < 0 || mask_width < 0)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions must be positive", kName);
  if (batch > 0 && total_query_tokens > 0) {
    if (max_query_len == 0)
      return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: max_query_len must cover the query rows", kName);
    if (mask_width < max_query_len)
      return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: tree_mask rows are shorter than max_query_len", kName);
    if (!tree_mask || !query_start_loc)
      return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: null pointer argument", kName);
  }
  return row_attention(kName, RowArgs{query, q_dtype, key_cache, value_cache, num_blocks, block_size, num_kv_heads,
                                      head_size, head_size_v, block_table, block_table_dtype, max_blocks_per_seq,
                                      query_start_loc, context_lens, tree_mask, mask_width, batch, num_heads,
                                      total_query_tokens, max_seq_len, scale, out, nullptr, 0, 0, workspace,
                                      workspace_bytes, stream});
}

extern "C" size_t hif8_paged_decode_attention_weights_workspace_size(int64_t batch, int64_t num_heads,
                                                                     int64_t num_kv_heads, int64_t head_size,
                                                                     int64_t head_size_v, int64_t max_seq_len) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_size <= 0 || head_size_v <= 0 || max_seq_len < 0 ||
      num_heads % num_kv_heads)
    return 0;
  return row_workspace(batch, num_heads, head_size_v, max_seq_len, true);
}

extern "C" int hif8_paged_decode_attention_weights(const void *query, int q_dtype, const uint8_t *key_cache,
                                                   const uint8_t *value_cache, int64_t num_blocks,
                                                   int64_t block_size, int64_t num_kv_heads, int64_t head_size,
                                                   int64_t head_size_v, const void *block_table,
                                                   int block_table_dtype, int64_t max_blocks_per_seq,
                                                   const int32_t *seq_lens, int64_t batch, int64_t num_heads,
                                                   int64_t max_seq_len, float scale, void *out, float *key_weights,
                                                   int64_t weights_stride, int accumulate, void *workspace,
                                                   size_t workspace_bytes, hif8_stream_t stream) {
  static const char *kName = "hif8_paged_decode_attention_weights";
  clear_error();
  if (!key_weights && batch > 0) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: null pointer argument", kName);
  if (!aligned(key_weights, 4))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: key_weights must be 4-byte aligned", kName);
  return row_attention(kName, RowArgs{query, q_dtype, key_cache, value_cache, num_blocks, block_size, num_kv_heads,
                                      head_size, head_size_v, block_table, block_table_dtype, max_blocks_per_seq,
                                      nullptr, seq_lens, nullptr, 0, batch, num_heads, batch, max_seq_len, scale, out,
                                      key_weights, weights_stride, accumulate, workspace, workspace_bytes, stream});
}
