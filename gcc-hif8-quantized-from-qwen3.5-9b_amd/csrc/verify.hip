// Verification of drafted tokens against the target model's probabilities, for
// gfx950 (hif8_verify_drafts).
//
// Row i of a request is a node of its drafts, p_i the target's probabilities of
// what follows it, x_i its token, u_i a number in [0, 1).  Row 0 holds a token
// that is known already.  From row 0 on:
//   drawn drafts (q_i: the probabilities that x_i was drawn from; a chain):
//     row i + 1 follows row i where u_{i+1} q_{i+1}(x_{i+1}) < p_i(x_{i+1}); at the
//     row that is not followed, w = max(p_i - q_{i+1}, 0), or p_i at the chain's end;
//   given drafts (no q; a chain or a tree): the children j of row i in rising order,
//     each with rest = 1 - the p_i of the tokens refused so far: j follows where
//     u_j rest < p_i(x_j); where none does, w is p_i without the children's tokens.
// The next token is the first v with w_0 + .. + w_v > u_0 sum(w).
//
// Every product, difference and sum is FP64: u q of two FP32 numbers is exact there,
// and a running sum of 152k FP32 probabilities in FP32 would be off by more than the
// smallest of them.
#include <stddef.h>

#include <algorithm>

#include "hif8_common.h"

namespace hif8 {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxNodes = 1024;  // rows of a request: their tokens, parents and numbers lie in LDS
constexpr int kChunk = 1024;     // entries whose sum is kept: sixteen per lane

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

struct VerifyParams {
  const float *probs;        // [total, ld_probs]
  const float *draft;        // [total, ld_draft] or null
  const void *tokens;        // [total] int32 or int64
  const int32_t *parents;    // [total] or null: a chain
  const float *uniforms;     // [total]
  const int32_t *start_loc;  // [batch + 1]
  int32_t *accepted;         // [batch, width]
  int32_t *counts;           // [batch]
  int64_t *next;             // [batch]
  double *sums;              // [batch, chunks]
  int32_t *last;             // [batch] row that is not followed, or -1: no rows
  int64_t ld_probs, ld_draft, vocab;
  int batch, total, width, chunks;
};

struct Nodes {
  double p[kMaxNodes];       // the target's probability of a row's token after its parent; 0: never taken
  int64_t token[kMaxNodes];
  float u[kMaxNodes];
  int parent[kMaxNodes];
  int path[kMaxNodes];
  int count;                 // rows accepted
  int last;
};

// The request's rows, clipped to the call's and to its width.
__device__ __forceinline__ void rows_of(const VerifyParams &p, int b, int &begin, int &count) {
  begin = max(p.start_loc[b], 0);
  count = max(min(min(p.start_loc[b + 1], p.total) - begin, p.width), 0);
}

template <typename TokT>
__device__ __forceinline__ void load_nodes(const VerifyParams &p, int begin, int n, Nodes &nd) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int64_t x = int64_t(static_cast<const TokT *>(p.tokens)[begin + i]);
    int par = p.parents ? p.parents[begin + i] : i - 1;
    if (i == 0 || par < 0 || par >= i) par = -1;  // follows nothing: never reached
    float pv = 0.f;
    if (par >= 0 && x >= 0 && x < p.vocab) pv = p.probs[int64_t(begin + par) * p.ld_probs + x];
    nd.token[i] = x;
    nd.parent[i] = par;
    nd.u[i] = p.uniforms[begin + i];
    nd.p[i] = pv > 0.f ? double(pv) : 0.;  // NaN too is never taken
  }
}

// Whether an earlier row than `child` with its parent has its token (a wavefront).
__device__ __forceinline__ bool seen_before(const Nodes &nd, int child) {
  const int lane = threadIdx.x & 63, par = nd.parent[child];
  const int64_t x = nd.token[child];
  for (int base = 0; base < child; base += kWave) {
    const int j = base + lane;
    if (__any(j < child && nd.parent[j] == par && nd.token[j] == x)) return true;
  }
  return false;
}

// The accepted path, by the first wavefront.  Rows are gone through once: children
// come after their parent.
__device__ __forceinline__ void walk(const VerifyParams &p, int begin, int n, Nodes &nd) {
  const int lane = threadIdx.x & 63;
  int now = 0, count = 1;
  double rest = 1.;
  if (lane == 0) nd.path[0] = 0;
  for (int base = 0; base < n; base += kWave) {
    const int i = base + lane;
    const int par = i < n ? nd.parent[i] : -1;
    int from = 0;
    while (from < kWave) {
      const uint64_t mask = __ballot(par == now) & (~uint64_t(0) << from);
      if (!mask) break;
      const int at = __builtin_ctzll(mask), child = base + at;
      from = at + 1;
      const double pv = nd.p[child], u = double(nd.u[child]);
      bool takes = false;
      if (p.draft) {
        const int64_t x = nd.token[child];
        if (pv > 0.) takes = u * double(p.draft[int64_t(begin + child) * p.ld_draft + x]) < pv;
      } else if (!seen_before(nd, child)) {
        takes = pv > 0. && u * rest < pv;
        rest = takes ? 1. : rest - pv;
      }
      if (takes) {
        if (lane == 0) nd.path[count] = child;
        now = child;
        ++count;
      }
    }
  }
  if (lane == 0) {
    nd.count = count;
    nd.last = now;
  }
}

// What entry v of a chunk weighs: w above, or 0 where it is no positive number.
__device__ __forceinline__ double positive(double w) { return w > 0. && w < __builtin_inf() ? w : 0.; }

// Sixteen entries from v on: four of each of four rounds of the wavefront.
struct Row {
  const float *probs, *draft;  // draft null: none
  int64_t vocab;
  __device__ __forceinline__ void weights(int64_t v, double (&w)[4]) const {
    if (v + 4 <= vocab) {
      const f32x4_a4 a = *reinterpret_cast<const f32x4_a4 *>(probs + v);
      if (draft) {
        const f32x4_a4 q = *reinterpret_cast<const f32x4_a4 *>(draft + v);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = positive(double(a[e]) - double(q[e]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = positive(double(a[e]));
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = v + e < vocab ? positive(draft ? double(probs[v + e]) - double(draft[v + e]) : double(probs[v + e])) : 0.;
  }
};

// Without drafts' probabilities the children of the last row strike their tokens out.
__device__ __forceinline__ void strike(const Nodes &nd, int n, int64_t v, double (&w)[4]) {
  for (int j = 1; j < n; ++j) {
    if (nd.parent[j] != nd.last) continue;
    const int64_t d = nd.token[j] - v;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d == e) w[e] = 0.;
  }
}

__device__ __forceinline__ double wave_sum_double(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

__device__ __forceinline__ Row row_of(const VerifyParams &p, int begin, int n, int last) {
  Row r{p.probs + int64_t(begin + last) * p.ld_probs, nullptr, p.vocab};
  if (p.draft && last + 1 < n) r.draft = p.draft + int64_t(begin + last + 1) * p.ld_draft;
  return r;
}

// A workgroup per (request, four chunks of the vocabulary).  Each finds the request's
// path for itself and sums its chunks of the weights; the first writes the path.
template <typename TokT>
__global__ __launch_bounds__(kThreads) void verify_sum_kernel(const VerifyParams p) {
  __shared__ Nodes nd;
  const int b = int(blockIdx.y), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int begin, n;
  rows_of(p, b, begin, n);
  if (n == 0) {  // uniform
    if (blockIdx.x == 0) {
      for (int i = tid; i < p.width; i += kThreads) p.accepted[int64_t(b) * p.width + i] = -1;
      if (tid == 0) {
        p.counts[b] = 0;
        p.last[b] = -1;
      }
    }
    return;
  }
  load_nodes<TokT>(p, begin, n, nd);
  __syncthreads();
  if (wave == 0) walk(p, begin, n, nd);
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = tid; i < p.width; i += kThreads) p.accepted[int64_t(b) * p.width + i] = i < nd.count ? nd.path[i] : -1;
    if (tid == 0) {
      p.counts[b] = nd.count;
      p.last[b] = nd.last;
    }
  }
  const int chunk = int(blockIdx.x) * kWaves + wave;
  if (chunk >= p.chunks) return;
  const Row row = row_of(p, begin, n, nd.last);
  double sum = 0.;
#pragma unroll
  for (int r = 0; r < kChunk / (4 * kWave); ++r) {
    const int64_t v = int64_t(chunk) * kChunk + 4 * (lane + kWave * r);
    double w[4];
    row.weights(v, w);
    if (!p.draft) strike(nd, n, v, w);
    sum += (w[0] + w[1]) + (w[2] + w[3]);
  }
  sum = wave_sum_double(sum);
  if (lane == 0) p.sums[int64_t(b) * p.chunks + chunk] = sum;
}

// Inclusive sum over the workgroup; `all` gets the total.  part: kWaves doubles of LDS.
__device__ __forceinline__ double block_upto(double mine, double *part, double &all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double upto = mine;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const double left = __shfl_up(upto, o, kWave);
    if (lane >= o) upto += left;
  }
  __syncthreads();
  if (lane == kWave - 1) part[wave] = upto;
  __syncthreads();
  double before = 0.;
  all = 0.;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += part[w];
    all += part[w];
  }
  return before + upto;
}

// The next token of a request: the chunk in which the running sum passes u_0 times
// the total, then the entry.  Sums of a chunk and of its entries may round apart:
// where no entry passes, it is the chunk's last with a weight.
template <typename TokT>
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(const VerifyParams p) {
  __shared__ Nodes nd;
  __shared__ double part[kWaves];
  __shared__ double before_s;
  __shared__ int chunk_s, any_s;
  __shared__ int64_t pick_s, some_s;
  const int b = int(blockIdx.x), tid = threadIdx.x;
  int begin, n;
  rows_of(p, b, begin, n);
  if (n == 0) {  // uniform
    if (tid == 0) p.next[b] = -1;
    return;
  }
  if (!p.draft) load_nodes<TokT>(p, begin, n, nd);
  if (tid == 0) {
    nd.last = p.last[b];
    chunk_s = 0x7FFFFFFF;
    any_s = -1;
    pick_s = INT64_MAX;
    some_s = -1;
    before_s = 0.;
  }
  __syncthreads();
  const Row drawn = row_of(p, begin, n, nd.last);
  const Row whole{drawn.probs, nullptr, p.vocab};
  const double *sums = p.sums + int64_t(b) * p.chunks;
  // Chunk sums, of p alone where no entry of the residual is left.
  double total = 0.;
  for (int c0 = 0; c0 < p.chunks; c0 += kThreads) {
    double all;
    block_upto(c0 + tid < p.chunks ? sums[c0 + tid] : 0., part, all);
    total += all;
  }
  const bool residual = total > 0.;  // else total is 0: every weight is
  auto chunk_weights = [&](int c, double (&w)[4]) {
    const int64_t v = int64_t(c) * kChunk + 4 * tid;
    if (residual) {
      drawn.weights(v, w);
      if (!p.draft) strike(nd, n, v, w);
    } else {
      whole.weights(v, w);
    }
  };
  auto chunk_sum = [&](int c) {  // every thread of the workgroup gets it
    double w[4], all;
    chunk_weights(c, w);
    block_upto((w[0] + w[1]) + (w[2] + w[3]), part, all);
    return all;
  };
  const double u = double(p.uniforms[begin]);
  double limit = u * total;
  if (residual) {
    double before = 0.;
    for (int c0 = 0; c0 < p.chunks; c0 += kThreads) {
      const int c = c0 + tid;
      const double mine = c < p.chunks ? sums[c] : 0.;
      double all;
      const double upto = before + block_upto(mine, part, all);
      if (mine > 0.) {
        atomicMax(&any_s, c);
        if (upto > limit) atomicMin(&chunk_s, c);
      }
      __syncthreads();
      if (chunk_s == c) before_s = upto - mine;
      if (chunk_s != 0x7FFFFFFF) break;  // uniform
      before += all;
    }
  } else {
    for (int c = 0; c < p.chunks; ++c) total += chunk_sum(c);
    limit = u * total;
    double before = 0.;
    for (int c = 0; c < p.chunks; ++c) {
      const double all = chunk_sum(c);
      if (tid == 0 && all > 0.) any_s = c;
      if (all > 0. && before + all > limit) {
        if (tid == 0) {
          chunk_s = c;
          before_s = before;
        }
        break;
      }
      before += all;
    }
  }
  __syncthreads();
  const bool found = chunk_s != 0x7FFFFFFF;
  const int c = found ? chunk_s : any_s;
  if (c < 0) {  // no entry weighs anything
    if (tid == 0) p.next[b] = -1;
    return;
  }
  double w[4], all;
  chunk_weights(c, w);
  const double mine = (w[0] + w[1]) + (w[2] + w[3]);
  double upto = before_s + (block_upto(mine, part, all) - mine);
  int64_t pick = -1, some = -1;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    upto += w[e];
    const int64_t v = int64_t(c) * kChunk + 4 * tid + e;
    if (w[e] > 0.) {
      some = v;
      if (pick < 0 && found && upto > limit) pick = v;
    }
  }
  if (pick >= 0) atomicMin(reinterpret_cast<unsigned long long *>(&pick_s), static_cast<unsigned long long>(pick));
  if (some >= 0) atomicMax(reinterpret_cast<long long *>(&some_s), static_cast<long long>(some));
  __syncthreads();
  if (tid == 0) p.next[b] = pick_s != INT64_MAX ? pick_s : some_s;
}

int64_t chunks_of(int64_t vocab) { return (vocab + kChunk - 1) / kChunk; }
size_t sums_bytes(int64_t batch, int64_t vocab) { return size_t(batch) * size_t(chunks_of(vocab)) * sizeof(double); }

}  // namespace
}  // namespace hif8

using namespace hif8;

extern "C" size_t hif8_verify_drafts_workspace_size(int64_t batch, int64_t vocab) {
  if (batch <= 0 || vocab <= 0) return 0;
  return sums_bytes(batch, vocab) + size_t(batch) * sizeof(int32_t);
}

extern "C" int hif8_verify_drafts(const float *target_probs, int64_t target_stride, const float *draft_probs,
                                  int64_t draft_stride, int64_t vocab, const void *draft_tokens, int tokens_dtype,
                                  const int32_t *parents, const float *uniforms, const int32_t *query_start_loc,
                                  int64_t batch, int64_t total_query_tokens, int64_t max_query_len, int32_t *accepted,
                                  int32_t *accepted_counts, int64_t *next_tokens, void *workspace,
                                  size_t workspace_bytes, hif8_stream_t stream) {
  static const char *kName = "hif8_verify_drafts";
  clear_error();
  if (vocab <= 0 || batch < 0 || total_query_tokens < 0 || max_query_len < 0 || target_stride < vocab ||
      (draft_probs && draft_stride < vocab))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions must be positive, rows at least vocab apart", kName);
  if (tokens_dtype != HIF8_INDEX_INT32 && tokens_dtype != HIF8_INDEX_INT64)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: draft_tokens must be int32 or int64", kName);
  if (draft_probs && parents)
    return fail(HIF8_ERR_UNSUPPORTED, "%s: draft_probs go with a chain of drafts, not with parents", kName);
  if (max_query_len > kMaxNodes)
    return fail(HIF8_ERR_UNSUPPORTED, "%s: at most %d rows per request", kName, kMaxNodes);
  if (batch > 0xFFFF || total_query_tokens > 0x7FFFFFFFll || vocab > (int64_t(1) << 40))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", kName);
  if (batch == 0) return HIF8_OK;
  if (!query_start_loc || !accepted_counts || !next_tokens || (max_query_len && !accepted) ||
      (total_query_tokens && (!target_probs || !draft_tokens || !uniforms)))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: null pointer argument", kName);
  const size_t need = hif8_verify_drafts_workspace_size(batch, vocab);
  if (!workspace || workspace_bytes < need)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes required (got %zu)", kName, need,
                workspace_bytes);
  if (!aligned(workspace, 8)) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace must be 8-byte aligned", kName);
  if (chunks_of(vocab) > 0x7FFFFFFll) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", kName);
  VerifyParams p{};
  p.probs = target_probs;
  p.draft = draft_probs;
  p.tokens = draft_tokens;
  p.parents = parents;
  p.uniforms = uniforms;
  p.start_loc = query_start_loc;
  p.accepted = accepted;
  p.counts = accepted_counts;
  p.next = next_tokens;
  p.sums = static_cast<double *>(workspace);
  p.last = reinterpret_cast<int32_t *>(static_cast<uint8_t *>(workspace) + sums_bytes(batch, vocab));
  p.ld_probs = target_stride;
  p.ld_draft = draft_stride;
  p.vocab = vocab;
  p.batch = int(batch);
  p.total = int(total_query_tokens);
  p.width = int(max_query_len);
  p.chunks = int(chunks_of(vocab));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid(unsigned((p.chunks + kWaves - 1) / kWaves), unsigned(batch));
  if (tokens_dtype == HIF8_INDEX_INT64) {
    verify_sum_kernel<int64_t><<<grid, kThreads, 0, s>>>(p);
    verify_pick_kernel<int64_t><<<unsigned(batch), kThreads, 0, s>>>(p);
  } else {
    verify_sum_kernel<int32_t><<<grid, kThreads, 0, s>>>(p);
    verify_pick_kernel<int32_t><<<unsigned(batch), kThreads, 0, s>>>(p);
  }
  return check_launch(kName);
}
