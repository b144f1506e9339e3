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
constexpr int kMaxNodes = 1024;  // rows of a request
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

// A request's rows, in LDS for as many as the call's longest one has.
struct Nodes {
  double *p;       // the target's probability of a row's token after its parent; 0: never taken
  double *q;       // u times what it was drawn with; u of a given token
  int64_t *token;
  int64_t *gone;   // tokens of the last row's children
  int *parent, *path;
  int *count;      // rows accepted, then the last of them, then the refused tokens
  static constexpr int kBytes = 4 * 8 + 2 * 4;  // per row
  __device__ Nodes(void *lds, int rows) {
    p = static_cast<double *>(lds);
    q = p + rows;
    token = reinterpret_cast<int64_t *>(q + rows);
    gone = token + rows;
    parent = reinterpret_cast<int *>(gone + rows);
    path = parent + rows;
    count = path + rows;
  }
};

// The request's rows, clipped to the call's and to its width.
__device__ __forceinline__ void rows_of(const VerifyParams &p, int b, int &begin, int &count) {
  clipped_rows(p.start_loc, b, p.total, begin, count);
  count = min(count, p.width);
}

__device__ __forceinline__ int parent_of(const VerifyParams &p, int begin, int i) {
  const int par = p.parents ? p.parents[begin + i] : i - 1;
  return par < 0 || par >= i ? -1 : par;  // follows nothing: never reached
}

template <typename TokT>
__device__ __forceinline__ void load_nodes(const VerifyParams &p, int begin, int n, const Nodes &nd) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int64_t x = int64_t(static_cast<const TokT *>(p.tokens)[begin + i]);
    const int par = parent_of(p, begin, i);
    float pv = 0.f, qv = 1.f;
    if (par >= 0 && x >= 0 && x < p.vocab) {
      pv = p.probs[int64_t(begin + par) * p.ld_probs + x];
      if (p.draft) qv = p.draft[int64_t(begin + i) * p.ld_draft + x];
    }
    nd.token[i] = x;
    nd.parent[i] = par;
    nd.q[i] = double(p.uniforms[begin + i]) * double(qv);  // exact
    nd.p[i] = pv > 0.f ? double(pv) : 0.;                  // NaN too is never taken
  }
}

// The accepted path of a chain, by the first wavefront: up to the first row that is refused.
__device__ __forceinline__ void follow(int n, const Nodes &nd) {
  const int lane = threadIdx.x & 63;
  int count = 1;
  for (int base = 1; base < n; base += kWave) {
    const int i = base + lane;
    const uint64_t refused = __ballot(i < n && !(nd.p[i] > 0. && nd.q[i] < nd.p[i]));
    if (refused) {
      count = base + __builtin_ctzll(refused);
      break;
    }
    count = min(base + kWave, n);
  }
  for (int i = lane; i < count; i += kWave) nd.path[i] = i;
  if (lane == 0) {
    nd.count[0] = count;
    nd.count[1] = count - 1;
    nd.count[2] = count < n ? 1 : 0;
    if (count < n) nd.gone[0] = nd.token[count];
  }
}

// The same of a tree.  Rows are gone through once: children come after their parent.
__device__ __forceinline__ void walk(int n, const Nodes &nd) {
  const int lane = threadIdx.x & 63;
  int now = 0, count = 1, gone = 0;  // gone: children of `now` refused so far
  double rest = 1.;
  if (lane == 0) nd.path[0] = 0;
  for (int base = 0; base < n; base += kWave) {
    const int i = base + lane;
    const int par = i < n ? nd.parent[i] : -1;
    const int64_t token = i < n ? nd.token[i] : 0;
    int from = 0;
    while (from < kWave) {
      const uint64_t mask = __ballot(par == now) & (~uint64_t(0) << from);
      if (!mask) break;
      const int at = __builtin_ctzll(mask), child = base + at;
      from = at + 1;
      // One that an earlier sibling had is refused with it.
      const int64_t x = nd.token[child];
      bool again = (__ballot(par == now && token == x) & ((uint64_t(1) << at) - 1)) != 0;
      for (int j0 = 0; j0 < gone && !again && base > 0; j0 += kWave)
        again = __any(j0 + lane < gone && nd.gone[j0 + lane] == x);
      bool takes = false;
      if (!again) {
        const double pv = nd.p[child];
        takes = pv > 0. && nd.q[child] * rest < pv;
        rest -= pv;
      }
      if (takes) {
        if (lane == 0) nd.path[count] = child;
        now = child;
        ++count;
        gone = 0;
        rest = 1.;
      } else {
        if (lane == 0) nd.gone[gone] = x;
        ++gone;
      }
    }
  }
  if (lane == 0) {
    nd.count[0] = count;
    nd.count[1] = now;
    nd.count[2] = gone;
  }
}

// What entry v of a chunk weighs: w above, or 0 where it is no positive number.
__device__ __forceinline__ double positive(double w) { return w > 0. && w < __builtin_inf() ? w : 0.; }

// A row of weights, four at a time.
struct Row {
  const float *probs, *draft;  // draft null: none
  int64_t vocab;
  __device__ __forceinline__ void weights(int64_t v, double *w) const {
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
// path for itself and sums its chunks of the weights; the first writes the path.  Bound by
// the probabilities' bytes: 64 chains of a 152k vocabulary, 78 MB, 16.1 us (4.8 TB/s); one
// chain of five 5.4 us, three round trips to HBM (tokens, their probabilities, the rows).
template <typename TokT>
__global__ __launch_bounds__(kThreads) void verify_sum_kernel(const VerifyParams p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const Nodes nd(smem, p.width);
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
  if (wave == 0) {
    if (p.parents) walk(n, nd);
    else follow(n, nd);
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = tid; i < p.width; i += kThreads) p.accepted[int64_t(b) * p.width + i] = i < nd.count[0] ? nd.path[i] : -1;
    if (tid == 0) {
      p.counts[b] = nd.count[0];
      p.last[b] = nd.count[1];
    }
  }
  const int chunk = int(blockIdx.x) * kWaves + wave;
  if (chunk >= p.chunks) return;
  const Row row = row_of(p, begin, n, nd.count[1]);
  double w[kChunk / kWave];
#pragma unroll
  for (int r = 0; r < kChunk / (4 * kWave); ++r)
    row.weights(int64_t(chunk) * kChunk + 4 * (lane + kWave * r), w + 4 * r);
  if (!p.draft) {
    // Given drafts: the tokens refused are struck out.
    for (int j = 0; j < nd.count[2]; ++j) {
      const int64_t d = nd.gone[j] - int64_t(chunk) * kChunk;
      if (d < 0 || d >= kChunk) continue;  // uniform
#pragma unroll
      for (int e = 0; e < kChunk / kWave; ++e)
        if (d == 4 * (lane + kWave * (e >> 2)) + (e & 3)) w[e] = 0.;
    }
  }
  double sum = 0.;
#pragma unroll
  for (int e = 0; e < kChunk / kWave; e += 4) sum += (w[e] + w[e + 1]) + (w[e + 2] + w[e + 3]);
  sum = wave_sum_double(sum);
  if (lane == 0) p.sums[int64_t(b) * p.chunks + chunk] = sum;
}

// Inclusive sum over a wavefront.
__device__ __forceinline__ double wave_upto(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const double left = __shfl_up(v, o, kWave);
    if (lane >= o) v += left;
  }
  return v;
}

// The next token of a request, a wavefront each: the chunk in which the running sum
// passes u_0 times the total, then the entry.  Sums of a chunk and of its entries may
// round apart: where no entry passes, it is the chunk's last with a weight.  Latency, 4.3 to
// 6.4 us: the sums, then a chunk.
template <typename TokT>
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(const VerifyParams p) {
  const int b = int(blockIdx.x) * kWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (b >= p.batch) return;
  const double *sums = p.sums + int64_t(b) * p.chunks;
  // Each lane's run of chunks.
  const int per = (p.chunks + kWave - 1) / kWave, c0 = min(lane * per, p.chunks), c1 = min(c0 + per, p.chunks);
  int begin, n;
  rows_of(p, b, begin, n);
  if (n == 0) {  // uniform
    if (lane == 0) p.next[b] = -1;
    return;
  }
  const double u = double(p.uniforms[begin]);
  const int last = p.last[b];
  const Row drawn = row_of(p, begin, n, last);
  const Row whole{drawn.probs, nullptr, p.vocab};
  double run = 0.;
  for (int c = c0; c < c1; ++c) run += sums[c];
  double upto = wave_upto(run);
  double total = __shfl(upto, kWave - 1, kWave);
  const bool residual = total > 0.;  // else it is 0: every weight is
  // Sixteen weights of a chunk, one after the other.
  auto weights = [&](int c, double (&w)[kChunk / kWave]) {
    const int64_t v0 = int64_t(c) * kChunk + kChunk / kWave * lane;
    const Row &row = residual ? drawn : whole;
#pragma unroll
    for (int e = 0; e < kChunk / kWave; e += 4) row.weights(v0 + e, w + e);
    if (!residual || p.draft) return;
    for (int base = last + 1; base < n; base += kWave) {
      const int i = base + lane;
      const bool child = i < n && parent_of(p, begin, i) == last;
      const int64_t token = child ? int64_t(static_cast<const TokT *>(p.tokens)[begin + i]) : 0;
      for (uint64_t left = __ballot(child); left; left &= left - 1) {
        const int64_t d = __shfl(token, __builtin_ctzll(left), kWave) - v0;
#pragma unroll
        for (int e = 0; e < kChunk / kWave; ++e)
          if (d == e) w[e] = 0.;
      }
    }
  };
  auto total_of = [](const double (&w)[kChunk / kWave]) {
    double s = 0.;
#pragma unroll
    for (int e = 0; e < kChunk / kWave; ++e) s += w[e];
    return s;
  };
  int chunk = -1;       // where the running sum passes
  int some = -1;        // the last chunk with a weight
  double before = 0., limit = 0.;
  if (residual) {
    limit = u * total;
    // The lane in whose run it passes, then the chunk of it.
    const uint64_t past = __ballot(run > 0. && upto > limit), any = __ballot(run > 0.);
    const int at = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(any);
    before = __shfl(upto - run, at, kWave);
    const int first = at * per, end = min(first + per, p.chunks);
    for (int c = first; c < end; c += kWave) {
      const double mine = c + lane < end ? sums[c + lane] : 0.;
      const double here = before + wave_upto(mine);
      const uint64_t over = __ballot(mine > 0. && here > limit), with = __ballot(mine > 0.);
      if (with) some = c + 63 - __builtin_clzll(with);
      if (over && past) {
        const int i = __builtin_ctzll(over);
        chunk = c + i;
        before = __shfl(here - mine, i, kWave);
        break;
      }
      before = __shfl(here, kWave - 1, kWave);
    }
  } else {
    // Rare: every weight of the residual is zero, and p itself is drawn from, chunk by chunk.
    double w[kChunk / kWave];
    total = 0.;
    for (int c = 0; c < p.chunks; ++c) {
      weights(c, w);
      total += wave_sum_double(total_of(w));
    }
    limit = u * total;
    for (int c = 0; c < p.chunks; ++c) {
      weights(c, w);
      const double all = wave_sum_double(total_of(w));
      if (!(all > 0.)) continue;
      some = c;
      if (before + all > limit) {
        chunk = c;
        break;
      }
      before += all;
    }
  }
  if (some < 0) {  // no entry weighs anything
    if (lane == 0) p.next[b] = -1;
    return;
  }
  const int c = chunk >= 0 ? chunk : some;
  double w[kChunk / kWave];
  weights(c, w);
  const double mine = total_of(w);
  double sum = before + (wave_upto(mine) - mine);
  int pick = -1, final = -1;
#pragma unroll
  for (int e = 0; e < kChunk / kWave; ++e) {
    sum += w[e];
    if (w[e] > 0.) final = e;
    if (w[e] > 0. && pick < 0 && chunk >= 0 && sum > limit) pick = e;
  }
  const uint64_t picks = __ballot(pick >= 0), finals = __ballot(final >= 0);
  if (picks ? lane == __builtin_ctzll(picks) : lane == 63 - __builtin_clzll(finals | 1))
    p.next[b] = int64_t(c) * kChunk + kChunk / kWave * lane + (picks ? pick : final);
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
  const size_t lds = size_t(max_query_len) * Nodes::kBytes + 16;
  const dim3 grid(unsigned((p.chunks + kWaves - 1) / kWaves), unsigned(batch));
  if (tokens_dtype == HIF8_INDEX_INT64) {
    verify_sum_kernel<int64_t><<<grid, kThreads, lds, s>>>(p);
    verify_pick_kernel<int64_t><<<unsigned((batch + kWaves - 1) / kWaves), kThreads, 0, s>>>(p);
  } else {
    verify_sum_kernel<int32_t><<<grid, kThreads, lds, s>>>(p);
    verify_pick_kernel<int32_t><<<unsigned((batch + kWaves - 1) / kWaves), kThreads, 0, s>>>(p);
  }
  return check_launch(kName);
}
