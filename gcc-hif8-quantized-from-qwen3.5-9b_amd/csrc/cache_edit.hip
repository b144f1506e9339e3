// Edits of the HiF8 paged KV cache in place, for gfx950: the rows of an accepted
// draft path move to the end of the context, and the rows of least accumulated
// attention weight are dropped.  Both move whole rows (codes and scale), byte
// for byte, and are bound by the bytes of the rows that move.
#include <stddef.h>

#include <algorithm>
#include <memory>
#include <new>
#include <type_traits>

#include "hif8_common.h"

namespace hif8 {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int clamp_rows(int n, int most) { return n < 0 ? 0 : (n > most ? most : n); }

// Flat slot of a request's row, or -1 where the table or the cache ends before it.
// Rows are below 2^31, so the division is a 32-bit one (a shift for powers of two).
struct Pages {
  int64_t width, num_blocks;
  int block_size, log2_block;  // log2_block -1: no power of two
};

template <typename BtT>
__device__ __forceinline__ int64_t slot_of(const BtT *bt, int64_t row, const Pages &pg) {
  if (row < 0 || row > 0x7FFFFFFF) return -1;
  const uint32_t r = uint32_t(row);
  const uint32_t col = pg.log2_block >= 0 ? r >> pg.log2_block : r / uint32_t(pg.block_size);
  if (int64_t(col) >= pg.width) return -1;
  const int64_t blk = int64_t(bt[col]);
  return blk < 0 || blk >= pg.num_blocks ? int64_t(-1) : blk * pg.block_size + (r - col * uint32_t(pg.block_size));
}

int log2_or_none(int64_t v) {
  int l = 0;
  while ((int64_t(1) << l) < v) ++l;
  return (int64_t(1) << l) == v ? l : -1;
}

// --------------------------------------------------------------- acceptance

// Caches (K and V of every layer) of one launch; up to 16 go with 0.2 KB of
// arguments instead of 1.6, which the host copies (12.2 -> 11.0 us a call).
constexpr int kMaxCaches = 128, kFewCaches = 16;

template <int kCaches>
struct AcceptParams {
  uint32_t *cache[kCaches];     // [num_blocks, block_size, words]
  int words[kCaches];           // 4-byte words of one token's rows, all KV heads
  const void *block_table;
  const int32_t *lens;          // [batch] rows before the drafts
  const int32_t *path;          // [batch, path_width] draft indices, rising
  const int32_t *counts;        // [batch]
  int32_t *new_lens;            // [batch]
  Pages pages;
  int path_width, caches;
};

// Row lens[b] + path[b][i] -> row lens[b] + i for i < counts[b], in every cache.
// A thread owns one 4-byte column of the rows and moves them in order, eight
// loads ahead of eight stores.  path rises, so path[j] >= j and a row that is
// written is never read later: the move is in place and needs no barrier.  Bound
// by latency (table, path, row: three round trips): 32 requests' paths of up to
// eight drafts in eight layers' caches take 7.6 us in one launch.
template <typename BtT, int kCaches>
__global__ __launch_bounds__(kThreads) void accept_kernel(const AcceptParams<kCaches> p) {
  constexpr int kAhead = 8;
  const int b = blockIdx.x, c = blockIdx.y;
  const int col = int(blockIdx.z) * kThreads + threadIdx.x;
  const int ctx = max(p.lens[b], 0), count = clamp_rows(p.counts[b], p.path_width);
  if (c == 0 && blockIdx.z == 0 && threadIdx.x == 0 && p.new_lens) p.new_lens[b] = ctx + count;
  const int words = p.words[c];
  if (col >= words) return;
  const BtT *bt = static_cast<const BtT *>(p.block_table) + size_t(b) * p.pages.width;
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
            a < 0 || a == i ? int64_t(-1) : slot_of(bt, int64_t(ctx) + a, p.pages);
        if (from >= 0) {
          to[j] = slot_of(bt, int64_t(ctx) + i, p.pages);
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
  int2 *moves;                         // [batch * Hkv, move_stride]: (to, from)
  int32_t *move_counts;                // [batch * Hkv]
  int64_t w_stride, move_stride;
  Pages pages;
  int hkv, key_words, value_words, max_len, keep_all, sinks;
};

typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// Copies the paired rows, 16 bytes per thread: consecutive threads take the
// pieces of a row's K, then of its V; four pieces of other rows are loaded
// before the first is stored.  Bound by HBM: 102 MB (read and written) of 32
// pairs cut from 16384 to 4096 rows take 29 us, 3.5 TB/s in pieces of 260 bytes.
template <typename BtT>
__device__ __forceinline__ void move_rows(const EvictParams &p, int bh, int count, uint64_t thread, uint64_t stride) {
  constexpr int kAhead = 4;
  const int b = bh / p.hkv, h = bh % p.hkv;
  const int2 *moves = p.moves + int64_t(bh) * p.move_stride;
  const BtT *bt = static_cast<const BtT *>(p.block_table) + size_t(b) * p.pages.width;
  const uint32_t kc = uint32_t(p.key_words + 3) / 4, per_row = kc + uint32_t(p.value_words + 3) / 4;
  const uint64_t pieces = uint64_t(count) * per_row;
  const bool few = pieces >> 32 == 0;  // uniform: 32-bit divisions
  for (uint64_t i0 = thread; i0 < pieces; i0 += kAhead * stride) {
    u32x4_a4 v[kAhead];
    uint32_t *to[kAhead];
    int words[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const uint64_t i = i0 + j * stride;
      words[j] = 0;
      if (i >= pieces) continue;
      const uint32_t row = few ? uint32_t(i) / per_row : uint32_t(i / per_row);
      uint32_t c = uint32_t(i - uint64_t(row) * per_row);
      const int2 m = moves[row];
      const int64_t d = slot_of(bt, m.x, p.pages), s = slot_of(bt, m.y, p.pages);
      if (d < 0 || s < 0) continue;
      const bool is_v = c >= kc;
      if (is_v) c -= kc;
      const int width = is_v ? p.value_words : p.key_words;
      uint32_t *cache = is_v ? p.value_cache : p.key_cache;
      const uint32_t *src = cache + (s * p.hkv + h) * width + 4 * c;
      to[j] = cache + (d * p.hkv + h) * width + 4 * c;
      words[j] = min(4, width - int(4 * c));
      if (words[j] == 4) {
        v[j] = *reinterpret_cast<const u32x4_a4 *>(src);
      } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (e < words[j]) v[j][e] = src[e];
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (words[j] == 4) {
        *reinterpret_cast<u32x4_a4 *>(to[j]) = v[j];
      } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (e < words[j]) to[j][e] = v[j][e];
      }
    }
  }
}

// Larger is kept first: protected rows, then weights in falling order, NaN last.
__device__ __forceinline__ uint32_t rank_of(float w, bool safe) {
  if (safe) return 0xFFFFFFFFu;
  if (__builtin_isnan(w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 counts as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;
constexpr int kBins = 2048;

// One workgroup per (request, KV head): the rank of the last kept row by radix
// selection (digits of 11, 11 and 10 bits from the top), then the dropped rows
// before the new length and the kept rows behind it, each in row order and
// paired one to one.  Every wavefront owns a run of consecutive rows, so ranks
// within it are ballots and only its totals cross the workgroup.  The ranks of
// up to 64 kHeld rows per wavefront stay in registers (kHeld 0: they are read
// again in every pass).  Bound by the latency of one read and about fifteen
// barriers: 7 us for 600 rows (11 with the move of 88 of them), 19 us for 32 pairs
// of 16384 rows each (one workgroup per pair leaves most of the GPU idle), 29 more
// for the rows that move afterwards.  With ranks read again in every pass, digits of
// eight bits and 4-byte moves the whole calls took 41 and 117 us.
template <int kHeld, typename Mover>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(const EvictParams p) {
  __shared__ int hist[kBins];
  __shared__ int red[kSelWaves][2];
  __shared__ int pick[3];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bh = blockIdx.x, b = bh / p.hkv;
  const int len = clamp_rows(p.lens[b], p.max_len);
  const int keep = min(max(p.keep ? p.keep[b] : p.keep_all, 0), len);
  if (tid == 0 && bh % p.hkv == 0) p.new_lens[b] = keep;
  if (keep == len) {  // uniform: nothing to drop
    if (tid == 0) p.move_counts[bh] = 0;
    return;
  }
  float *w = p.weights + int64_t(bh) * p.w_stride;
  int32_t *pos = p.positions ? p.positions + int64_t(bh) * p.w_stride : nullptr;
  const int from = p.protect_from ? p.protect_from[b] : 0x7FFFFFFF;
  const int steps = (len + kSelThreads - 1) / kSelThreads;  // 64-row steps of a wavefront
  const int row0 = wave * steps * kWave + lane;
  auto load = [&](int t) {
    const int at = pos ? pos[t] : t;
    return rank_of(w[t], at < p.sinks || (p.protect_from && at >= from));
  };
  uint32_t held[kHeld ? kHeld : 1];
  if constexpr (kHeld > 0) {
    // Every load is issued before the first is used; rows past the end repeat the last.
    float wv[kHeld];
    int at[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) wv[i] = w[min(row0 + i * kWave, len - 1)];
    if (pos) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) at[i] = pos[min(row0 + i * kWave, len - 1)];
    } else {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) at[i] = row0 + i * kWave;
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      held[i] = rank_of(wv[i], (at[i] < p.sinks) | (p.protect_from && at[i] >= from));
  }
  // f(row, rank, is a row) for the wavefront's rows in order; every lane takes part.
  auto each = [&](auto f) {
    if constexpr (kHeld > 0) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        if (i >= steps) break;
        f(row0 + i * kWave, held[i], row0 + i * kWave < len);
      }
    } else {
      for (int i = 0; i < steps; ++i) {
        const int t = row0 + i * kWave;
        f(t, t < len ? load(t) : 0u, t < len);
      }
    }
  };

  // Rows with rank >> shift above `limit` are kept, and the first `need` of those equal to it.
  uint32_t limit = 0xFFFFFFFFu;
  int shift = 0, need = 0;
  if (keep > 0) {
    need = keep;
    limit = 0;
    int width = 11;
    for (shift = 21;; shift -= width) {
      for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      each([&](int, uint32_t k, bool in) {
        if (in && (shift == 21 || (k >> (shift + width)) == limit))
          atomicAdd(&hist[(k >> shift) & ((1u << width) - 1u)], 1);
      });
      __syncthreads();
      // From the top: thread i holds bins 2047 - 2 i and 2046 - 2 i.
      const int h0 = hist[kBins - 1 - 2 * tid], h1 = hist[kBins - 2 - 2 * tid];
      int sum = h0 + h1;
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) {
        const int up = __shfl_up(sum, o, kWave);
        if (lane >= o) sum += up;
      }
      if (lane == kWave - 1) red[wave][0] = sum;
      __syncthreads();
      int base = 0;
      for (int i = 0; i < wave; ++i) base += red[i][0];
      const int before = base + sum - h0 - h1;  // rows in higher bins
      if (before < need && need <= before + h0 + h1) {  // one thread
        const bool first = need <= before + h0;
        pick[0] = first ? kBins - 1 - 2 * tid : kBins - 2 - 2 * tid;
        pick[1] = need - before - (first ? 0 : h0);
        pick[2] = first ? h0 : h1;
      }
      __syncthreads();
      limit = (limit << width) | uint32_t(pick[0]);
      need = pick[1];
      if (shift == 0 || need == pick[2]) break;  // the whole bin is kept: no finer digit matters
      if (shift == 10) width = 10;
      __syncthreads();
    }
  }
  // Totals of the wavefront's rows equal to the limit where not all of those are
  // kept, then of its dropped and moving rows.
  const bool ties = keep == 0 || need < pick[2];  // uniform
  const uint32_t least = limit << shift;
  int equal = 0;
  if (ties) {
    each([&](int, uint32_t k, bool in) { equal += __popcll(__ballot(in && (k >> shift) == limit)); });
    if (lane == 0) red[wave][0] = equal;
    __syncthreads();
    equal = 0;
    for (int i = 0; i < wave; ++i) equal += red[i][0];
  }
  const uint64_t below = (uint64_t(1) << lane) - 1;
  auto kept = [&](uint32_t k, bool in, int &seen) {
    if (!ties) return in && k >= least;
    const bool same = in && (k >> shift) == limit;
    const uint64_t ball = __ballot(same);
    const bool yes = in && keep > 0 && ((k >> shift) > limit || (same && seen + __popcll(ball & below) < need));
    seen += __popcll(ball);
    return yes;
  };
  int seen = equal, holes = 0, movers = 0;
  each([&](int t, uint32_t k, bool in) {
    const bool yes = kept(k, in, seen);
    holes += __popcll(__ballot(in && t < keep && !yes));
    movers += __popcll(__ballot(yes && t >= keep));
  });
  __syncthreads();
  if (lane == 0) {
    red[wave][0] = holes;
    red[wave][1] = movers;
  }
  __syncthreads();
  holes = movers = 0;
  for (int i = 0; i < wave; ++i) {
    holes += red[i][0];
    movers += red[i][1];
  }
  int count = 0;
  for (int i = 0; i < kSelWaves; ++i) count += red[i][0];
  int2 *moves = p.moves + int64_t(bh) * p.move_stride;
  seen = equal;
  each([&](int t, uint32_t k, bool in) {
    const bool yes = kept(k, in, seen);
    const bool hole = in && t < keep && !yes, mover = yes && t >= keep;
    const uint64_t hb = __ballot(hole), mb = __ballot(mover);
    if (hole) moves[holes + __popcll(hb & below)].x = t;
    if (mover) moves[movers + __popcll(mb & below)].y = t;
    holes += __popcll(hb);
    movers += __popcll(mb);
  });
  if (tid == 0) p.move_counts[bh] = count;
  __threadfence_block();
  __syncthreads();
  for (int i = tid; i < count; i += kSelThreads) {
    const int2 m = moves[i];
    w[m.x] = w[m.y];
    if (pos) pos[m.x] = pos[m.y];
  }
  __syncthreads();
  for (int t = keep + tid; t < len; t += kSelThreads) w[t] = 0.f;
  if constexpr (!std::is_void_v<Mover>) move_rows<Mover>(p, bh, count, uint64_t(tid), kSelThreads);
}

template <typename BtT>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(const EvictParams p) {
  move_rows<BtT>(p, int(blockIdx.y), p.move_counts[blockIdx.y], uint64_t(blockIdx.x) * kThreads + threadIdx.x,
                 uint64_t(gridDim.x) * kThreads);
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
  // Two threads would move the same rows, one of them onto rows that the other has yet to read.
  struct Span {
    uintptr_t first;
    uint64_t bytes;
  };
  const std::unique_ptr<Span[]> spans(new (std::nothrow) Span[size_t(num_caches)]);
  if (!spans) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: too many caches", kName);
  for (int64_t i = 0; i < num_caches; ++i)
    spans[i] = {reinterpret_cast<uintptr_t>(caches[i]), uint64_t(num_blocks) * uint64_t(block_size) * uint64_t(row_bytes[i])};
  std::sort(spans.get(), spans.get() + num_caches, [](const Span &a, const Span &b) { return a.first < b.first; });
  for (int64_t i = 1; i < num_caches; ++i)
    if (spans[i].first - spans[i - 1].first < spans[i - 1].bytes)
      return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: caches must not overlap", kName);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const auto launch = [&](auto most) {
    constexpr int kCaches = decltype(most)::value;
    for (int64_t c0 = 0; c0 < num_caches; c0 += kCaches) {
      AcceptParams<kCaches> p{};
      p.caches = int(std::min<int64_t>(num_caches - c0, kCaches));
      for (int i = 0; i < p.caches; ++i) {
        p.cache[i] = static_cast<uint32_t *>(caches[c0 + i]);
        p.words[i] = int(row_bytes[c0 + i] / 4);
      }
      p.block_table = block_table;
      p.lens = context_lens;
      p.path = accepted;
      p.counts = accepted_counts;
      p.new_lens = c0 == 0 ? new_lens : nullptr;
      p.pages = Pages{max_blocks_per_seq, num_blocks, int(block_size), log2_or_none(block_size)};
      p.path_width = int(accepted_width);
      const dim3 grid(unsigned(batch), unsigned(p.caches), unsigned((widest + kThreads - 1) / kThreads));
      if (block_table_dtype == HIF8_INDEX_INT64) accept_kernel<int64_t><<<grid, kThreads, 0, s>>>(p);
      else accept_kernel<int32_t><<<grid, kThreads, 0, s>>>(p);
    }
  };
  if (num_caches <= kFewCaches) launch(std::integral_constant<int, kFewCaches>{});
  else launch(std::integral_constant<int, kMaxCaches>{});
  return check_launch(kName);
}

extern "C" size_t hif8_kv_evict_workspace_size(int64_t batch, int64_t num_kv_heads, int64_t max_seq_len) {
  if (batch <= 0 || num_kv_heads <= 0 || max_seq_len <= 0) return 0;
  // The lists of pairs, then a count per (request, KV head).
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
  p.moves = static_cast<int2 *>(workspace);
  p.move_counts = reinterpret_cast<int32_t *>(p.moves + size_t(batch) * num_kv_heads * lists);
  p.pages = Pages{max_blocks_per_seq, num_blocks, int(block_size), log2_or_none(block_size)};
  p.w_stride = weights_stride;
  p.move_stride = int64_t(lists);
  p.hkv = int(num_kv_heads);
  p.key_words = int((head_size + 4) / 4);
  p.value_words = int((head_size_v + 4) / 4);
  p.max_len = int(max_seq_len);
  p.keep_all = int(std::min<int64_t>(keep_all, 0x7FFFFFFF));
  p.sinks = int(std::min<int64_t>(sinks, 0x7FFFFFFF));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const unsigned bh = unsigned(batch * num_kv_heads);
  const bool i64 = block_table_dtype == HIF8_INDEX_INT64;
  const int64_t per_row = (p.key_words + 3) / 4 + (p.value_words + 3) / 4;
  const int64_t kept = std::min<int64_t>(p.keep_all, max_seq_len);
  const int64_t most_moves = keep ? max_seq_len / 2 : std::min(kept, max_seq_len - kept);
  if (max_seq_len <= kSelThreads && most_moves * per_row <= 5 * kSelThreads) {
    // The workgroup that selects rows moves them too where that is at most five
    // pieces per thread: 88 rows of 600 (D = 256) take 15.7 us against 18.2 with a
    // launch for the move, 256 of 1024 would take 21.8 against 18.7.
    if (i64) evict_select_kernel<1, int64_t><<<bh, kSelThreads, 0, s>>>(p);
    else evict_select_kernel<1, int32_t><<<bh, kSelThreads, 0, s>>>(p);
    return check_launch(kName);
  }
  if (max_seq_len <= 4 * kSelThreads) evict_select_kernel<4, void><<<bh, kSelThreads, 0, s>>>(p);
  else if (max_seq_len <= 16 * kSelThreads) evict_select_kernel<16, void><<<bh, kSelThreads, 0, s>>>(p);
  else if (max_seq_len <= 32 * kSelThreads) evict_select_kernel<32, void><<<bh, kSelThreads, 0, s>>>(p);
  else evict_select_kernel<0, void><<<bh, kSelThreads, 0, s>>>(p);
  // Four pieces per thread where there are rows for it, up to about eight workgroups per CU.
  const int64_t most = int64_t(lists) * per_row;
  const unsigned movers = unsigned(std::min<int64_t>((most + 4 * kThreads - 1) / (4 * kThreads), std::max<int64_t>(1, 2048 / bh)));
  if (i64) evict_move_kernel<int64_t><<<dim3(movers, bh), kThreads, 0, s>>>(p);
  else evict_move_kernel<int32_t><<<dim3(movers, bh), kThreads, 0, s>>>(p);
  return check_launch(kName);
}
