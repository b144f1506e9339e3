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
#include <type_traits>

#include "mfma_lookup.h"

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
  // Matrix-core kernels.
  float *part;                 // [key tiles, rows of this chunk * Hq, 2]: maximum, sum
  float *part_w;               // [row splits, batch, Hkv, w_pad] sums, or null: straight into weights
  int64_t magic, group_magic;  // ceil(2^36 / (block_size / 16)), ceil(2^32 / group)
  int64_t w_pad;
  int tok_lo, tok_hi;          // query tokens of this chunk
  int tiles, row_splits, split_rows;
  int max_query;               // query rows of a request that the launches are sized for
};

__device__ __forceinline__ int clamp_rows(int n, int most) { return n < 0 ? 0 : (n > most ? most : n); }

// Query rows of request b, clipped to the query tensor and to the longest request told (start_loc is caller data).
__device__ __forceinline__ void request_rows(const WeightParams &p, int b, int &begin, int &count) {
  clipped_rows(p.start_loc, b, p.total_q, begin, count);
  count = min(count, p.max_query);
}

// Rows that query row i of a request with `len` cached rows sees.
__device__ __forceinline__ int rows_of(const WeightParams &p, int len, int count, int i) {
  return p.causal ? clamp_rows(len - count + i + 1, len) : len;
}

// Any head size up to 512: (maximum, 1 / sum) of a (query row, head) by a
// workgroup whose wavefronts take every fourth cache row.  This kernel and the next
// are bound as the any-shape attention is, the next also by the query rows, which
// every cached row loads again: a prompt of 1024 with 16 heads of 96 takes 33 ms,
// with heads of 256 46 us on the matrix cores.
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
    float sum = 0.f, block = 0.f;
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
      for (int i = first; i < count; ++i) {
        float part = 0.f;  // a query token's heads, then the tokens: the sum of many small terms stays near
        for (int g = 0; g < p.group; ++g) {
          const size_t r = size_t(begin + i) * p.hq + h * p.group + g;
          const uint16_t *q = static_cast<const uint16_t *>(p.query) + r * p.d;
          float dot = 0.f;
#pragma unroll
          for (int j = 0; j < kPerLane; ++j) {
            const int dim = lane + kWave * j;
            if (dim < p.d) dot = fmaf(half_bits_to_float<kBf16>(q[dim]), kv[j], dot);
          }
          part += __builtin_amdgcn_exp2f(wave_sum(dot) * ksc - p.stat[2 * r]) * p.stat[2 * r + 1];
        }
        block += part;
        if ((i & 63) == 63) {
          sum += block;
          block = 0.f;
        }
      }
      sum += block;
    }
    if (lane == 0) w[t] = p.accumulate ? w[t] + sum : sum;
  }
}

// ---------------------------------------------------- on the matrix cores
//
// Head sizes 64, 128 and 256, pages of a multiple of 16 rows.  A workgroup of
// four wavefronts owns 256 cached rows of a (request, KV head), 64 per
// wavefront: their codes are decoded once into MFMA A operands (key =
// lane % 16) that stay in registers, and the (token, head) rows of the queries
// go by as B operands, 32 at a time through a ring in LDS filled by DMA in
// operand order.  The keys are stationary because every query row then costs
// one pass of 8 D / 256 LDS reads for 256 keys, and column sums need no
// exchange.  Two passes over S = K Q^T:
//   kSums false: per query row the maximum and the sum of 2^(x - maximum) over
//     the 256 keys, joined over the wavefronts in LDS, to `part`;
//   kSums true: with every row's maximum and sum known, each lane adds up
//     2^(x - M) / L of its keys over the rows, joined over the lanes at the end.
// A third small kernel joins `part` over the key tiles, a fourth the sums over
// the row splits; all orders of summation are fixed.
//
// What bounds it: a causal prompt of 4096 tokens (16 query, 4 KV heads of 256:
// 2 x 68.7 GFLOP at the visible half) takes 103 to 115 us a pass, 0.6 PFLOP/s.  A
// stage costs a wavefront 1024 cycles of matrix instructions and about as many
// of vector ones (an exponential per logit among them, at a quarter of the rate),
// and the two wavefronts of a SIMD overlap these in part.  Decoding the keys (256
// lookups per lane, 6000 cycles) and what comes before is a sixth of it, and most
// of a call with few query rows: 32 tokens over 4 x 8192 rows take 18 to 20 us a
// pass, of 35 MB.  Storing the logits for the second pass would write and read 67
// MB there; raising the wavefronts' priority around the products changed nothing.
constexpr int kKeys = 256;    // cached rows of a workgroup
constexpr int kStage = 32;    // query rows of a ring stage
constexpr int kRing = 3;

__device__ __forceinline__ void row_place(const WeightParams &p, int h, int r, int &tok, int &head) {
  tok = int((uint64_t(uint32_t(r)) * uint64_t(p.group_magic)) >> 32);
  head = h * p.group + (r - tok * p.group);
}

// The (token, head) rows, counted within the request and KV head, of the chunk's
// query tokens that see cached row t0 or a later one.
__device__ __forceinline__ void rows_that_see(const WeightParams &p, int t0, int len, int begin, int count, int &first,
                                              int &end) {
  const int lo = max(p.causal ? max(t0 - (len - count), 0) : 0, p.tok_lo - begin);
  const int hi = max(min(count, p.tok_hi - begin), 0);
  first = min(max(lo, 0), hi) * p.group;
  end = hi * p.group;
}

template <int kD, bool kBf16, bool kSums, typename BtT>
__global__ __launch_bounds__(kThreads, 2) void key_pass_mfma(const WeightParams p) {
  constexpr int kRow = kD + 4;
  constexpr int kQS = kD / 32;
  constexpr int kSlices = kD / 64;
  constexpr int kStageBytes = kStage * kD * 2;
  constexpr int kDma = kQS / 2;  // DMA instructions of a wavefront per stage
  static_assert(kRing * kStageBytes <= kLookupBytes, "the ring reuses the table's LDS");
  struct Smem {
    uint32_t table[kLookupBytes / 4];  // then the ring
    float2 ml[2][4][kStage];           // a stage's (maximum, sum) per wavefront
  };
  __shared__ __attribute__((aligned(16))) Smem sm;
  const uint32_t table = lds_address(sm.table);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;

  // The key tiles of one (request, KV head, row split) read the same queries:
  // their blocks are equal modulo 8 (the grid's x), on one XCD.
  const int outer = int(blockIdx.z) * 8 + int(blockIdx.x), tile = int(blockIdx.y);
  const int bs = outer / p.hkv, h = outer - bs * p.hkv;
  const int b = p.row_splits == 1 ? bs : bs / p.row_splits, split = bs - b * p.row_splits;
  if (b >= p.batch) return;  // padding block (uniform)
  const int len = clamp_rows(p.lens[b], p.max_len);
  const int t0 = tile * kKeys;
  if (t0 >= len) return;  // uniform
  int begin, count;
  request_rows(p, b, begin, count);
  // Query rows of this chunk that see row t0 or later, and this split of them.
  const int shift = p.causal ? len - count : len;     // row i sees rows up to shift + i (causal)
  int row_first, row_end;
  rows_that_see(p, t0, len, begin, count, row_first, row_end);
  const int r_lo = int(min(int64_t(row_first) + int64_t(split) * p.split_rows, int64_t(row_end)));
  const int r_hi = int(min(int64_t(r_lo) + p.split_rows, int64_t(row_end)));
  if (split > 0 && r_lo >= r_hi) return;  // uniform: nothing is read of this split
  const int stages = r_hi > r_lo ? (r_hi - r_lo + kStage - 1) / kStage : 0;
  const int key0 = t0 + 64 * wave;  // first key of this wavefront

  float acc[4][4];  // column sums of keys key0 + 16 kb + 4 g + e over rows n mod 16
#pragma unroll
  for (int kb = 0; kb < 4; ++kb)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[kb][e] = 0.f;

  if (stages > 0) {
    // Decode the wavefront's keys.
    const BtT *bt = static_cast<const BtT *>(p.block_table) + size_t(b) * p.bt_stride;
    const uint32_t rec = uint32_t(p.hkv) * kRow;
    const int gr = min(key0 + 16 * (lane & 3), len - 1) >> 4;  // lane i % 4 looks up 16-row group i
    const int col = int((uint64_t(gr) * uint64_t(p.magic)) >> 36);
    const int64_t blk = int64_t(bt[col]);
    const bool there = blk >= 0 && blk < p.num_blocks && key0 + 16 * (lane & 3) < len;
    const int64_t off_lane =
        there ? (blk * p.block_size + 16 * (gr - col * (p.block_size >> 4))) * int64_t(rec) + int64_t(h) * kRow : int64_t(-1);
    const uint32_t ok_groups = uint32_t(__ballot(off_lane >= 0)) & 15u;
    typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
    lk_u32x4 raw[4][kSlices];
    const uint8_t *base[4];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      const int lo = __builtin_amdgcn_readlane(int(uint64_t(off_lane)), kb);
      const int hi = __builtin_amdgcn_readlane(int(uint64_t(off_lane) >> 32), kb);
      const int64_t off = int64_t((uint64_t(uint32_t(hi)) << 32) | uint32_t(lo));
      base[kb] = p.key_cache + (off < 0 ? 0 : off);
#pragma unroll
      for (int i = 0; i < kSlices; ++i)
        raw[kb][i] = *reinterpret_cast<const u32x4_a4 *>(base[kb] + uint32_t(n) * rec + 16u * g + 64 * i);
    }
    fill_lookup<kBf16, kThreads>(sm.table, reinterpret_cast<uint32_t *>(sm.ml), tid);
    lds_barrier();
    const uint32_t lane4 = uint32_t(4 * lane);
    lk_u32x4 kf[4][kQS];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
      for (int i = 0; i < kQS; i += 2) {
        // Sixteen lookups at a time, packed here: left alone, the compiler holds
        // the halves apart until the loop and spills them.
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = i; j < i + 2; ++j) {
          kf[kb][j] = look8<false>(raw[kb][i >> 1][2 * (j & 1)], raw[kb][i >> 1][2 * (j & 1) + 1], lane4, table);
#pragma unroll
          for (int w = 0; w < 4; ++w) asm volatile("" : "+v"(kf[kb][j][w]));
        }
      }
    }
    lds_barrier();  // the ring takes the table's place
    // The row scales, only now: held over the lookups they were spilled one by one.
    float ksc[4][4];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        ksc[kb][e] = *reinterpret_cast<const float *>(base[kb] + uint32_t(4 * g + e) * rec + kD) * p.scale_log2;

    // Stage s: rows r_lo + 32 s .. + 31; rows past the last repeat it.  Wavefront
    // w brings half of the operands of row block w / 2.
    const uint16_t *query = static_cast<const uint16_t *>(p.query);
    auto fetch = [&](int s) {
      const int r = min(r_lo + kStage * s + 16 * (wave >> 1) + n, r_hi - 1);
      int tok, head;
      row_place(p, h, r, tok, head);
      const uint16_t *q = query + (size_t(begin + tok) * p.hq + head) * kD + 16 * g;
      const uint32_t to = table + uint32_t((s % kRing) * kStageBytes) + uint32_t((wave >> 1) * kQS * 1024);
#pragma unroll
      for (int j = 0; j < kDma; ++j) {
        const int i = (wave & 1) * kDma + j;
        dma16(q + 64 * (i >> 1) + 8 * (i & 1), to + 1024u * uint32_t(i));
      }
    };
    float2 st[2] = {};  // (M, 1 / L) of this lane's rows in the stage
    auto load_stats = [&](int s) {
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        const int r = r_lo + kStage * s + 16 * rb + n;
        int tok, head;
        row_place(p, h, min(r, r_hi - 1), tok, head);
        st[rb] = reinterpret_cast<const float2 *>(p.stat)[size_t(begin + tok) * p.hq + head];
      }
    };
    fetch(0);
    if (stages > 1) fetch(1);
    if constexpr (kSums) load_stats(0);
    for (int s = 0; s < stages; ++s) {
      if (s + 1 < stages) wait_vmcnt<kDma>();  // this stage's copies; the next one's may be in flight
      else wait_vmcnt<0>();
      lds_barrier();  // every wavefront's copies have landed, and it is done with the stage before
      if constexpr (!kSums) {
        // Join the previous stage's rows over the wavefronts.
        if (s > 0 && tid < kStage) {
          const int r = r_lo + kStage * (s - 1) + tid;
          int tok, head;
          row_place(p, h, r, tok, head);
          float2 v = sm.ml[(s - 1) & 1][0][tid];
#pragma unroll
          for (int w = 1; w < 4; ++w) {
            const float2 o = sm.ml[(s - 1) & 1][w][tid];
            const float mx = fmaxf(v.x, o.x);
            const float a = v.y != 0.f ? __builtin_amdgcn_exp2f(v.x - mx) * v.y : 0.f;
            const float c = o.y != 0.f ? __builtin_amdgcn_exp2f(o.x - mx) * o.y : 0.f;
            v = float2{mx, a + c};
          }
          const size_t chunk_rows = size_t(p.tok_hi - p.tok_lo) * p.hq;
          reinterpret_cast<float2 *>(p.part)[size_t(tile) * chunk_rows + size_t(begin + tok - p.tok_lo) * p.hq + head] = v;
        }
      }
      // The statistics arrive here, before newer copies are in flight: a wait for
      // them further down would wait for those too.
      float2 cur[2] = {st[0], st[1]};
      if constexpr (kSums) {
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
          asm volatile("" : "+v"(cur[rb].x), "+v"(cur[rb].y));
          if (r_lo + kStage * s + 16 * rb + n >= r_hi) cur[rb].y = 0.f;
        }
      }
      if (s + 2 < stages) fetch(s + 2);
      if constexpr (kSums) {
        if (s + 1 < stages) load_stats(s + 1);
      }
      const lk_u32x4 *q = reinterpret_cast<const lk_u32x4 *>(reinterpret_cast<const uint8_t *>(sm.table) +
                                                            (s % kRing) * kStageBytes);
      const int r0 = r_lo + kStage * s;
      lk_f32x4 d[2][4];
      auto product = [&](int rb) __attribute__((always_inline)) {
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) d[rb][kb] = lk_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kQS; ++i) {
          const lk_u32x4 qf = q[(rb * kQS + i) * kWave + lane];
#pragma unroll
          for (int kb = 0; kb < 4; ++kb) d[rb][kb] = mfma_16x16x32<kBf16>(kf[kb][i], qf, d[rb][kb]);
        }
      };
      // The rows of block rb: whether they see key kb, e, unless all of them see all.
      auto finish = [&](auto all, int rb, int lim) __attribute__((always_inline)) {
        constexpr bool kAll = decltype(all)::value;
        auto visible = [&](int kb, int e) {
          return bool(((ok_groups >> kb) & 1u) & uint32_t(key0 + 16 * kb + 4 * g + e < lim));
        };
        if constexpr (kSums) {
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w = __builtin_amdgcn_exp2f(fmaf(d[rb][kb][e], ksc[kb][e], -cur[rb].x));
              const float sum = fmaf(w, cur[rb].y, acc[kb][e]);
              acc[kb][e] = kAll || visible(kb, e) ? sum : acc[kb][e];
            }
        } else {
          float mx = -__builtin_inff();
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = d[rb][kb][e] * ksc[kb][e];
              d[rb][kb][e] = kAll || visible(kb, e) ? x : -__builtin_inff();
              mx = fmaxf(mx, d[rb][kb][e]);
            }
          mx = max_over_groups(mx);
          const float use = mx == -__builtin_inff() ? 0.f : mx;
          float l = 0.f;
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) l += __builtin_amdgcn_exp2f(d[rb][kb][e] - use);
          l = sum_over_groups(l);
          if (g == 0) sm.ml[s & 1][wave][16 * rb + n] = float2{mx, l};
        }
      };
      // Every row of the stage sees every key of the wavefront (uniform).
      int tok0, head0;
      row_place(p, h, r0, tok0, head0);
      const bool full = key0 + 64 <= len && ok_groups == 15u && (!p.causal || key0 + 63 <= shift + tok0) &&
                        (!kSums || r0 + kStage <= r_hi);
      product(0);
      __builtin_amdgcn_sched_barrier(0);
      if (full) {
        // The second block's products and the first one's exponentials in turn: the
        // wavefronts of a SIMD take their stages in step, so that neither unit was
        // busy half of the time when each wavefront did one thing after the other.
        product(1);
        finish(std::true_type{}, 0, 0);
#pragma unroll
        for (int i = 0; i < 4 * kQS; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction
          __builtin_amdgcn_sched_group_barrier(0x002, 128 / (4 * kQS) > 4 ? 8 : 4, 0);  // vector instructions
        }
        __builtin_amdgcn_sched_barrier(0);
        finish(std::true_type{}, 1, 0);
      } else {
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
          int tok, head;
          row_place(p, h, min(r0 + 16 * rb + n, r_hi - 1), tok, head);
          int lim = p.causal ? min(len, shift + tok + 1) : len;
          if (kSums && r0 + 16 * rb + n >= r_hi) lim = 0;  // its statistics need not be a number
          finish(std::false_type{}, rb, lim);
          if (rb == 0) product(1);
        }
      }
    }
    if constexpr (!kSums) {
      lds_barrier();
      const int s = stages - 1;
      const int r = r_lo + kStage * s + tid;
      if (tid < kStage && r < r_hi) {
        int tok, head;
        row_place(p, h, r, tok, head);
        float2 v = sm.ml[s & 1][0][tid];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          const float2 o = sm.ml[s & 1][w][tid];
          const float mx = fmaxf(v.x, o.x);
          const float a = v.y != 0.f ? __builtin_amdgcn_exp2f(v.x - mx) * v.y : 0.f;
          const float c = o.y != 0.f ? __builtin_amdgcn_exp2f(o.x - mx) * o.y : 0.f;
          v = float2{mx, a + c};
        }
        const size_t chunk_rows = size_t(p.tok_hi - p.tok_lo) * p.hq;
        reinterpret_cast<float2 *>(p.part)[size_t(tile) * chunk_rows + size_t(begin + tok - p.tok_lo) * p.hq + head] = v;
      }
    }
  }
  if constexpr (kSums) {
    // Every lane of a group has the group's 16 sums; lane n keeps that of its own
    // key, for one load and one store (key by key they took 5900 cycles, now 900).
    float v = 0.f;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float sum = sum_over_columns(acc[kb][e]);
        v = n == 4 * kb + e ? sum : v;
      }
    const int t = key0 + 16 * (n >> 2) + 4 * g + (n & 3);
    if (t < len) {
      if (p.part_w) {
        p.part_w[((int64_t(split) * p.batch + b) * p.hkv + h) * p.w_pad + t] = v;
      } else {
        float *w = p.weights + (int64_t(b) * p.hkv + h) * p.w_stride + t;
        *w = p.accumulate ? *w + v : v;
      }
    }
  }
}

// (M, 1 / L) of every (query row, head) of a chunk from its key tiles: 64 of them
// per workgroup, wavefront w taking tiles w, w + 4, ... (few rows leave most of the
// GPU idle, and what they wait for is one load after the other: 2048 rows over 32
// tiles took 6.4 us with a thread each).
__global__ __launch_bounds__(kThreads) void key_stats_join(const WeightParams p) {
  __shared__ float2 red[kWaves][kWave];
  const int64_t rows = int64_t(p.tok_hi - p.tok_lo) * p.hq;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i = min(int64_t(blockIdx.x) * kWave + lane, rows - 1);
  const int row = p.tok_lo + int(i / p.hq);
  int lo = 0, hi = p.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (p.start_loc[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  int begin, count;
  request_rows(p, lo, begin, count);
  const bool owned = row >= begin && row - begin < count;  // not behind the last request
  const int end = owned ? rows_of(p, clamp_rows(p.lens[lo], p.max_len), count, row - begin) : 0;
  const int tiles = (end + kKeys - 1) / kKeys;
  const float2 *part = reinterpret_cast<const float2 *>(p.part) + i;
  float m = -__builtin_inff(), l = 0.f;
  auto add = [&](float2 v) {
    const float mx = fmaxf(m, v.x);
    l = (l != 0.f ? __builtin_amdgcn_exp2f(m - mx) * l : 0.f) + (v.y != 0.f ? __builtin_amdgcn_exp2f(v.x - mx) * v.y : 0.f);
    m = mx;
  };
#pragma unroll 8
  for (int t = wave; t < tiles; t += kWaves) add(part[int64_t(t) * rows]);
  red[wave][lane] = float2{m, l};
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) add(red[w][lane]);
  if (owned && int64_t(blockIdx.x) * kWave + lane < rows)
    reinterpret_cast<float2 *>(p.stat)[int64_t(p.tok_lo) * p.hq + i] =
        float2{m == -__builtin_inff() ? 0.f : m, l != 0.f ? 1.f / l : 0.f};
}

// Adds the row splits' sums, in order.
__global__ __launch_bounds__(kThreads) void key_sums_join(const WeightParams p) {
  const int t = int(blockIdx.x) * kThreads + threadIdx.x, h = int(blockIdx.y), b = int(blockIdx.z);
  const int len = clamp_rows(p.lens[b], p.max_len);
  if (t >= len) return;
  const int64_t bh = int64_t(b) * p.hkv + h;
  int begin, count, first, end;
  request_rows(p, b, begin, count);
  rows_that_see(p, t / kKeys * kKeys, len, begin, count, first, end);
  const int splits = max(1, int((int64_t(end) - first + p.split_rows - 1) / p.split_rows));
  float v = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) v += p.part_w[(int64_t(s) * p.batch * p.hkv + bh) * p.w_pad + t];
  float *w = p.weights + bh * p.w_stride + t;
  *w = p.accumulate ? *w + v : v;
}

// ------------------------------------------------------------- host side

struct WeightPlan {
  bool mfma;
  int tiles, row_splits, split_rows;
  int64_t chunk_tokens;  // query tokens whose partial statistics are held at once
};

constexpr int64_t kPartBytes = int64_t(64) << 20;

// Query rows of a workgroup.  512 workgroups run at a time (two per CU); one
// costs its rows and, for its keys' decode, about 128 more at D = 256, and the
// last ones leave half a workgroup's time of idle CUs.  For one causal prompt
// of 4096 tokens, 4 KV heads of 4 query heads each, both passes measured 327 us
// with 128 rows, 244 with 256, 237 with 384, 233 with 576, 220 with 672, 223
// with 768, 250 with 1024, 272 with 1152 (one workgroup per slot, unevenly over
// the XCDs).
int64_t best_split(int64_t items, int64_t tiles, int64_t d, int64_t group, int64_t max_query, int64_t max_len, bool causal) {
  const int64_t rows = max_query * group, step = std::max<int64_t>(1, tiles / 32);
  int64_t best = 0, best_cost = 0;
  for (int64_t split = 128;; split += std::max<int64_t>(32, split / 16 / 32 * 32)) {
    split = std::min<int64_t>(split, (rows + kStage - 1) / kStage * kStage);
    int64_t groups = 0;
    for (int64_t j = 0; j < tiles; j += step) {  // a sample of the tiles where there are many
      const int64_t first = causal ? std::max<int64_t>(0, j * kKeys - (max_len - max_query)) * group : 0;
      groups += std::max<int64_t>(1, (rows - std::min(first, rows) + split - 1) / split) * std::min(step, tiles - j);
    }
    const int64_t count = items * groups;
    const int64_t cost = std::max<int64_t>(512, count + 256) * (split + 32 + 3 * d / 8);
    if (!best || cost < best_cost) {
      best = split;
      best_cost = cost;
    }
    if (split >= rows || split >= 8192) break;
  }
  return best;
}

WeightPlan plan_weights(int64_t batch, int64_t heads, int64_t hkv, int64_t d, int64_t block_size, int64_t total_q,
                        int64_t max_query, int64_t max_len, bool causal) {
  WeightPlan pl{};
  const int64_t group = heads / hkv;
  pl.mfma = (d == 64 || d == 128 || d == 256) && block_size % 16 == 0 && block_size / 16 < (int64_t(1) << 20) &&
            (max_len / 16 + 1) * (block_size / 16) < (int64_t(1) << 36) && max_query * group * group < (int64_t(1) << 31);
  if (!pl.mfma) return pl;
  pl.tiles = int((max_len + kKeys - 1) / kKeys);
  const int64_t rows = max_query * group;
  pl.split_rows = int(best_split(batch * hkv, pl.tiles, d, group, max_query, max_len, causal));
  pl.row_splits = int((rows + pl.split_rows - 1) / pl.split_rows);
  pl.chunk_tokens = std::min<int64_t>(total_q, std::max<int64_t>(64, kPartBytes / (int64_t(pl.tiles) * heads * 8)));
  return pl;
}

// The statistics, then the chunk's partial ones, then the row splits' sums.
struct WeightSpace {
  size_t stat, part, part_w;
};

WeightSpace weight_space(const WeightPlan &pl, int64_t batch, int64_t heads, int64_t hkv, int64_t total_q,
                         int64_t max_len) {
  WeightSpace w{};
  w.stat = (size_t(total_q) * heads * 8 + 255) / 256 * 256;
  if (pl.mfma) {
    w.part = (size_t(pl.tiles) * size_t(pl.chunk_tokens) * heads * 8 + 255) / 256 * 256;
    if (pl.row_splits > 1) w.part_w = size_t(pl.row_splits) * batch * hkv * size_t(pl.tiles) * kKeys * 4;
  }
  return w;
}

template <int kD, bool kBf16, typename BtT>
void launch_weights(WeightParams p, const WeightPlan &pl, hipStream_t s) {
  const dim3 blocks(8, unsigned(p.tiles), unsigned((int64_t(p.batch) * p.hkv * p.row_splits + 7) / 8));
  for (int64_t lo = 0; lo < p.total_q; lo += pl.chunk_tokens) {
    p.tok_lo = int(lo);
    p.tok_hi = int(std::min<int64_t>(p.total_q, lo + pl.chunk_tokens));
    key_pass_mfma<kD, kBf16, false, BtT><<<blocks, kThreads, 0, s>>>(p);
    const int64_t rows = int64_t(p.tok_hi - p.tok_lo) * p.hq;
    key_stats_join<<<unsigned((rows + kWave - 1) / kWave), kThreads, 0, s>>>(p);
  }
  p.tok_lo = 0;
  p.tok_hi = p.total_q;
  key_pass_mfma<kD, kBf16, true, BtT><<<blocks, kThreads, 0, s>>>(p);
  if (p.part_w)
    key_sums_join<<<dim3(unsigned((p.max_len + kThreads - 1) / kThreads), unsigned(p.hkv), unsigned(p.batch)), kThreads, 0,
                    s>>>(p);
}

template <bool kBf16, typename BtT>
void launch_key_weights(const WeightParams &p, const WeightPlan &pl, unsigned rows, unsigned sums, hipStream_t s) {
  if (!pl.mfma) {
    if (rows) key_stats_any<kBf16, BtT><<<rows, kThreads, 0, s>>>(p);
    key_sums_any<kBf16, BtT><<<sums, kThreads, 0, s>>>(p, int((p.max_len + 63) / 64));
  } else if (p.d == 64) {
    launch_weights<64, kBf16, BtT>(p, pl, s);
  } else if (p.d == 128) {
    launch_weights<128, kBf16, BtT>(p, pl, s);
  } else {
    launch_weights<256, kBf16, BtT>(p, pl, s);
  }
}

}  // namespace
}  // namespace hif8

using namespace hif8;

extern "C" size_t hif8_key_weights_workspace_size(int64_t batch, int64_t num_heads, int64_t num_kv_heads,
                                                  int64_t head_size, int64_t block_size, int64_t total_query_tokens,
                                                  int64_t max_query_len, int64_t max_seq_len, int causal) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_size <= 0 || block_size <= 0 ||
      total_query_tokens < 0 || max_query_len < 0 || max_seq_len <= 0 || num_heads % num_kv_heads)
    return 0;
  // Either kernel: the query's alignment, which also decides, is not known here.
  const WeightPlan pl = plan_weights(batch, num_heads, num_kv_heads, head_size, block_size, total_query_tokens,
                                     std::max<int64_t>(max_query_len, 1), max_seq_len, causal != 0);
  const WeightSpace w = weight_space(pl, batch, num_heads, num_kv_heads, total_query_tokens, max_seq_len);
  return w.stat + w.part + w.part_w;
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
  WeightPlan pl = plan_weights(batch, num_heads, num_kv_heads, head_size, block_size, total_query_tokens,
                               std::max<int64_t>(max_query_len, 1), max_seq_len, causal != 0);
  const WeightSpace w = weight_space(pl, batch, num_heads, num_kv_heads, total_query_tokens, max_seq_len);
  const size_t need = w.stat + w.part + w.part_w;
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
  p.max_query = int(std::min<int64_t>(max_query_len, total_query_tokens));
  p.causal = causal ? 1 : 0;
  p.accumulate = accumulate ? 1 : 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  if (pl.mfma) {
    p.part = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + w.stat);
    if (w.part_w) p.part_w = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + w.stat + w.part);
    p.w_pad = int64_t(pl.tiles) * kKeys;
    p.magic = ((int64_t(1) << 36) + block_size / 16 - 1) / (block_size / 16);
    p.group_magic = ((int64_t(1) << 32) + p.group - 1) / p.group;
    p.tiles = pl.tiles;
    p.row_splits = pl.row_splits;
    p.split_rows = pl.split_rows;
    // 32-bit launch sizes, and operands that the copies into LDS can take.
    if (!aligned(query, 16) || batch > 0xFFFF || num_kv_heads > 0xFFFF ||
        pl.tiles > 0xFFFF || (batch * num_kv_heads * pl.row_splits + 7) / 8 > 0xFFFF)
      pl.mfma = false;
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool bf16 = q_dtype == HIF8_DTYPE_BF16, i64 = block_table_dtype == HIF8_INDEX_INT64;
  const unsigned rows = unsigned(total_query_tokens * num_heads), sums = unsigned(batch * num_kv_heads * tiles);
  if (bf16 && i64) launch_key_weights<true, int64_t>(p, pl, rows, sums, s);
  else if (bf16) launch_key_weights<true, int32_t>(p, pl, rows, sums, s);
  else if (i64) launch_key_weights<false, int64_t>(p, pl, rows, sums, s);
  else launch_key_weights<false, int32_t>(p, pl, rows, sums, s);
  return check_launch(kName);
}
