// A few query rows per request over the whole HiF8 paged cache, for gfx950.
//
//   hif8_tree_attention                  drafted tokens under a tree mask
//   hif8_paged_decode_attention_weights  one token per request, and the sum of
//                                        its heads' softmax weights per cached row
//   hif8_window_attention                new tokens within a sliding window
//
// o_i = sum_t p_it V_t with p_i = softmax over the rows t that query row i sees
// of scale * q_i . K_t; a query row that sees nothing gets zeros.  K_t and V_t
// are dec(code) * row scale.  Logits, maxima, weights, their sums and the scales
// are FP32 numbers (a weight below 2^-126 of its row's largest is zero); the
// any-shape kernel multiplies FP32 throughout, the matrix cores take codes and
// query as they are and the weights with V's scale in 16 bits, see below.
#include <stddef.h>

#include <algorithm>
#include <type_traits>

#include "mfma_lookup.h"
#include "row_attention.h"

namespace hif8 {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxSplits = 256;  // any-shape kernel
constexpr int kMaxParts = 512;   // parts of a query row: splits, or workers

// Any head size up to 512, group, block size and alignment: a workgroup per
// (query row, head, split), its wavefronts taking every fourth cache row with a
// running maximum and sum each, joined through LDS.  Bound by its lookups in a
// global table and a reduction over the lanes for every (query head, cached row):
// 8 x 16 drafts of 16 heads of 96 over 4096 rows take 1.8 ms, where heads of 256
// take 50 us on the matrix cores.
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
  if (left_out(p, count)) return;  // uniform
  const int ctx = clamp_rows(p.lens[b], p.max_len);
  const WindowRows win = p.window ? window_rows(p, ctx, count) : WindowRows{ctx, 0, 0};
  const int at = ctx - count + (row - begin);  // window: this query row's position
  const int len = p.window ? win.rows : rows_seen(p, ctx, count);
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
    const int real = p.window ? win.real(t) : t;
    const int64_t blk = int64_t(bt[real / p.block_size]);
    const bool seen = blk >= 0 && blk < p.num_blocks &&
                      (p.window ? window_sees(p, at, real) : t < ctx || mask[t - ctx] != 0);
    float x = -__builtin_inff();
    if (seen) {
      const int64_t slot = blk * p.block_size + real % p.block_size;
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
  const bool whole = p.num_splits == 1;      // the join leaves the output to this workgroup
  if (threadIdx.x == 0 && (!whole || p.x)) { // one split's are read for weights alone, and there is no room for others
    p.part_ml[2 * part] = mx;
    p.part_ml[2 * part + 1] = total;
  }
  if (!whole && !(total != 0.f)) return;     // nothing seen: this split's outputs are not read
  const float inv = total != 0.f ? 1.f / total : 0.f;
  for (int dim = threadIdx.x; dim < p.dv; dim += kThreads) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      if (f[w] != 0.f) y += f[w] * red_o[w][dim];
    if (whole) static_cast<uint16_t *>(p.out)[size_t(blockIdx.x) * p.dv + dim] = float_to_half_bits<kBf16>(y * inv);
    else p.part_o[part * p.dv + dim] = y * inv;
  }
}

// ---------------------------------------------------- on the matrix cores
//
// Head sizes 64, 128 and 256 (K and V alike), pages of a multiple of 16 rows.
// A workgroup is a worker for (KV head, 16 kRB query rows); its query rows are
// the (draft, head) pairs of the KV head, so every cached code is decoded once
// for all of them.  The tiles of kT cache rows of all requests, one after the
// other, are dealt out to the workers in equal runs (one worker for each
// workgroup that fits on the GPU), so ragged lengths leave none idle; a run that
// reaches into another request goes on with that one's query rows.  Per tile:
//   * S^T = K Q^T: the wavefronts share the tile's rows, loaded from HBM straight
//     into the MFMA A operand (row = lane % 16, 16 codes per lane) and decoded
//     there by the table of mfma_lookup.h; Q is the B operand, in registers (up
//     to 32 rows) or in LDS in operand order (64);
//   * w = 2^(x - m) is the weight, summed in FP32, and P = w s f in fp16 goes to
//     LDS: s is V's row scale, so that V itself stays the exact dec(code), and f a
//     power of two per query row that puts the largest |P| in (1/4, 1] 2^kTop.
//     m and f stand until some |P| passes fp16's range (or the sum of w 2^40); then the
//     wavefronts' largest x and x + log2 |s| meet in LDS, O and the sum are scaled
//     and P is written again, so nearly all tiles have one barrier.  m follows
//     the logits alone and f what is multiplied with V: with one reference for
//     both, rows whose scales lie 2^126 apart fell out of the sum.  P is rounded
//     once: 2^-11 of it, or 2^-25 where it is subnormal (below 2^-14), which is at
//     most 2^-31 of the row's largest; what that leaves may be a second P (rest_of);
//   * O^T += V^T P^T: every wavefront takes 64 dims of 32 or 64 rows, 4 bytes of
//     each row per lane, transposed by the lookup itself (byte q of eight words).
// The next tile's K loads are issued as soon as S is done, its V loads after O.
// Where there are several parts of a row, each is divided by its own sum and f.
//
// What bounds it (16 query and 4 KV heads of 256, 8 x 16384 cached rows, 171 MB):
// one token per request runs at 3.9 TB/s (43 us; reads of one head's rows reach 4.4
// on this layout, a plain stream 6.1); 32 tokens each take 111 us, where the LDS
// lookups (128 per lane and tile), the query operands from LDS and the vector
// instructions around them add up, as the eight wavefronts go through a tile's
// phases together.  In cycles per tile there: S 2100 to 2800, loads 1300 + 700, logits 600, P 1200,
// O 2400 to 2900.  Two workgroups of 16 query rows per row tile, each decoding
// the cache for itself, took 195 us.  Short calls (512 rows) are latency: 10 to 13
// us and 5 for the join, of which the dependent reads of lengths, table and rows
// are three round trips to HBM.  Within a window: 32 requests of a token each over 4096
// rows 67 us (4.1 TB/s) + 8.5 of join, one over 1024 rows 9.9 + 4.7, 11 requests of up to
// five drafts over 1000 rows (24 / 8 heads of 128) 20 + 7.

// log2 of what P stays below where its power of two is chosen.  Below 2^-14 P is
// subnormal, so the higher it starts the smaller the weights that keep their bits
// beside a large one of a V near zero (a first token that draws all attention);
// the lower, the seldomer rows outgrow fp16.  At 8 a weight of 2^-24 is off by at
// most 2^-7 of itself.  With 2, 6, 8 and 10: 8 x 16k under 32 drafts 109.6, 111.7,
// 114.3 and 121.5 us, ragged trees 45.4, 46.8, 48.7 and 51.6, decode 59.8 to 60.2.
// Rows that have grown past it move back whenever the wavefronts meet (only those
// about to overflow: 123 us with 8).
constexpr float kTop = 8.f;
constexpr float kLazy = 14.f;        // log2 of what a weight may reach before a new choice moves the maximum too
constexpr float kMostSum = 0x1p40f;  // weights that add up to more are chosen again without a large P (V scales near zero)

// Wavefronts of a workgroup: four, two workgroups to a CU; with 64 query rows
// eight, one workgroup, since the table and the query rows in LDS leave no room
// for two and the registers of four none for the rows (24 heads of 128 under 61
// drafts each: 44 us against 50 in row tiles of 32; 48 now).
// One of eight too for P in two parts of 32 rows, which leave a second workgroup no
// LDS either, and for a window's 32 rows of 128 dims (7 rows of 32 / 8 heads, 8
// requests within 4096: 39.0 us, in two of four 42.6; 32 within 1024 37.4 and 42.6).
constexpr int waves_of(int d, int row_blocks, bool win, bool rest) {
  return row_blocks > 2 || (row_blocks == 2 && ((win && d == 128) || (rest && d == 64))) ? 8 : 4;
}
constexpr int max_of(int a, int b) { return a > b ? a : b; }
// Cache rows of a tile.  256 of them at D = 64 left one workgroup to a CU (32
// drafts of 16 heads over 8 x 16k: 111 us against 73).
constexpr int tile_rows_of(int d, int row_blocks, bool win, bool rest) {
  return d == 256 && row_blocks <= 2 ? 64 : 32 * waves_of(d, row_blocks, win, rest) / (d / 64) > 128 ? 256 : 128;
}
// Whether what P's rounding to fp16 leaves is multiplied too, as a second P: under a
// window with an fp16 output, which rounds no further than P does (error against
// float64 3.0e-4 without and 2.1e-4 with it; a bf16 output's own is 1.7e-3).  8
// requests within 4096 rows, 16 / 4 heads of 256: one token 28.1 -> 28.9 us, 6 rows
// 37.6 -> 39.5, 40 rows 71 -> 84; 32 / 8 heads of 128, 40 rows 86 -> 104; 16 / 4 of
// 64, 40 rows 42 -> 54.  1 to 4 % of a call is the look for infinities in V.
constexpr bool rest_of(bool bf16, bool window) { return window && !bf16; }

template <int kD, bool kBf16, int kRB, bool kX, bool kWin, typename BtT>
__global__ __launch_bounds__(64 * waves_of(kD, kRB, kWin, rest_of(kBf16, kWin)), 2) void row_attention_mfma(const RowAttnParams p,
                                                                            const uint32_t page_magic) {
  constexpr bool kRest = rest_of(kBf16, kWin);
  constexpr int kW = waves_of(kD, kRB, kWin, kRest);  // wavefronts
  constexpr bool kQLds = kRB > 2;         // the query rows lie in LDS, in operand order, instead of registers
  constexpr int kRow = kD + 4;
  constexpr int kT = tile_rows_of(kD, kRB, kWin, kRest);  // cache rows of a tile
  constexpr int kKB = kT / 16 / kW;       // 16-row blocks of a wavefront in S
  constexpr int kQS = kD / 32;            // MFMA steps over the head dims
  constexpr int kSlices = kD / 64;        // 64-dim slices of V
  constexpr int kVG = kW / kSlices;       // wavefronts that share a slice, kVR rows of the tile each
  constexpr int kVR = kT / kVG;
  constexpr int kGroups = kT / 16;        // 16-row groups of a tile
  static_assert(kGroups < 32 && kVR % 32 == 0 && kKB * kW * 16 == kT, "a bit per group, whole MFMA steps");
  constexpr int kRows = 16 * kRB;
  constexpr int kPStride = kT + 8;        // fp16 values of a row of P in LDS
  constexpr int kP = kRows * kPStride * (kRest ? 2 : 1);  // values of P, and of its rest behind it
  // Two buffers of P where that leaves room for two workgroups of four wavefronts, or one of eight.
  constexpr int kBuffers =
      (kW == 8 ? !kRest : kLookupBytes + 4 * kP + 32 * kRows + 64 <= 81920 - 1024) ? 2 : 1;
  struct Smem {
    uint32_t table[kLookupBytes / 4];     // at LDS byte 0: a lookup's address needs no addition
    // P of a tile and of the next; at a segment's end the shares of O of wavefronts of one slice.
    __attribute__((aligned(16))) uint16_t pt[max_of(kBuffers * kP, (kVG - 1) * kSlices * 2048)];
    lk_u32x4 q[kQLds ? kRB * kQS * kWave : 1];
    float top[2][kW][kRows];              // a wavefront's largest logit, and logit + log2 of V's scale, per query row
    int grow[2];                          // the last tile (counted from 1) whose P grew too large, by parity
  };
  __shared__ __attribute__((aligned(16))) Smem sm;
  const uint32_t table = lds_address(sm.table);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const uint32_t lane4 = uint32_t(4 * lane);
  // The row tiles of one (worker, KV head) read the same cache rows: their blocks
  // are equal modulo 8 (the grid's x), on one XCD.  So are all of a worker's KV
  // heads, whose rows share cache lines, where that spreads the workers evenly.
  const int outer = int(blockIdx.z) * 8 + int(blockIdx.x), rest = int(blockIdx.y);
  int worker = outer, rt = rest, h = 0;
  if (p.heads_together) {
    if (p.row_tiles == 1) rt = 0, h = rest;
    else h = rest / p.row_tiles, rt = rest - h * p.row_tiles;
  } else {
    worker = outer / p.hkv;
    h = outer - worker * p.hkv;
  }
  if (worker >= p.workers) return;  // padding block (uniform)
  // This worker's run of the requests' tiles, and the running total per request
  // (kept for the join by the first workgroup).  incl: of the first 64 requests.
  struct Request {
    int begin, count, ctx;
  };
  auto request = [&](int i) {
    Request r;
    request_rows(p, i, r.begin, r.count);
    r.ctx = clamp_rows(p.lens[i], p.max_len);
    if (kWin && left_out(p, r.count)) r.count = 0;
    return r;
  };
  // Cache rows that a request's query rows see, pushed together under a window.
  auto rows_of = [&](const Request &r) {
    if constexpr (kWin) return r.count > 0 ? window_rows(p, r.ctx, r.count).rows : 0;
    else return rows_seen(p, r.ctx, r.count);
  };
  auto tiles_of = [&](const Request &r) { return int((uint32_t(rows_of(r)) + uint32_t(kT) - 1) / kT); };
  int total = 0, incl = 0;
  Request early{};  // lane i: request i
  for (int base = 0; base < p.batch; base += kWave) {
    const int i = base + lane;
    const Request r = request(min(i, p.batch - 1));
    const int mine = i < p.batch ? tiles_of(r) : 0;
    const int upto = wave_prefix(mine);
    if (base == 0) {
      incl = upto;
      early = r;
    }
    if (worker == 0 && rt == 0 && h == 0 && wave == 0 && i < p.batch) p.plan[i] = total + upto - mine;
    total += __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  if (worker == 0 && rt == 0 && h == 0 && tid == 0) p.plan[p.batch] = total;
  const int workers = min(p.workers, total);  // a tile each at least: no part is left unwritten
  if (worker >= workers) return;              // uniform
  int cur, run_end;
  if (total < 1 << 22) {  // workers is at most 512: the divisions have 32 bits
    cur = int(uint32_t(total) * uint32_t(worker) / uint32_t(workers));
    run_end = int(uint32_t(total) * uint32_t(worker + 1) / uint32_t(workers));
  } else {
    cur = int(int64_t(total) * worker / workers);
    run_end = int(int64_t(total) * (worker + 1) / workers);
  }
  // The request of tile `cur`.  The first one's numbers are in some lane already.
  int b = 0, first = 0;
  auto among_early = [&]() {
    b = __builtin_ctzll(__ballot(incl > cur));
    first = b ? __builtin_amdgcn_readlane(incl, b - 1) : 0;
  };
  Request now{};
  bool known = p.batch <= kWave;
  if (known) {
    among_early();
    now = Request{__builtin_amdgcn_readlane(early.begin, b), __builtin_amdgcn_readlane(early.count, b),
                  __builtin_amdgcn_readlane(early.ctx, b)};
  }
  bool filled = false;
  int tile_no = 0;  // tiles done, over all segments
  if (tid < 2) sm.grow[tid] = 0;

  const uint32_t rec = uint32_t(p.hkv) * kRow;
  const int bs16 = p.block_size >> 4;
  const int vslice = wave % kSlices, vgroup = wave / kSlices;
  const uint32_t k_off = uint32_t(n) * rec + 16u * g;              // K: row n, codes 16 g + 64 i
  uint32_t v_off[4], s_off[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v_off[e] = uint32_t(4 * g + e) * rec + uint32_t(64 * vslice + 4 * n);  // V: row 4 g + e, four dims
    s_off[e] = uint32_t(4 * g + e) * rec + uint32_t(kD);                   // scale of row 4 g + e
  }

  while (cur < run_end) {
  // This segment: the run's tiles of one request (uniform).
  if (!known) {
    if (p.batch <= kWave) {
      among_early();
    } else {
      int before = 0;
      for (int base = 0; base < p.batch; base += kWave) {
        const int i = base + lane;
        const int upto = before + wave_prefix(i < p.batch ? tiles_of(request(i)) : 0);
        const uint64_t past = __ballot(upto > cur);
        if (past) {
          const int at = __builtin_ctzll(past);
          b = base + at;
          first = at ? __builtin_amdgcn_readlane(upto, at - 1) : before;
          break;
        }
        before = __builtin_amdgcn_readlane(upto, kWave - 1);
      }
    }
    b = __builtin_amdgcn_readfirstlane(b);
    now = request(b);
  }
  known = false;
  const int begin = now.begin, count = now.count;
  const int rows = count * p.group;
  const int ctx = now.ctx;
  const int len = rows_of(now);
  const WindowRows win = kWin ? window_rows(p, ctx, count) : WindowRows{0, 0, 0};
  const int tile_first = cur - first;
  const int seg_tiles = min(run_end - cur, int((uint32_t(len) + kT - 1) / kT) - tile_first);
  cur += seg_tiles;
  const bool last_of_run = cur >= run_end;
  if (rt * kRows >= rows) continue;  // uniform: the request has no query rows here
  const int t_begin = tile_first * kT, t_end = min(t_begin + seg_tiles * kT, len);
  const int ntiles = seg_tiles;
  const bool whole = t_begin == 0 && t_end == len;  // this segment holds all of the request's cache rows
  // Rows of part_ml and part_o.  Only the first and the last segment of a run can hold
  // a part of a request: two places per worker, however many requests there are.
  const size_t part_row = (size_t(worker) + b) * p.hkv + h;
  const size_t part_out = (size_t(2 * worker) + (last_of_run ? 1 : 0)) * p.hkv + h;

  // The query token of row r: r / group.
  auto token_of = [&](int r) { return int(__umulhi(2u * uint32_t(r), p.group_magic)); };
  // This lane's query row in row block rb (column n): whether there is one, its
  // row of the query and its head (of the request's first row where there is none).
  // Worked out where it is needed: held over the loop they cost registers.
  struct Row {
    bool ok;
    int query, head;
  };
  auto row_at = [&](int rb) {
    int r = rt * kRows + 16 * rb + n;
    asm volatile("" : "+v"(r));
    const bool ok = r < rows;
    const int tok = ok ? token_of(r) : 0;
    return Row{ok, begin + tok, h * p.group + (ok ? r - tok * p.group : 0)};
  };
  const BtT *bt = static_cast<const BtT *>(p.block_table) + size_t(b) * p.bt_stride;
  // Lane i % kGroups looks up 16-row group i of a tile; the entry is loaded a
  // tile ahead of its use.
  auto group_of = [&](int t0) {
    const int t = min(t0 + 16 * (lane & (kGroups - 1)), t_end - 1);
    return (kWin ? win.real(t) : t) >> 4;
  };
  auto block_at = [&](int t0) {
    const int gr = group_of(t0);
    return bt[__umulhi(2u * uint32_t(gr), page_magic)];  // not widened here: that would wait for it
  };
  // Byte offset of the group's first row of this KV head, or -1.
  const uint32_t page_bytes = uint32_t(p.block_size) * rec;
  auto offset_at = [&](int t0, BtT entry) {
    const int64_t blk = int64_t(entry);
    const uint32_t gr = uint32_t(group_of(t0));
    const uint32_t in16 = gr - __umulhi(2u * gr, page_magic) * uint32_t(bs16);
    return blk >= 0 && blk < p.num_blocks && t0 + 16 * (lane & (kGroups - 1)) < t_end
               ? int64_t(uint64_t(uint32_t(blk)) * page_bytes + (16u * in16 * rec + uint32_t(h * kRow)))
               : int64_t(-1);
  };
  auto uniform_offset = [&](int64_t off, int group) {
    const int lo = __builtin_amdgcn_readlane(int(uint64_t(off)), group);
    const int hi = __builtin_amdgcn_readlane(int(uint64_t(off) >> 32), group);
    return int64_t((uint64_t(uint32_t(hi)) << 32) | uint32_t(lo));
  };

  lk_u32x4 kraw[kKB][kSlices];
  float ks[kKB][4], vs[kKB][4];
  uint32_t vraw[kVR / 32][8];
  int64_t off_lane = -1;   // group offsets of the tile whose K is in flight
  uint32_t ok_groups = 0;  // its groups that lie in the cache, a bit each
  // Buffer loads: the 16-row group's address in scalar registers, a 32-bit offset
  // per lane (64-bit addresses per load were spilled), nothing past the group.
  const int span = int(15 * rec + uint32_t(kRow));
  auto group_rows = [&](const uint8_t *cache, int group) {
    const int64_t off = uniform_offset(off_lane, group);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(cache + (off < 0 ? 0 : off)), 0, span, 0x00027000);
  };
  auto load_k = [&]() {
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb) {
      const auto kp = group_rows(p.key_cache, wave * kKB + kb), vp = group_rows(p.value_cache, wave * kKB + kb);
#pragma unroll
      for (int i = 0; i < kSlices; ++i)
        kraw[kb][i] = __builtin_bit_cast(lk_u32x4, __builtin_amdgcn_raw_buffer_load_b128(kp, k_off + 64 * i, 0, 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ks[kb][e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(kp, s_off[e], 0, 0));
        vs[kb][e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(vp, s_off[e], 0, 0));
      }
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int j = 0; j < kVR / 16; ++j) {
      const auto vp = group_rows(p.value_cache, kVR / 16 * vgroup + j);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        vraw[j >> 1][4 * (j & 1) + e] = __builtin_amdgcn_raw_buffer_load_b32(vp, v_off[e], 0, 0);
    }
  };

  // The query rows first: what is waited for last must not be issued behind the cache.
  // Step 2 i + s of a row block: dims 64 i + 16 g + 8 s + [0, 8).
  lk_u32x4 qf[kQLds ? 1 : kRB][kQLds ? kRB * kQS / kW : kQS];
  if constexpr (kQLds) {
#pragma unroll
    for (int j = 0; j < kRB * kQS / kW; ++j) {
      const int f = wave * (kRB * kQS / kW) + j, i = f % kQS;
      const int r = min(rt * kRows + 16 * (f / kQS) + n, rows - 1), tok = token_of(r);
      const uint16_t *q = static_cast<const uint16_t *>(p.query) +
                          (size_t(begin + tok) * p.hq + h * p.group + (r - tok * p.group)) * kD + 16 * g;
      qf[0][j] = *reinterpret_cast<const lk_u32x4 *>(q + 64 * (i >> 1) + 8 * (i & 1));
    }
  } else {
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb) {
      const Row row = row_at(rb);
      const uint16_t *q = static_cast<const uint16_t *>(p.query) + (size_t(row.query) * p.hq + row.head) * kD + 16 * g;
#pragma unroll
      for (int i = 0; i < kQS; ++i) qf[rb][i] = *reinterpret_cast<const lk_u32x4 *>(q + 64 * (i >> 1) + 8 * (i & 1));
    }
  }
  const BtT blk_first = block_at(t_begin);
  BtT blk_next = block_at(min(t_begin + kT, t_end - 1));
  off_lane = offset_at(t_begin, blk_first);
  ok_groups = uint32_t(__ballot(off_lane >= 0));
  load_k();
  load_v();
  if (!filled) {  // while the first loads are on their way
    fill_lookup<kBf16, 64 * kW>(sm.table, reinterpret_cast<uint32_t *>(sm.pt), tid);
    filled = true;
  }
  int64_t xrow[kX ? kRB : 1];  // rows of p.x, or -1
  if constexpr (kX) {
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb) {
      const Row row = row_at(rb);
      xrow[rb] = row.ok ? int64_t(row.query) * p.hq + row.head : -1;
    }
  }
  lk_f32x4 oacc[kRB][4];
  float m[kRB], f[kRB], l[kRB];
#pragma unroll
  for (int rb = 0; rb < kRB; ++rb) {
    m[rb] = -__builtin_inff();
    f[rb] = 0x1p126f;
    l[rb] = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) oacc[rb][q] = lk_f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if constexpr (kQLds) {
#pragma unroll
    for (int j = 0; j < kRB * kQS / kW; ++j) sm.q[(wave * (kRB * kQS / kW) + j) * kWave + lane] = qf[0][j];
  }
  lds_barrier();
  // The query rows have arrived: without this the loop would wait for them, and
  // with them for every load behind them, in every iteration.  Columns of no
  // row repeat a row of the request and are not written.
  if constexpr (!kQLds) {
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
      for (int i = 0; i < kQS; ++i) asm volatile("" : "+v"(qf[rb][i]));
  }

  // f(no row is masked, row block) for every row block: one copy for all of them,
  // whose latencies overlap, where the registers last for it.
  auto rows_with = [](bool full, auto f) __attribute__((always_inline)) {
    constexpr bool kTogether = kRB * kKB * (kX ? 2 : 1) <= 4;
    if (kTogether && full) {
#pragma unroll
      for (int rb = 0; rb < kRB; ++rb) f(std::true_type{}, rb);
      return;
    }
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb) {
      if (!kTogether && full) f(std::true_type{}, rb);
      else f(std::false_type{}, rb);
    }
  };

  for (int it = 0; it < ntiles; ++it) {
    const int t0 = t_begin + it * kT;
    const uint32_t ok_now = ok_groups;
    // Every row of the tile lies in the cache and every query row sees it (uniform).
    bool full = (ok_now & ((1u << kGroups) - 1u)) == (1u << kGroups) - 1u;
    if constexpr (kWin) {
      // Behind the first rows the tile starts in the last query row's window and ends at or before the first one.
      full = full && t0 + kT <= t_end && t0 >= win.head && int64_t(win.real(t0)) > int64_t(ctx) - 1 - p.window &&
             win.real(t0) + kT - 1 <= ctx - count;
    } else {
      full = full && t0 + kT <= min(ctx, t_end);
    }
    // The rows each query row sees: bit 4 kb + e for cache row 4 g + e of block kb.  All
    // mask bytes are loaded before one is used (clamped into the row; what is no
    // draft does not look at its byte).
    uint32_t seen[kRB];
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb) seen[rb] = 0xFFFFFFFFu;
    if (kWin && !full) {
#pragma unroll
      for (int rb = 0; rb < kRB; ++rb) {
        const int at = ctx - count + (row_at(rb).query - begin);
        uint32_t bits = 0;
#pragma unroll
        for (int kb = 0; kb < kKB; ++kb) {
          const int t = t0 + 16 * (wave * kKB + kb) + 4 * g, real = win.real(t);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool vis = bool((ok_now >> (wave * kKB + kb)) & 1u) & (t + e < t_end) & window_sees(p, at, real + e);
            bits |= uint32_t(vis) << (4 * kb + e);
          }
        }
        seen[rb] = bits;
      }
    } else if (!full) {
      const int base = t0 + 16 * wave * kKB + 4 * g;
      uint32_t byte[kRB][kKB][4];
      if (p.mask) {  // uniform
        const int last = int(min(p.mask_stride, int64_t(p.max_len)) - 1);
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb) {
          const uint8_t *mrow = p.mask + size_t(row_at(rb).query) * p.mask_stride;
#pragma unroll
          for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) byte[rb][kb][e] = mrow[min(max(base + 16 * kb + e - ctx, 0), last)];
        }
      } else {
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
          for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) byte[rb][kb][e] = 1;
      }
#pragma unroll
      for (int rb = 0; rb < kRB; ++rb) {
        uint32_t bits = 0;
#pragma unroll
        for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = base + 16 * kb + e;
            const bool vis = bool((ok_now >> (wave * kKB + kb)) & 1u) & (t < t_end) & ((t < ctx) | (byte[rb][kb][e] != 0));
            bits |= uint32_t(vis) << (4 * kb + e);
          }
        seen[rb] = bits;
      }
    }
    // S^T of this wavefront's rows.
    lk_f32x4 s[kRB][kKB];
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb) {
#pragma unroll
      for (int rb = 0; rb < kRB; ++rb) s[rb][kb] = lk_f32x4{0.f, 0.f, 0.f, 0.f};
      // The lookups (and the query rows) of a step are on their way while the
      // step before multiplies.  Further ahead they would spill.
      auto codes = [&](int i) { return look8<false>(kraw[kb][i >> 1][2 * (i & 1)], kraw[kb][i >> 1][2 * (i & 1) + 1], lane4, table); };
      auto query = [&](int rb, int i) { return kQLds ? sm.q[(rb * kQS + i) * kWave + lane] : qf[kQLds ? 0 : rb][kQLds ? 0 : i]; };
      lk_u32x4 a = codes(0), q[kRB];
#pragma unroll
      for (int rb = 0; rb < kRB; ++rb) q[rb] = query(rb, 0);
#pragma unroll
      for (int i = 0; i < kQS; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        lk_u32x4 a_next = a, q_next[kRB];
        if (i + 1 < kQS) a_next = codes(i + 1);
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb) q_next[rb] = i + 1 < kQS ? query(rb, i + 1) : q[rb];
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb) s[rb][kb] = mfma_16x16x32<kBf16>(a, q[rb], s[rb][kb]);
        a = a_next;
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb) q[rb] = q_next[rb];
      }
    }
    float ksc[kKB][4], vsc[kKB][4];
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ksc[kb][e] = ks[kb][e] * p.scale_log2;
        vsc[kb][e] = vs[kb][e];
        // Taken here, before the registers of ks and vs are loaded again.
        asm volatile("" : "+v"(ksc[kb][e]), "+v"(vsc[kb][e]));
      }
    // The next tile's K, in flight from here to the next S.  Past the last tile
    // the loads go on, to the cache's first rows: loads under a condition would
    // be copied, and so waited for, where the branches meet.
    const BtT blk = blk_next;
    blk_next = block_at(min(t0 + 2 * kT, t_end - 1));
    off_lane = offset_at(t0 + kT, blk);
    ok_groups = uint32_t(__ballot(off_lane >= 0));
    load_k();
    // Logits (base 2).
    float x[kRB][kKB][4];
    auto logits = [&](auto all, int rb) __attribute__((always_inline)) {
      constexpr bool kAll = decltype(all)::value;
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float z = s[rb][kb][e] * ksc[kb][e];
          x[rb][kb][e] = kAll || ((seen[rb] >> (4 * kb + e)) & 1u) ? z : -__builtin_inff();
        }
        if constexpr (kX) {
          const int t = t0 + 16 * (wave * kKB + kb) + 4 * g;
          if (xrow[rb] >= 0 && t < t_end)
            *reinterpret_cast<lk_f32x4 *>(p.x + xrow[rb] * p.x_stride + t) =
                lk_f32x4{x[rb][kb][0], x[rb][kb][1], x[rb][kb][2], x[rb][kb][3]};
        }
      }
    };
    rows_with(full, logits);
    // P against the maximum and the power of two as they stand, which they do in
    // most tiles: one barrier.  Where some wavefront's rows outgrew them (and in a
    // segment's first tile), all of them meet once more for new ones and write P again.
    ++tile_no;
    uint16_t *pt = sm.pt + (kBuffers == 2 ? (tile_no & 1) * kP : 0);
    float psum[kRB];
    bool grow = false;
    auto weights = [&](auto all, int rb) __attribute__((always_inline)) {
      constexpr bool kAll = decltype(all)::value;
      const float ref = m[rb] == -__builtin_inff() ? 0.f : m[rb];
      float most = 0.f;
      psum[rb] = 0.f;
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float pw = __builtin_amdgcn_exp2f(x[rb][kb][e] - ref);
          const bool vis = kAll || ((seen[rb] >> (4 * kb + e)) & 1u);
          const float sum = psum[rb] + pw;
          psum[rb] = vis ? sum : psum[rb];
          w[e] = vis ? pw * vsc[kb][e] * f[rb] : 0.f;
          most = fmaxf(most, fabsf(w[e]));
        }
        const int j = wave * kKB + kb;
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        uint16_t *to = pt + (16 * rb + n) * kPStride + 32 * (j >> 1) + 8 * g + 4 * (j & 1);
        auto store = [&](uint16_t *at) {
          *reinterpret_cast<u32x2 *>(at) =
              u32x2{uint32_t(float_to_f16_bits(w[0])) | (uint32_t(float_to_f16_bits(w[1])) << 16),
                    uint32_t(float_to_f16_bits(w[2])) | (uint32_t(float_to_f16_bits(w[3])) << 16)};
        };
        store(to);
        if constexpr (kRest) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float high = float(static_cast<_Float16>(w[e]));
            w[e] = fabsf(high) < __builtin_inff() ? w[e] - high : 0.f;  // exact
          }
          store(to + kRows * kPStride);
        }
      }
      // A row that has seen nothing yet has no maximum: what it sees first sets one.
      grow |= (most > 65504.f) | (psum[rb] > kMostSum) | ((m[rb] == -__builtin_inff()) & (kAll | (seen[rb] != 0)));
    };
    auto put = [&]() __attribute__((always_inline)) { rows_with(full, weights); };
    if (it > 0) {
      put();
      if (__any(grow) && lane == 0) sm.grow[tile_no & 1] = tile_no;
      lds_barrier();
    }
    if (it == 0 || sm.grow[tile_no & 1] == tile_no) {  // uniform
#pragma unroll
      for (int rb = 0; rb < kRB; ++rb) {
        float tx = -__builtin_inff(), ty = tx;
#pragma unroll
        for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            tx = fmaxf(tx, x[rb][kb][e]);  // what is not seen is -infinity, whatever its scale
            if (vsc[kb][e] != 0.f) ty = fmaxf(ty, x[rb][kb][e] + float(__builtin_amdgcn_frexp_expf(vsc[kb][e])));
          }
        tx = max_over_groups(tx);
        ty = max_over_groups(ty);
        if (g == 0) {
          sm.top[0][wave][16 * rb + n] = tx;
          sm.top[1][wave][16 * rb + n] = ty;
        }
      }
      lds_barrier();
#pragma unroll
      for (int rb = 0; rb < kRB; ++rb) {
        float tx = sm.top[0][0][16 * rb + n], ty = sm.top[1][0][16 * rb + n];
#pragma unroll
        for (int w = 1; w < kW; ++w) {
          tx = fmaxf(tx, sm.top[0][w][16 * rb + n]);
          ty = fmaxf(ty, sm.top[1][w][16 * rb + n]);
        }
        // True where there is no maximum yet; also where a weight above one could take its V scale past float32.
        const bool rise = tx > m[rb] + kLazy || (tx > m[rb] && ty - m[rb] > 127.f);
        const float m_new = rise ? tx : m[rb];
        const float lf = float(__builtin_amdgcn_frexp_expf(f[rb]) - 1);  // f = 2^lf; P < 2^(ty - m + lf)
        if (rise || ty - m_new + lf > kTop) {
          // O is in units of 2^(m - lf), which only grows: what it holds stays in range.
          const bool none = m[rb] == -__builtin_inff();
          const float lf_new = fminf(fmaxf(floorf(m_new - fmaxf(none ? m[rb] : m[rb] - lf, ty - kTop)), -126.f), 126.f);
          const float of_l = none ? 0.f : __builtin_amdgcn_exp2f(m[rb] - m_new);
          const float of_o = none ? 0.f : __builtin_amdgcn_exp2f((m[rb] - m_new) + (lf_new - lf));
          l[rb] *= of_l;
#pragma unroll
          for (int q = 0; q < 4; ++q) oacc[rb][q] *= of_o;
          m[rb] = m_new;
          f[rb] = __uint_as_float(uint32_t(int(lf_new) + 127) << 23);
        }
      }
      put();
      lds_barrier();
    }
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb) l[rb] += psum[rb];
    // O^T += V^T P^T: slots 8 g + e of a 32-row step are rows 4 g + e of its
    // first 16, then of its second 16, as P lies in LDS.
    bool apart = !full;
    if (kRest && full) {
      // Two products of an infinity, with P and with what its rounding leaves, which is zero or of
      // the other sign, would be a NaN.
      uint32_t finite = 0x80808080u;
#pragma unroll
      for (int i = 0; i < kVR / 32; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) finite &= finite_bytes(vraw[i][j]);
      apart = __any(finite != 0x80808080u);
    }
    if (apart) {
      // Rows that are not there, then infinities and NaN among the drafts (or within a
      // window): a query row that does not see one must not meet it in the product.
      bool odd = false;
#pragma unroll
      for (int j = 0; j < kVR / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t &w = vraw[j >> 1][4 * (j & 1) + e];
          const int t = t0 + kVR * vgroup + 16 * j + 4 * g + e;
          w = bool((ok_now >> (kVR / 16 * vgroup + j)) & 1u) & (t < t_end) ? w : 0u;
          odd |= (kWin | (t >= ctx)) & some_not_finite(w);
        }
      if (__any(odd)) {
#pragma unroll 1
        for (int k = 0; k < kVR / 4; ++k) {
          const int j = k >> 2, e = k & 3;
          uint32_t w = 0;
#pragma unroll
          for (int i = 0; i < kVR / 4; ++i) w = i == k ? vraw[i >> 3][i & 7] : w;
          const int t_lane = t0 + kVR * vgroup + 16 * j + 4 * g + e;
#pragma unroll 1
          for (int byte = 0; byte < 4; ++byte) {
            const uint32_t c = (w >> (8 * byte)) & 0xFFu;
            const bool bad = (kWin || t_lane >= ctx) && ((c & 0x7Fu) == 0x6Fu || c == 0x80u);
            uint64_t left = __ballot(bad);
            if (bad) w &= ~(0xFFu << (8 * byte));
            while (left) {
              const int src = __builtin_ctzll(left);
              left &= left - 1;
              const float v = __uint_as_float(decode_bits(uint32_t(__builtin_amdgcn_readlane(int(c), src))));
              const int sg = src >> 4, sn = src & 15;       // row 4 sg + e, dims 64 vslice + 4 sn + byte
              const int t = t0 + kVR * vgroup + 16 * j + 4 * sg + e;
              const int at = kVR * vgroup + 32 * (j >> 1) + 8 * sg + 4 * (j & 1) + e;
#pragma unroll
              for (int rb = 0; rb < kRB; ++rb) {
                // (t, dim) is element sn % 4 of accumulator `byte` in the lanes of group sn / 4.
                const Row row = row_at(rb);
                bool vis = g == (sn >> 2) && row.ok;
                if constexpr (kWin) vis = vis && window_sees(p, ctx - count + (row.query - begin), win.real(t));
                else vis = vis && p.mask[size_t(row.query) * p.mask_stride + (t - ctx)] != 0;
                const uint16_t pb = pt[(16 * rb + n) * kPStride + at];
                const float add = vis ? ((pb & 0x8000u) ? -v : v) : 0.f;
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                  for (int x = 0; x < 4; ++x)
                    if (q == byte && x == (sn & 3) && vis) oacc[rb][q][x] += add;
              }
            }
          }
#pragma unroll
          for (int i = 0; i < kVR / 4; ++i)
            if (i == k) vraw[i >> 3][i & 7] = w;
        }
      }
    }
#pragma unroll
    for (int hf = 0; hf < kVR / 32; ++hf) {
      lk_u32x4 pf[kRB], pr[kRest ? kRB : 1];
#pragma unroll
      for (int rb = 0; rb < kRB; ++rb) {
        const uint16_t *at = pt + (16 * rb + n) * kPStride + kVR * vgroup + 32 * hf + 8 * g;
        pf[rb] = *reinterpret_cast<const lk_u32x4 *>(at);
        if constexpr (kRest) pr[rb] = *reinterpret_cast<const lk_u32x4 *>(at + kRows * kPStride);
      }
      // As above: the next byte's lookups are on their way while one multiplies.
      lk_u32x4 a = look_column<0, true>(vraw[hf], lane4, table);
      auto column = [&](auto byte) {
        constexpr int q = decltype(byte)::value;
        __builtin_amdgcn_sched_barrier(0);
        lk_u32x4 next = a;
        if constexpr (q < 3) next = look_column<q + 1, true>(vraw[hf], lane4, table);
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb) {
          oacc[rb][q] = mfma_16x16x32<false>(a, pf[rb], oacc[rb][q]);
          if constexpr (kRest) oacc[rb][q] = mfma_16x16x32<false>(a, pr[rb], oacc[rb][q]);
        }
        a = next;
      };
      column(std::integral_constant<int, 0>{});
      column(std::integral_constant<int, 1>{});
      column(std::integral_constant<int, 2>{});
      column(std::integral_constant<int, 3>{});
    }
    load_v();
    if constexpr (kBuffers == 1) lds_barrier();  // the next tile writes P where this one is read
  }

  // The wavefronts' shares of the softmax sum, and of O where some share a slice.
  lds_barrier();
#pragma unroll
  for (int rb = 0; rb < kRB; ++rb) {
    const float lt = sum_over_groups(l[rb]);
    if (g == 0) sm.top[0][wave][16 * rb + n] = lt;
  }
  if constexpr (kVG > 1) {
    lk_f32x4 *spill = reinterpret_cast<lk_f32x4 *>(sm.pt);
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb) {
      if (rb > 0) lds_barrier();
      if (vgroup > 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q) spill[(((vgroup - 1) * kSlices + vslice) * 4 + q) * kWave + lane] = oacc[rb][q];
      }
      lds_barrier();
      if (vgroup == 0) {
#pragma unroll
        for (int og = 0; og < kVG - 1; ++og)
#pragma unroll
          for (int q = 0; q < 4; ++q) oacc[rb][q] += spill[((og * kSlices + vslice) * 4 + q) * kWave + lane];
      }
    }
  } else {
    lds_barrier();
  }
  if (vgroup == 0) {
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb) {
      const Row row = row_at(rb);
      if (!row.ok) continue;
      float sum = sm.top[0][0][16 * rb + n];
#pragma unroll
      for (int w = 1; w < kW; ++w) sum += sm.top[0][w][16 * rb + n];
      // O / (l f): l first, f is a power of two that may be far from one.
      const float inv = sum != 0.f ? 1.f / sum : 0.f, inv_f = 1.f / f[rb];
      const size_t in_part = size_t(rt * kRows + 16 * rb + n);
      const int dim = 64 * vslice + 16 * g;  // element e of accumulator q: dim + 4 e + q
      if (whole) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          w[i] = uint32_t(float_to_half_bits<kBf16>(oacc[rb][(2 * i) & 3][i >> 1] * inv * inv_f)) |
                 (uint32_t(float_to_half_bits<kBf16>(oacc[rb][(2 * i + 1) & 3][i >> 1] * inv * inv_f)) << 16);
        lk_u32x4 *o = reinterpret_cast<lk_u32x4 *>(static_cast<uint16_t *>(p.out) +
                                                   (size_t(row.query) * p.hq + row.head) * kD + dim);
        o[0] = lk_u32x4{w[0], w[1], w[2], w[3]};
        o[1] = lk_u32x4{w[4], w[5], w[6], w[7]};
      } else {
        lk_f32x4 *po = reinterpret_cast<lk_f32x4 *>(p.part_o + (part_out * p.rows_cap + in_part) * kD + dim);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          po[e] = lk_f32x4{oacc[rb][0][e], oacc[rb][1][e], oacc[rb][2][e], oacc[rb][3][e]} * inv * inv_f;
      }
      if (g == 0 && vslice == 0) {
        const size_t r = part_row * p.rows_cap + in_part;
        p.part_ml[2 * r] = m[rb];
        p.part_ml[2 * r + 1] = sum;
      }
    }
  }
  lds_barrier();  // the next segment writes sm.top and sm.pt
  }
}

// Joins the parts of every query row and, where the call asks for them, adds
// the heads' weights onto the cached rows:
//   M = max_s m_s, L = sum_s 2^(m_s - M) l_s, out = sum_s 2^(m_s - M) l_s / L o_s,
// o_s the part's own attention (so that nothing in it is larger than a V row),
//   weights[b, h, t] (+)= sum over the heads of h of 2^(x_t - M) / L.
// The first blocks take outputs.  kWide false (few query rows, each with many
// parts): a (row, head, 64 dims) per block, 16 threads of four dims by 16
// groups of parts; kWide true: a (row, head) per wavefront, four dims per lane.
// The rest take 1024 cached rows of a (request, KV head) each.  Every sum has
// one order.
constexpr int kSliceDims = 64;
constexpr int kWeightKeys = 4 * kThreads;

// Where the partial results of query row `row` (request b, its row `tok`) and
// `head` lie: `count` of them, (maximum, sum) `stride` rows apart from `first` on,
// outputs o_stride apart from o_first on, the last of them o_back rows before.
// None: it saw nothing.
struct Parts {
  size_t first, stride;
  int count;
  size_t o_first, o_stride, o_back;
  __device__ size_t output(int s) const { return o_first + s * o_stride - (s == count - 1 ? o_back : 0); }
};

__device__ __forceinline__ Parts parts_of(const RowAttnParams &p, int b, int row, int tok, int head) {
  if (p.workers == 0) {
    int begin, count;
    request_rows(p, b, begin, count);
    const int ctx = clamp_rows(p.lens[b], p.max_len);
    const int len = p.window ? window_rows(p, ctx, count).rows : rows_seen(p, ctx, count);
    const size_t first = (size_t(row) * p.hq + head) * p.num_splits;
    return Parts{first, 1, (len + p.split_tokens - 1) / p.split_tokens, first, 1, 0};
  }
  // Tiles lo .. hi - 1 are the request's; worker w of them has floor(total w / workers) on.
  const int total = p.plan[p.batch], lo = p.plan[b], hi = p.plan[b + 1];
  const int64_t in_request = int64_t(tok) * p.group + head % p.group;
  if (lo == hi || in_request >= p.rows_cap) return Parts{0, 1, 0, 0, 1, 0};  // nothing seen, or past the longest request told
  const int workers = min(p.workers, total);
  int w0, w1, w1_end;
  if (total < 1 << 22) {  // workers is at most 512: the division has 32 bits
    w0 = int((uint32_t(lo + 1) * uint32_t(workers) - 1) / uint32_t(total));
    w1 = int((uint32_t(hi) * uint32_t(workers) - 1) / uint32_t(total));
    w1_end = int(uint32_t(total) * uint32_t(w1 + 1) / uint32_t(workers));
  } else {
    w0 = int((int64_t(lo + 1) * workers - 1) / total);
    w1 = int((int64_t(hi) * workers - 1) / total);
    w1_end = int(int64_t(total) * (w1 + 1) / workers);
  }
  // The request's segment is the last of every worker's run but w1's, which goes on
  // with other requests unless it ends with this one.
  const size_t step = size_t(p.hkv) * p.rows_cap, within = size_t(head / p.group) * p.rows_cap + size_t(in_request);
  return Parts{(size_t(w0) + b) * step + within, step, w1 - w0 + 1, size_t(2 * w0 + 1) * step + within, 2 * step,
               w1_end > hi ? step : 0};
}

// Whether the attention kernel has written this query row's output itself.
__device__ __forceinline__ bool written(const RowAttnParams &p, const Parts &parts) {
  return p.workers > 0 ? parts.count == 1 : p.num_splits == 1;
}

// (M, 1 / L) over the parts; every lane of the calling wavefront gets them.
__device__ __forceinline__ void join_stats(const RowAttnParams &p, const Parts &parts, float &m, float &inv) {
  const int lane = threadIdx.x & 63;
  float mx = -__builtin_inff();
  for (int s = lane; s < parts.count; s += kWave) mx = fmaxf(mx, p.part_ml[2 * (parts.first + s * parts.stride)]);
  mx = wave_max(mx);
  float total = 0.f;
  for (int s = lane; s < parts.count; s += kWave) {
    // A part that saw nothing has l = 0; one with a NaN logit has l = NaN, whatever its maximum.
    const float *ml = p.part_ml + 2 * (parts.first + s * parts.stride);
    if (ml[1] != 0.f) total += __builtin_amdgcn_exp2f(ml[0] - mx) * ml[1];
  }
  total = wave_sum(total);
  m = mx == -__builtin_inff() ? 0.f : mx;
  inv = total != 0.f ? 1.f / total : 0.f;
}

template <bool kBf16, bool kWide>
__global__ __launch_bounds__(kThreads) void row_attention_join(const RowAttnParams p, int dim_slices) {
  __shared__ float red[kThreads / 16][kSliceDims + 4];
  __shared__ float fac[kMaxParts];
  __shared__ float stat[kWave][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t out_rows = int64_t(p.total_q) * p.hq;
  const int64_t out_blocks = kWide ? (out_rows + kWaves - 1) / kWaves : out_rows * dim_slices;
  if (kWide && int64_t(blockIdx.x) < out_blocks) {
    const int64_t r = int64_t(blockIdx.x) * kWaves + wave;
    if (r >= out_rows) return;
    const int row = int(r / p.hq);
    const int b = request_of_row(p, row);
    uint16_t *o_row = static_cast<uint16_t *>(p.out) + size_t(r) * p.dv;
    if (b < 0) {
      if (p.zero_rest)
        for (int dim = lane; dim < p.dv; dim += kWave) o_row[dim] = 0;
      return;
    }
    int begin, count;
    request_rows(p, b, begin, count);
    if (left_out(p, count)) return;
    const Parts parts = parts_of(p, b, row, row - begin, int(r) - row * p.hq);
    if (written(p, parts)) return;
    float m, inv;
    join_stats(p, parts, m, inv);
    for (int d4 = 4 * lane; d4 < p.dv; d4 += 4 * kWave) {
      f32x4_t acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int s = 0; s < parts.count; ++s) {
        const float *ml = p.part_ml + 2 * (parts.first + s * parts.stride);
        const f32x4_t v = *reinterpret_cast<const f32x4_t *>(p.part_o + parts.output(s) * p.dv + d4);
        // A part that saw nothing was not written (any-shape kernel): its rubbish may be no number.
        if (ml[1] != 0.f) acc += __builtin_amdgcn_exp2f(ml[0] - m) * ml[1] * inv * v;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) o_row[d4 + e] = float_to_half_bits<kBf16>(acc[e]);
    }
    return;
  }
  if (int64_t(blockIdx.x) < out_blocks) {
    const int slice = int(blockIdx.x) % dim_slices;
    const int r = int(blockIdx.x) / dim_slices, row = r / p.hq;
    const int b = request_of_row(p, row);
    const int dim = slice * kSliceDims + tid;
    if (b < 0) {  // uniform
      if (p.zero_rest && tid < kSliceDims && dim < p.dv) static_cast<uint16_t *>(p.out)[size_t(r) * p.dv + dim] = 0;
      return;
    }
    int begin, count;
    request_rows(p, b, begin, count);
    if (left_out(p, count)) return;  // uniform
    const Parts parts = parts_of(p, b, row, row - begin, r - row * p.hq);
    if (written(p, parts)) return;  // uniform
    float m, inv;
    join_stats(p, parts, m, inv);
    if (wave == 0)
      for (int s = lane; s < parts.count; s += kWave) {
        const float *ml = p.part_ml + 2 * (parts.first + s * parts.stride);
        fac[s] = ml[1] != 0.f ? __builtin_amdgcn_exp2f(ml[0] - m) * ml[1] * inv : 0.f;
      }
    __syncthreads();
    const int d4 = slice * kSliceDims + 4 * (tid & 15), g = tid >> 4;
    f32x4_t acc{0.f, 0.f, 0.f, 0.f};
    if (d4 < p.dv) {
      for (int s = g; s < parts.count; s += kThreads / 16)
        if (fac[s] != 0.f) acc += fac[s] * *reinterpret_cast<const f32x4_t *>(p.part_o + parts.output(s) * p.dv + d4);
    }
    *reinterpret_cast<f32x4_t *>(&red[g][4 * (tid & 15)]) = acc;
    __syncthreads();
    if (tid >= kSliceDims || dim >= p.dv) return;
    float y = 0.f;
#pragma unroll
    for (int j = 0; j < kThreads / 16; ++j) y += red[j][tid];
    static_cast<uint16_t *>(p.out)[size_t(r) * p.dv + dim] = float_to_half_bits<kBf16>(y);
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
  const size_t r0 = size_t(b) * p.hq + size_t(h) * p.group;
  f32x4_t acc{0.f, 0.f, 0.f, 0.f};
  for (int g0 = 0; g0 < p.group; g0 += kWave) {
    const int here = min(kWave, p.group - g0);
    __syncthreads();
    for (int j = wave; j < here; j += kWaves) {
      float m, inv;
      join_stats(p, parts_of(p, b, b, 0, h * p.group + g0 + j), m, inv);
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
  int split_tokens, num_splits;              // any-shape kernel
  int row_blocks, row_tiles, workers, tile_rows;  // matrix cores: 16-row blocks of a workgroup (0: any-shape kernel)
  int64_t parts, outputs;                    // partial results: rows of part_ml and of part_o
  uint32_t magic;                            // ceil(2^31 / 16-row groups of a page)
};

// The matrix-core kernel's shapes; the query's and output's alignment comes on top.
// Row groups and the bytes of a page have 31 bits there (a page of 2 GiB goes to the other kernel).
bool mfma_rows(int64_t d, int64_t dv, int64_t hkv, int64_t block_size, int64_t max_len) {
  return (d == 64 || d == 128 || d == 256) && dv == d && block_size % 16 == 0 && block_size / 16 < (int64_t(1) << 20) &&
         (max_len / 16 + 1) * (block_size / 16) < (int64_t(1) << 31) &&
         block_size * hkv * (d + 4) < (int64_t(1) << 31);
}

RowPlan plan_rows(bool mfma, int64_t batch, int64_t total_q, int64_t heads, int64_t hkv, int64_t d, int64_t block_size,
                  int64_t max_query, int64_t max_len, bool win, bool rest) {
  RowPlan pl{};
  const int64_t len = std::max<int64_t>(max_len, 1);
  if (!mfma) {
    // About 2048 workgroups, at least 64 cache rows each.
    int64_t splits = std::max<int64_t>(1, 2048 / std::max<int64_t>(total_q * heads, 1));
    splits = std::min<int64_t>(splits, (len + 63) / 64);
    splits = std::min<int64_t>(splits, kMaxSplits);
    pl.split_tokens = int((len + splits - 1) / splits);
    pl.num_splits = int((len + pl.split_tokens - 1) / pl.split_tokens);
    pl.parts = total_q * heads * pl.num_splits;
    pl.outputs = pl.num_splits > 1 ? pl.parts : 0;
    return pl;
  }
  const int64_t rows = std::max<int64_t>(max_query, 1) * (heads / hkv);
  pl.row_blocks = rows <= 16 ? 1 : rows <= 32 || d < 128 ? 2 : 4;
  pl.row_tiles = int((rows + 16 * pl.row_blocks - 1) / (16 * pl.row_blocks));
  pl.magic = uint32_t(((int64_t(1) << 31) + block_size / 16 - 1) / (block_size / 16));
  // A workgroup for each slot that the GPU has: eight wavefronts per CU.
  pl.tile_rows = tile_rows_of(int(d), pl.row_blocks, win, rest);
  const int64_t tiles = batch * ((len + pl.tile_rows - 1) / pl.tile_rows);
  const int64_t slots = 2048 / waves_of(int(d), pl.row_blocks, win, rest) / (hkv * pl.row_tiles);
  pl.workers = int(std::min<int64_t>(std::max<int64_t>(slots, 1), tiles));
  pl.parts = (pl.workers + batch) * hkv * pl.row_tiles * 16 * pl.row_blocks;
  pl.outputs = 2 * pl.workers * hkv * pl.row_tiles * 16 * pl.row_blocks;
  return pl;
}

int64_t x_stride_of(int64_t max_len) { return (std::max<int64_t>(max_len, 1) + 63) / 64 * 64; }

// The partial results, the logits (weights), the plan.
struct RowSpace {
  size_t o, ml, x, plan;
  size_t total() const { return o + ml + x + plan; }
};

RowSpace row_space(const RowPlan &pl, int64_t batch, int64_t total_q, int64_t heads, int64_t dv, int64_t max_len,
                   bool weights) {
  auto round = [](size_t v) { return (v + 255) / 256 * 256; };
  RowSpace w{};
  w.o = round(size_t(pl.outputs) * dv * sizeof(float));
  const bool unread = !pl.row_blocks && pl.num_splits == 1 && !weights;
  w.ml = round(unread ? 1 : size_t(pl.parts) * 2 * sizeof(float));
  if (weights) w.x = round(size_t(total_q) * heads * size_t(x_stride_of(max_len)) * sizeof(float));
  if (pl.row_blocks) w.plan = round(size_t(batch + 1) * sizeof(int32_t));
  return w;
}

// x: XCDs; y: blocks that share a worker's cache rows; z: the workers (by KV head) in eights.
dim3 row_grid(const RowAttnParams &p) {
  const int outer = p.heads_together ? p.workers : p.workers * p.hkv;
  return dim3(8, unsigned(p.row_tiles * (p.heads_together ? p.hkv : 1)), unsigned((outer + 7) / 8));
}

template <int kD, bool kBf16, int kRB, typename BtT>
void launch_rows(const RowAttnParams &p, uint32_t magic, hipStream_t s) {
  const unsigned threads = 64 * waves_of(kD, kRB, p.window != 0, rest_of(kBf16, p.window != 0));
  const dim3 blocks = row_grid(p);
  if (p.window) row_attention_mfma<kD, kBf16, kRB, false, true, BtT><<<blocks, threads, 0, s>>>(p, magic);
  else if (p.x) row_attention_mfma<kD, kBf16, kRB, true, false, BtT><<<blocks, threads, 0, s>>>(p, magic);
  else row_attention_mfma<kD, kBf16, kRB, false, false, BtT><<<blocks, threads, 0, s>>>(p, magic);
}

template <bool kBf16, typename BtT>
void launch_row_attention(const RowAttnParams &p, const RowPlan &pl, hipStream_t s) {
  if (!pl.row_blocks) {
    row_attention_any<kBf16, BtT><<<dim3(unsigned(p.total_q) * unsigned(p.hq), unsigned(p.num_splits)), kThreads, 0, s>>>(p);
    return;
  }
  const auto with_dim = [&](auto dim) {
    constexpr int kD = decltype(dim)::value;
    if (pl.row_blocks == 1) launch_rows<kD, kBf16, 1, BtT>(p, pl.magic, s);
    else if (kD < 128 || pl.row_blocks == 2) launch_rows<kD, kBf16, 2, BtT>(p, pl.magic, s);
    else launch_rows<kD, kBf16, kD < 128 ? 2 : 4, BtT>(p, pl.magic, s);
  };
  if (p.d == 64) with_dim(std::integral_constant<int, 64>{});
  else if (p.d == 128) with_dim(std::integral_constant<int, 128>{});
  else with_dim(std::integral_constant<int, 256>{});
}

}  // namespace

int64_t rows_bound(int64_t max_len, int64_t max_query, int64_t window, int64_t sinks) {
  return window ? std::min(max_len, (sinks + 15) / 16 * 16 + window + max_query + 15) : max_len;
}

// Bytes for either kernel: the query's alignment, which also decides, is not known here.
size_t row_workspace(int64_t batch, int64_t total_q, int64_t heads, int64_t hkv, int64_t d, int64_t dv,
                     int64_t block_size, int64_t max_query, int64_t max_len, bool weights) {
  size_t need = 0;
  for (const bool mfma : {false, true}) {
    if (mfma && !mfma_rows(d, dv, hkv, block_size, max_len)) continue;
    // Under a window there are as many workers or fewer.
    const RowPlan pl = plan_rows(mfma, batch, total_q, heads, hkv, d, block_size, max_query, max_len, false, false);
    need = std::max(need, row_space(pl, batch, total_q, heads, dv, max_len, weights).total());
  }
  return need;
}

int check_row_args(const char *name, const RowArgs &a) {
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
  return HIF8_OK;
}

int row_attention(const char *name, const RowArgs &a) {
  if (const int st = check_row_args(name, a)) return st;
  if (a.batch == 0 || a.total_q == 0) return HIF8_OK;
  const int64_t most_rows = rows_bound(a.max_len, a.max_query, a.window, a.sinks);
  const size_t need = row_workspace(a.batch, a.total_q, a.heads, a.hkv, a.d, a.dv, a.block_size, a.max_query, most_rows,
                                    a.weights != nullptr);
  if (!a.workspace || a.workspace_bytes < need)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes required (got %zu)", name, need,
                a.workspace_bytes);
  if (!aligned(a.workspace, 16))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned", name);

  const int64_t group = a.heads / a.hkv, longest = std::max<int64_t>(a.max_query, 1);
  const bool mfma = mfma_rows(a.d, a.dv, a.hkv, a.block_size, a.max_len) && aligned(a.query, 16) && aligned(a.out, 16) &&
                    longest * group < 0xFFFF * 16 && (longest * group + 64) * group < (int64_t(1) << 31);  // the grid's y, token_of
  if (mfma && a.batch * (a.max_len / 64 + 1) > 0x7FFFFFFFll / 2)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", name);
  const RowPlan pl = plan_rows(mfma, a.batch, a.total_q, a.heads, a.hkv, a.d, a.block_size, a.max_query, most_rows,
                               a.window != 0, rest_of(a.q_dtype == HIF8_DTYPE_BF16, a.window != 0));
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
  p.zero_rest = a.zero_rest;
  p.window = int(a.window);
  p.sinks = int(a.sinks);
  p.most_rows = int(most_rows);
  p.long_rows = a.long_rows ? int(a.long_rows) : 0x7FFFFFFF;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  const size_t rows = size_t(a.total_q) * a.heads;
  const RowSpace space = row_space(pl, a.batch, a.total_q, a.heads, a.dv, most_rows, a.weights != nullptr);
  uint8_t *ws = static_cast<uint8_t *>(a.workspace);
  p.part_o = reinterpret_cast<float *>(ws);
  p.part_ml = reinterpret_cast<float *>(ws + space.o);
  if (a.weights) {
    p.x = reinterpret_cast<float *>(ws + space.o + space.ml);
    p.x_stride = x_stride_of(a.max_len);
    p.weights = a.weights;
    p.w_stride = a.w_stride;
  }
  if (mfma) {
    p.plan = reinterpret_cast<int32_t *>(ws + space.o + space.ml + space.x);
    p.workers = pl.workers;
    p.heads_together = pl.workers % 8 == 0;
    p.row_tiles = pl.row_tiles;
    p.rows_cap = pl.row_tiles * 16 * pl.row_blocks;
    p.group_magic = uint32_t(((int64_t(1) << 31) + p.group - 1) / p.group);
  }
  const int dim_slices = int((a.dv + kSliceDims - 1) / kSliceDims);
  // From 1024 (row, head) pairs on, a wavefront each fills the GPU (192 rows of 16
  // heads, about four parts each: 37 us in slices).
  const bool wide = int64_t(rows) >= 1024;
  const int64_t join_blocks = (wide ? (int64_t(rows) + kWaves - 1) / kWaves : int64_t(rows) * dim_slices) +
                              (a.weights ? a.batch * a.hkv * ((a.max_len + kWeightKeys - 1) / kWeightKeys) : 0);
  if (std::max(join_blocks, int64_t(rows)) > 0xFFFFFFFFll / kThreads)  // threads of one launch
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", name);
  hipStream_t s = reinterpret_cast<hipStream_t>(a.stream);
  const bool bf16 = a.q_dtype == HIF8_DTYPE_BF16, i64 = a.bt_dtype == HIF8_INDEX_INT64;
  if (bf16 && i64) launch_row_attention<true, int64_t>(p, pl, s);
  else if (bf16) launch_row_attention<true, int32_t>(p, pl, s);
  else if (i64) launch_row_attention<false, int64_t>(p, pl, s);
  else launch_row_attention<false, int32_t>(p, pl, s);
  const unsigned blocks = unsigned(join_blocks);
  if (bf16 && wide) row_attention_join<true, true><<<blocks, kThreads, 0, s>>>(p, dim_slices);
  else if (bf16) row_attention_join<true, false><<<blocks, kThreads, 0, s>>>(p, dim_slices);
  else if (wide) row_attention_join<false, true><<<blocks, kThreads, 0, s>>>(p, dim_slices);
  else row_attention_join<false, false><<<blocks, kThreads, 0, s>>>(p, dim_slices);
  return check_launch(name);
}

}  // namespace hif8

using namespace hif8;

extern "C" size_t hif8_tree_attention_workspace_size(int64_t batch, int64_t num_heads, int64_t num_kv_heads,
                                                     int64_t head_size, int64_t head_size_v, int64_t block_size,
                                                     int64_t total_query_tokens, int64_t max_query_len,
                                                     int64_t max_seq_len) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_size <= 0 || head_size_v <= 0 ||
      block_size <= 0 || total_query_tokens <= 0 || max_query_len <= 0 || max_seq_len < 0 || num_heads % num_kv_heads)
    return 0;
  return row_workspace(batch, total_query_tokens, num_heads, num_kv_heads, head_size, head_size_v, block_size,
                       max_query_len, max_seq_len, false);
}

namespace {

int tree_attention(const char *name, const RowArgs &a) {
  clear_error();
  if (a.max_query < 0 || a.mask_stride < 0)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions must be positive", name);
  if (a.batch > 0 && a.total_q > 0) {
    if (a.max_query == 0)
      return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: max_query_len must cover the query rows", name);
    if (a.mask_stride < a.max_query)
      return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: tree_mask rows are shorter than max_query_len", name);
    if (!a.mask || !a.start_loc) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: null pointer argument", name);
  }
  return row_attention(name, a);
}

}  // namespace

extern "C" int hif8_tree_attention(const void *query, int q_dtype, const uint8_t *key_cache,
                                   const uint8_t *value_cache, int64_t num_blocks, int64_t block_size,
                                   int64_t num_kv_heads, int64_t head_size, int64_t head_size_v,
                                   const void *block_table, int block_table_dtype, int64_t max_blocks_per_seq,
                                   const int32_t *query_start_loc, const int32_t *context_lens,
                                   const uint8_t *tree_mask, int64_t mask_width, int64_t batch, int64_t num_heads,
                                   int64_t total_query_tokens, int64_t max_query_len, int64_t max_seq_len,
                                   float scale, void *out, void *workspace, size_t workspace_bytes,
                                   hif8_stream_t stream) {
  return tree_attention("hif8_tree_attention",
                        RowArgs{query, q_dtype, key_cache, value_cache, num_blocks, block_size, num_kv_heads, head_size,
                                head_size_v, block_table, block_table_dtype, max_blocks_per_seq, query_start_loc,
                                context_lens, tree_mask, mask_width, batch, num_heads, total_query_tokens, max_query_len,
                                max_seq_len, scale, out, nullptr, 0, 0, 0, workspace, workspace_bytes, stream});
}

extern "C" int hif8_tree_attention_padded(const void *query, int q_dtype, const uint8_t *key_cache,
                                          const uint8_t *value_cache, int64_t num_blocks, int64_t block_size,
                                          int64_t num_kv_heads, int64_t head_size, int64_t head_size_v,
                                          const void *block_table, int block_table_dtype, int64_t max_blocks_per_seq,
                                          const int32_t *query_start_loc, const int32_t *context_lens,
                                          const uint8_t *tree_mask, int64_t mask_width, int64_t batch, int64_t num_heads,
                                          int64_t total_query_tokens, int64_t max_query_len, int64_t max_seq_len,
                                          float scale, void *out, void *workspace, size_t workspace_bytes,
                                          hif8_stream_t stream) {
  return tree_attention("hif8_tree_attention_padded",
                        RowArgs{query, q_dtype, key_cache, value_cache, num_blocks, block_size, num_kv_heads, head_size,
                                head_size_v, block_table, block_table_dtype, max_blocks_per_seq, query_start_loc,
                                context_lens, tree_mask, mask_width, batch, num_heads, total_query_tokens, max_query_len,
                                max_seq_len, scale, out, nullptr, 0, 0, 1, workspace, workspace_bytes, stream});
}

extern "C" size_t hif8_paged_decode_attention_weights_workspace_size(int64_t batch, int64_t num_heads,
                                                                     int64_t num_kv_heads, int64_t head_size,
                                                                     int64_t head_size_v, int64_t block_size,
                                                                     int64_t max_seq_len) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_size <= 0 || head_size_v <= 0 || block_size <= 0 ||
      max_seq_len < 0 || num_heads % num_kv_heads)
    return 0;
  return row_workspace(batch, batch, num_heads, num_kv_heads, head_size, head_size_v, block_size, 1, max_seq_len, true);
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
                                      nullptr, seq_lens, nullptr, 0, batch, num_heads, batch, 1, max_seq_len, scale, out,
                                      key_weights, weights_stride, accumulate, 0, workspace, workspace_bytes, stream});
}
