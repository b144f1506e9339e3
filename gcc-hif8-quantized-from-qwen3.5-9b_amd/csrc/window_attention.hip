// Attention within a sliding window over the HiF8 paged cache, for gfx950: the
// query row at position P sees the cached rows t <= P with t > P - window or
// t < sinks.  o = sum_t p_t V_t, p the softmax of scale * q . K_t over the rows
// seen; K_t and V_t are dec(code) * row scale; a row that sees nothing gets zeros.
//
// Requests of few query rows run on the kernels of row_attention.hip.  Longer ones
// (chunks of a prompt, whole prompts) run here, in two steps:
//   * window_image_kernel decodes every 32 cached rows that some query row of the
//     request sees into an image: the MFMA operands of K and of V^T as fragments
//     of 1 KiB, 16 bytes a lane, and the row scales beside them.  Codes are exact in
//     bf16 and fp16, so nothing is rounded;
//   * window_attention_kernel: a workgroup takes items (request, KV head, up to 256 or
//     384 (token, head) rows), 32 rows a wavefront, and walks the images of
//     the rows it sees.  Per image S^T = K Q^T and O^T += V^T P^T on
//     v_mfma_f32_32x32x16, a softmax with a running maximum between them;
//   * window_join_kernel joins the items that lie in several workgroups' runs.
// The rows seen are pushed together in groups of 16 (WindowRows), so the first rows
// cost their own groups and no tile of their own.
#include <stddef.h>

#include <algorithm>
#include <type_traits>

#include "mfma_lookup.h"
#include "row_attention.h"

namespace hif8 {
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
// Query and output rows: global memory takes any alignment in one access.
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32_a2 __attribute__((aligned(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;  // of the kernels around the attention
constexpr int kKeys = 32;      // cached rows of an image
// Wavefronts of the attention's workgroups, 32 (token, head) rows each, and workgroups per
// CU: as many wavefronts as the registers hold, in few workgroups, since every one copies
// the images into its own LDS.
constexpr int waves_of(int d) { return d == 128 ? 12 : 8; }
constexpr int groups_per_cu(int d) { return d == 64 ? 2 : 1; }
constexpr int rows_of(int d) { return 32 * waves_of(d); }
constexpr int kStages = 4;     // images in LDS: two that are worked on, two on their way
constexpr int kMaxSlots = 1024;  // requests of a pass

// An image: K fragments [D / 16], V fragments [D / 32][2], then K's scales (times the
// softmax scale, base 2) [32], V's [32], and four words: rows that are there, rows whose V
// holds an infinity or NaN, and Room of V's scales.
constexpr int frag_bytes(int d) { return 2 * kKeys * d * 2; }
constexpr int img_bytes(int d) { return (frag_bytes(d) + 8 * kKeys + 16 + 1023) / 1024 * 1024; }

struct WindowParams {
  RowAttnParams r;       // request split, lengths, table, caches, window
  uint8_t *img;          // [slots][hkv][tiles]
  int4 *items;           // [most_items][2] of each item: (request, slot, KV head, first query row), (request's first row, rows, cached rows, 0)
  int32_t *plan;         // [items + 1] images before each item, kStart more for each, the last entry all of them
  int32_t *plan_items;   // [1] items of the pass
  int32_t *plan_first;   // [workers] the item in which each run begins
  float *part_o;         // [2 workers][rows_of(D)][D]
  float *part_ml;        // [2 workers][rows_of(D)][2]
  int tiles;             // images per (slot, KV head)
  int slots, first_slot; // requests of this pass; slot s holds the (first_slot + s)-th long request
  int tokens;            // of an item
  int most_items, workers;
  int zero_rest;         // one request: rows of the query outside it get zeros here
};

__device__ __forceinline__ bool is_long(const RowAttnParams &p, int b) {
  int begin, count;
  request_rows(p, b, begin, count);
  return count > 0 && left_out(p, count);
}

// The s-th long request, or -1 (64 requests per round of the wavefront; uniform).
__device__ __forceinline__ int long_request(const RowAttnParams &p, int s) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < p.batch; base += kWave) {
    const uint64_t mask = __ballot(base + lane < p.batch && is_long(p, base + lane));
    const int here = __popcll(mask);
    if (s < here) {
      const int rank = __popcll(mask & ((uint64_t(1) << lane) - 1));
      return base + __builtin_ctzll(__ballot(((mask >> lane) & 1u) != 0 && rank == s));
    }
    s -= here;
  }
  return -1;
}

// The work of a pass: items (KV head, rows_of(D) rows of it) of its requests, one request after
// the other, and the images that each sees.  The images of all items, one item after the
// other, are dealt out to the workers in equal runs, one worker for each workgroup that
// fits on the GPU: an item that does not end in its worker's run goes on in the next
// one's, and its parts are joined afterwards.  An item counts kStart images more than it
// sees, for its start and end (with none a run of fifteen short items took 399 us where
// the others took 262 to 320).  Whole items in two rounds left CUs idle for
// a fifth of the time (8192 rows within 2048: 343 us, of which the workgroups ran 270).

constexpr int kStart = 4;

// The images that the query rows tok0 .. of a request see: the first `sinks` of them, and
// those from `near` on, `total` in all.
struct Walk {
  int sinks, near, total;
  __device__ int image(int i) const { return i < sinks ? i : i - sinks + near; }
};

__device__ __forceinline__ Walk walk_of(const WindowParams &p, int len, int count, const WindowRows &win, int tok0) {
  const int first_at = len - count;  // position of the request's first query row
  const int last = min(win.rows, max(0, first_at + min(tok0 + p.tokens, count) - win.skip));
  const int low = int(max(int64_t(first_at) + tok0 + 1 - p.r.window, int64_t(win.skip))) - win.skip;
  const int sinks = (min(p.r.sinks, last) + kKeys - 1) / kKeys;
  const int near = max(low / kKeys, sinks);
  return Walk{sinks, near, sinks + max((last + kKeys - 1) / kKeys - near, 0)};
}

// Worker w of `workers` has the images floor(total w / workers) on.
__device__ __forceinline__ int run_begin(int total, int w, int workers) { return int(int64_t(total) * w / workers); }

// The plan, by one workgroup.
__device__ void make_plan(const WindowParams &p) {
  __shared__ int first[kMaxSlots], owner[kMaxSlots];  // items before each slot's request, the request
  __shared__ int sums[kThreads / kWave];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int items = 0, rank = -p.first_slot, slots = 0;
  for (int base = 0; base < p.r.batch; base += kWave) {
    const int b = base + lane;
    const bool lng = b < p.r.batch && is_long(p.r, b);
    const uint64_t mask = __ballot(lng);
    const int slot = rank + __popcll(mask & ((uint64_t(1) << lane) - 1));
    rank += __popcll(mask);
    int n = 0;
    const bool mine = lng && slot >= 0 && slot < p.slots;
    if (mine) {
      int begin, count;
      request_rows(p.r, b, begin, count);
      n = int(min(int64_t((count + p.tokens - 1) / p.tokens) * p.r.hkv, int64_t(p.most_items)));
    }
    const int upto = items + wave_prefix(n);
    if (mine && wave == 0) {
      first[slot] = upto - n;
      owner[slot] = b;
    }
    items = min(__builtin_amdgcn_readlane(upto, kWave - 1), p.most_items);  // more only where start_loc is wrong
    slots += __popcll(__ballot(mine));
  }
  __syncthreads();
  int before = 0;
  for (int base = 0; base < items; base += kThreads) {
    const int item = base + tid;
    int mine = 0;
    if (item < items) {
      int s = 0, hi = slots - 1;
      while (s < hi) {
        const int mid = (s + hi + 1) / 2;
        if (first[mid] <= item) s = mid;
        else hi = mid - 1;
      }
      int begin, count;
      request_rows(p.r, owner[s], begin, count);
      const int len = clamp_rows(p.r.lens[owner[s]], p.r.max_len);
      // The last query rows, which see most, first.
      const int tiles = (count + p.tokens - 1) / p.tokens, in = item - first[s];
      const int tok0 = (tiles - 1 - in % tiles) * p.tokens;
      mine = walk_of(p, len, count, window_rows(p.r, len, count), tok0).total;
      if (mine) mine += kStart;
      p.items[2 * item] = make_int4(owner[s], s, in / tiles, tok0);
      p.items[2 * item + 1] = make_int4(begin, count, len, 0);
    }
    const int upto = wave_prefix(mine);
    if (lane == kWave - 1) sums[wave] = upto;
    __syncthreads();
    int left = before;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) {
      left += w < wave ? sums[w] : 0;
      before += sums[w];
    }
    if (item < items) p.plan[item] = left + upto - mine;
    __syncthreads();
  }
  if (tid == 0) {
    p.plan[items] = before;
    *p.plan_items = items;
  }
  __syncthreads();
  // The last item that starts at or before a run does; it has images.
  const int workers = min(p.workers, before);
  for (int w = tid; w < workers; w += kThreads) {
    const int at = run_begin(before, w, workers);
    int lo = 0, hi = items - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (p.plan[mid] <= at) lo = mid;
      else hi = mid - 1;
    }
    p.plan_first[w] = lo;
  }
}

// ------------------------------------------------------------------ images

// A query row's P = 2^(x - r) * V's scale, x its logits: r stands until some P could reach
// 2^kMost (fp16 ends at 2^16), and is then the least at which every P that the row has seen
// stays below 2^kTop.
constexpr float kTop = 7.f, kMost = 15.f;

// How far a logit may lie above its row's r over an image whose scales of V are at most
// `most` and at least `least`; -infinity where some are zero or not within 2^-60 to 2^60:
// sums of 2^(x - r) could leave float32's range there.  And whether one power of two bounds
// all of the scales tightly.
struct Room {
  float logit;
  uint32_t even;
};
__device__ __forceinline__ Room room_of(float most, float least) {
  const int e = __builtin_amdgcn_frexp_expf(most);
  return Room{least >= 0x1p-60f && most <= 0x1p60f ? kMost - float(e) : -__builtin_inff(),
              e == __builtin_amdgcn_frexp_expf(least) ? 1u : 0u};
}

// A workgroup per (slot, KV head, kThreads / D * 32 rows): threads take 16 codes of a K
// row, and 4 codes of eight V rows each.  Bound by the bytes (4 of image and 2 of cache
// per (row, dim), K and V together): 4 x 4608 rows of 4 KV heads of 256, 113 MB, 31 us
// (3.7 TB/s).  The KV
// heads of one tile, whose rows share cache lines, have block ids equal modulo 8: one XCD.
template <int kD, bool kBf16, typename BtT>
__global__ __launch_bounds__(kThreads) void window_image_kernel(const WindowParams p) {
  constexpr int kTiles = kThreads / kD;         // images of a workgroup
  constexpr int kChunks = kD / 16;              // 16-code chunks of a row
  constexpr int kPerTile = kThreads / kTiles;   // threads of an image
  constexpr int kLoads = kKeys * kChunks / kPerTile;
  static_assert(kPerTile == kD && kD % 64 == 0, "a wavefront works on one image");
  __shared__ uint32_t dec[256];  // the query's type below, fp16 (0 where not finite) above
  __shared__ uint32_t odd[kTiles], top[kTiles], low[kTiles];
  const int tid = threadIdx.x;
  if (blockIdx.x < 8) {  // the first eight make the plan or nothing
    if (blockIdx.x == 0) make_plan(p);
    return;
  }
  const int xcd = int(blockIdx.x) & 7, rest = (int(blockIdx.x) >> 3) - 1;
  const int h = rest % p.r.hkv;
  const int group = (rest / p.r.hkv) * 8 + xcd;  // tiles of one slot after the other
  const int groups = (p.tiles + kTiles - 1) / kTiles;
  const int slot = group / groups;
  if (slot >= p.slots) return;                   // padding block (uniform)
  const int b = long_request(p.r, p.first_slot + slot);
  if (b < 0) return;                             // uniform
  int begin, count;
  request_rows(p.r, b, begin, count);
  const int len = clamp_rows(p.r.lens[b], p.r.max_len);
  const WindowRows win = window_rows(p.r, len, count);
  const int first = (group - slot * groups) * kTiles;
  if (first * kKeys >= win.rows) return;         // uniform
  {
    const uint32_t f = decode_bits(uint32_t(tid));
    const bool finite = (tid & 0x7F) != 0x6F && tid != 0x80;
    const uint32_t half = float_to_f16_bits(__uint_as_float(f));
    dec[tid] = (kBf16 ? f >> 16 : half) | (finite ? half << 16 : 0u);
    if (tid < kTiles) {
      odd[tid] = top[tid] = 0;
      low[tid] = 0x7F800000u;
    }
  }
  // Everything of an image is the same in a whole wavefront.
  const int in_group = __builtin_amdgcn_readfirstlane(tid / kPerTile), tile = first + in_group, at = tid % kPerTile;
  const BtT *bt = static_cast<const BtT *>(p.r.block_table) + size_t(b) * p.r.bt_stride;
  const int64_t rec = int64_t(p.r.hkv) * (kD + 4);
  // Offset of this KV head's row in the first row of each of the two groups of 16, or -1.
  auto group_offset = [&](int t) -> int64_t {
    if (t >= win.rows) return -1;
    const int real = win.real(t), col = real / p.r.block_size;
    const int64_t blk = int64_t(bt[col]);
    if (blk < 0 || blk >= p.r.num_blocks) return -1;
    return (blk * p.r.block_size + (real - col * p.r.block_size)) * rec + int64_t(h) * (kD + 4);
  };
  const int64_t off0 = group_offset(tile * kKeys), off1 = group_offset(tile * kKeys + 16);
  auto offset_of = [&](int key) -> int64_t {
    const int64_t off = key < 16 ? off0 : off1;
    return off < 0 || tile * kKeys + key >= win.rows ? int64_t(-1) : off + (key & 15) * rec;
  };
  uint8_t *im = p.img + ((size_t(slot) * p.r.hkv + h) * p.tiles + tile) * img_bytes(kD);
  const bool mine = tile * kKeys < win.rows;
  // K: thread -> (key, chunk), consecutive threads consecutive keys.
  u32x4 kraw[kLoads];
  int64_t koff[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int e = at + kPerTile * i, key = e % kKeys, chunk = e / kKeys;
    koff[i] = offset_of(key);
    kraw[i] = u32x4{0, 0, 0, 0};
    if (koff[i] >= 0) kraw[i] = *reinterpret_cast<const u32x4_a4 *>(p.r.key_cache + koff[i] + 16 * chunk);
  }
  // V: thread -> (four dims, eight keys): slot j of half h2, step s is key 16 s + 8 (j / 4) + 4 h2 + j % 4.
  const int quad = at % (kD / 4), sh = at / (kD / 4), vs = sh >> 1, vh = sh & 1;
  uint32_t vraw[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t off = offset_of(16 * vs + 8 * (j >> 2) + 4 * vh + (j & 3));
    vraw[j] = 0;
    if (off >= 0) vraw[j] = *reinterpret_cast<const uint32_t *>(p.r.value_cache + off + 4 * quad);
  }
  float ksc = 0.f, vsc = 0.f;
  bool there = false;
  if (at < kKeys) {
    const int64_t off = offset_of(at);
    there = off >= 0;
    if (there) {
      ksc = *reinterpret_cast<const float *>(p.r.key_cache + off + kD) * p.r.scale_log2;
      vsc = *reinterpret_cast<const float *>(p.r.value_cache + off + kD);
    }
  }
  __syncthreads();
  if (mine) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int e = at + kPerTile * i, key = e % kKeys, chunk = e / kKeys;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        u32x4 o;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t c = kraw[i][2 * half + (w >> 1)] >> (16 * (w & 1));
          o[w] = __builtin_amdgcn_perm(dec[(c >> 8) & 0xFFu], dec[c & 0xFFu], 0x05040100u);
        }
        *reinterpret_cast<u32x4 *>(im + 1024 * chunk + 16 * (key + 32 * half)) = o;
      }
    }
    uint32_t bad = 0;  // keys of this thread with a value that is not finite
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (some_not_finite(vraw[j])) bad |= 1u << (16 * vs + 8 * (j >> 2) + 4 * vh + (j & 3));
    if (bad) atomicOr(&odd[in_group], bad);
    uint8_t *vim = im + frag_bytes(kD) / 2 + 1024 * ((4 * quad / 32) * 2 + vs) + 16 * (4 * quad % 32 + 32 * vh);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      u32x4 o;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        o[w] = __builtin_amdgcn_perm(dec[(vraw[2 * w + 1] >> (8 * q)) & 0xFFu], dec[(vraw[2 * w] >> (8 * q)) & 0xFFu],
                                     0x07060302u);
      *reinterpret_cast<u32x4 *>(vim + 16 * q) = o;
    }
    if (at < kKeys) {
      const bool finite = fabsf(vsc) < __builtin_inff();
      float *sc = reinterpret_cast<float *>(im + frag_bytes(kD));
      sc[at] = ksc;
      sc[kKeys + at] = finite ? vsc : 0.f;
      if (!finite) atomicOr(&odd[in_group], 1u << at);
      if (there) {
        const uint32_t size = finite ? __float_as_uint(fabsf(vsc)) : 0u;
        atomicMax(&top[in_group], size);
        atomicMin(&low[in_group], size);
      }
    }
    const uint64_t seen = __ballot(there);  // the image's first wavefront
    if (at == 0) reinterpret_cast<uint32_t *>(im + frag_bytes(kD))[2 * kKeys] = uint32_t(seen);
  }
  __syncthreads();
  if (mine && at == 0) {
    const Room room = room_of(__uint_as_float(top[in_group]), __uint_as_float(low[in_group]));
    uint32_t *words = reinterpret_cast<uint32_t *>(im + frag_bytes(kD)) + 2 * kKeys;
    words[1] = odd[in_group];
    words[2] = __float_as_uint(room.logit);
    words[3] = room.even;
  }
}

// --------------------------------------------------------------- attention

template <bool kBf16>
__device__ __forceinline__ f32x16_t mfma32(u32x4 a, u32x4 b, f32x16_t c) {
  if constexpr (kBf16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lk_bf16x8, a), __builtin_bit_cast(lk_bf16x8, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lk_f16x8, a), __builtin_bit_cast(lk_f16x8, b), c, 0,
                                                  0, 0);
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{lo, hi}, f16x2_t));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
  if constexpr (kBf16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{lo, hi}, bf16x2_t));
  return pack_f16(lo, hi);
}

__device__ __forceinline__ float max_of_halves(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum_of_halves(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// A value that is the same in all lanes, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Reference of a query row that has seen nothing: below every logit, and a number, so that
// no difference of references is a NaN.
constexpr float kNone = -3.402823466e38f;

// 32 rows that a wavefront holds as S^T and O^T lie (row lane % 32, value(db, q): dims 32 db
// + 8 q + 4 (lane / 32) + [0, 4)) to their places in out, at(row) or -1: through LDS, since
// their eight-byte pieces in 32 rows at a time kept the next item waiting for 8 us.
template <int kD>
constexpr int kRowsLds = 32 * (2 * kD + 16);

template <int kD, bool kBf16, typename Value, typename At>
__device__ __forceinline__ void store_rows(uint8_t *lds, uint16_t *out, Value value, At at) {
  constexpr int kPitch = 2 * kD + 16, kPerRow = kD / 8;  // 16-byte pieces of a row
  const int lane = threadIdx.x & 63, n = lane & 31, hf = lane >> 5;
#pragma unroll
  for (int db = 0; db < kD / 32; ++db)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4_t v = value(db, q);
      *reinterpret_cast<u32x2 *>(lds + n * kPitch + 64 * db + 16 * q + 8 * hf) =
          u32x2{pack_out<kBf16>(v[0], v[1]), pack_out<kBf16>(v[2], v[3])};
    }
  __builtin_amdgcn_wave_barrier();
#pragma unroll 4
  for (int i = 0; i < 32; i += kWave / kPerRow) {
    const int row = i + lane / kPerRow, piece = lane % kPerRow;
    const u32x4 v = *reinterpret_cast<const u32x4 *>(lds + row * kPitch + 16 * piece);
    const int64_t to = at(row);
    if (to >= 0) *reinterpret_cast<u32x4_a2 *>(out + to + 8 * piece) = v;
  }
}

// Bound by three things that overlap in part: 16 query and 4 KV heads of 256, 8192 rows within
// 2048, take 275 to 300 us (0.85 PFLOP/s).  The matrix cores are busy 41 % of that (2.06 GHz
// under this load), the vector units 33 %, and LDS is at its peak while all four SIMDs
// multiply, since a wavefront reads a whole image for its 32 rows.  64 rows a wavefront (half
// the reads, one wavefront a SIMD, the softmax beside the products of the image before)
// took 510 us a call against 340, 390 if O^T had never to be scaled.
template <int kD, bool kBf16, typename BtT>
__global__ __launch_bounds__(64 * waves_of(kD), waves_of(kD) * groups_per_cu(kD) / 4) void window_attention_kernel(const WindowParams p) {
  constexpr int kQS = kD / 16;   // MFMA steps over the head dims
  constexpr int kDB = kD / 32;   // 32-dim blocks of O^T
  constexpr int kImg = img_bytes(kD);
  constexpr int kCopies = kImg / 1024;
  constexpr int kAheadK = 2, kAheadV = 2;
  // Fp16 outputs round no further than P does: what that leaves of P is multiplied too (error
  // against float64 2.1e-4 in place of 3.0e-4; 2 x 4096 rows within 2048, 16 / 8 heads of 64, 161
  // -> 182 us, 2 x 1024 rows of 16 / 4 heads of 256 131 -> 147).
  constexpr bool kRest = !kBf16;
  constexpr int kWaves = waves_of(kD), kRows = rows_of(kD);
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];  // kStages images

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, hf = lane >> 5;
  if (p.zero_rest) {  // rows of the query outside the only request
    int begin, count;
    request_rows(p.r, 0, begin, count);
    const int words = p.r.hq * (kD / 2);
    const int64_t all = int64_t(p.r.total_q - min(count, p.r.total_q)) * words;
    for (int64_t i = int64_t(blockIdx.x) * 64 * kWaves + tid; i < all; i += int64_t(gridDim.x) * 64 * kWaves) {
      const int row = int(i / words);
      static_cast<u32_a2 *>(p.r.out)[i + (row < begin ? 0 : int64_t(count) * words)] = 0;
    }
  }
  // Neighbouring runs see nearly the same images: they are one XCD's.
  const int per_xcd = p.workers / 8, worker = (int(blockIdx.x) & 7) * per_xcd + (int(blockIdx.x) >> 3);
  const int items = uniform(*p.plan_items), images = uniform(p.plan[items]);
  const int workers = min(p.workers, images);  // an image each at least
  if (worker >= workers) return;               // uniform
  int cur = run_begin(images, worker, workers);
  const int run_end = run_begin(images, worker + 1, workers);
  int item = uniform(p.plan_first[worker]);
  const uint32_t lds0 = lds_address(smem);

  for (; cur < run_end; ++item) {
  // This segment: the run's images of one item.
  const int item_first = uniform(p.plan[item]), item_end = uniform(p.plan[item + 1]);
  const int4 it = p.items[2 * item], of = p.items[2 * item + 1];
  if (item_end <= cur) continue;  // an item without images (uniform)
  const int seen = item_end - item_first - kStart;
  const int t_begin = cur - item_first, t_end = min(min(run_end, item_end) - item_first, seen);
  cur = min(run_end, item_end);
  if (t_begin >= t_end) continue;  // uniform
  const bool whole = t_begin == 0 && t_end == seen;
  const int part = 2 * worker + (cur >= run_end ? 1 : 0);
  const int b = uniform(it.x), slot = uniform(it.y), h = uniform(it.z), tok0 = uniform(it.w);
  const int begin = uniform(of.x), count = uniform(of.y), len = uniform(of.z);
  const WindowRows win = window_rows(p.r, len, count);
  const Walk walk = walk_of(p, len, count, win, tok0);
  const int first_at = len - count;
  const int tok_end = min(tok0 + p.tokens, count);

  // This lane's query row, column n of the wavefront's 32: whether there is one, its token
  // and where it lies in query and output.  Worked out where it is needed: held over the
  // loop it costs registers.
  struct Row {
    bool ok;
    int tok;
    size_t at;
  };
  auto row_of = [&]() {
    int row = wave * 32 + n;
    asm volatile("" : "+v"(row));
    const int in_tile = int(__umulhi(2u * uint32_t(row), p.r.group_magic)), tok = tok0 + in_tile;
    const bool ok = tok < tok_end;
    return Row{ok, tok, (size_t(begin + (ok ? tok : 0)) * p.r.hq + h * p.r.group + (ok ? row - in_tile * p.r.group : 0)) * kD};
  };
  const Row mine = row_of();
  const int at = mine.ok ? first_at + mine.tok : -1;  // its position
  // Positions of the wavefront's rows (it may have none).
  const int at_lo = first_at + tok0 + int(__umulhi(2u * uint32_t(wave * 32), p.r.group_magic));
  const int at_hi = min(first_at + tok0 + int(__umulhi(2u * uint32_t(wave * 32 + 31), p.r.group_magic)), first_at + tok_end - 1);

  const uint8_t *img = p.img + (size_t(slot) * p.r.hkv + h) * p.tiles * kImg;
  auto copy = [&](int i, int stage) {
    const uint8_t *src = img + size_t(walk.image(i)) * kImg;
    for (int j = wave; j < kCopies; j += kWaves)
      dma16_offset(src + 1024 * j, uint32_t(16 * lane), lds0 + uint32_t(stage) * kImg + 1024u * j);
  };
  u32x4 qf[kQS];  // lane: dims 16 i + 8 hf + [0, 8) of row n
  {
    const uint16_t *q = static_cast<const uint16_t *>(p.r.query) + mine.at + 8 * hf;
#pragma unroll
    for (int i = 0; i < kQS; ++i) qf[i] = *reinterpret_cast<const u32x4_a2 *>(q + 16 * i);
  }
  lds_barrier();  // the segment before is done with both stages
  copy(t_begin, 0);
  if (t_begin + 1 < t_end) copy(t_begin + 1, 1);

  f32x16_t oacc[kDB];
#pragma unroll
  for (int db = 0; db < kDB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) oacc[db][e] = 0.f;
  // P's reference r and the sum of weights l, in units of 2^r.  Both are of what this query
  // row sees: scales that it does not see would take its P below fp16's range.  Where some of
  // the images' scales lie far from one, l is in units of 2^m, m the largest logit, so that
  // neither it nor P leaves float32's range (two loops: one for both took 5 % longer).
  float r = kNone, m = kNone, l = 0.f;
  uint32_t odd_seen = 0;
  // The query rows have arrived: without this the loop would wait for them, and with them
  // for the copies behind them, at every image.
#pragma unroll
  for (int k = 0; k < kQS; ++k) asm volatile("" : "+v"(qf[k]));

  auto images_of = [&](auto apart) __attribute__((always_inline)) {
    constexpr bool kApart = decltype(apart)::value;
    for (int i = t_begin; i < t_end; ++i) {
      const int stage = (i - t_begin) % kStages;
      if (stage % 2 == 0) {
        wait_vmcnt<0>();  // this wavefront's part of images i and i + 1
        lds_barrier();    // every wavefront's; and all are done with the other two stages
        if (i + 2 < t_end) copy(i + 2, stage ^ 2);
        if (i + 3 < t_end) copy(i + 3, (stage ^ 2) + 1);
      }
      if (at_lo > at_hi) continue;  // a wavefront without rows (uniform)
      const uint8_t *im = smem + stage * kImg;
      const u32x4 *kf = reinterpret_cast<const u32x4 *>(im) + lane;
      const u32x4 *vf = reinterpret_cast<const u32x4 *>(im + frag_bytes(kD) / 2) + lane;
      const float *sc = reinterpret_cast<const float *>(im + frag_bytes(kD));
      const uint32_t there = __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint32_t *>(sc)[2 * kKeys]);
      odd_seen |= __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint32_t *>(sc)[2 * kKeys + 1]);
      const float room = __int_as_float(uniform(reinterpret_cast<const int *>(sc)[2 * kKeys + 2]));
      const int even = uniform(reinterpret_cast<const int *>(sc)[2 * kKeys + 3]);
      // S^T: element e is key 8 (e / 4) + 4 hf + e % 4 of row n.
      f32x16_t s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.f;
      // A ring of fragments: each is read kAhead products (32 cycles apiece) before its own,
      // which is about what LDS takes; further ahead they would spill.
      u32x4 ka[kAheadK + 1];
#pragma unroll
      for (int k = 0; k < kAheadK; ++k) ka[k] = kf[64 * k];
#pragma unroll
      for (int k = 0; k < kQS; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        if (k + kAheadK < kQS) ka[(k + kAheadK) % (kAheadK + 1)] = kf[64 * (k + kAheadK)];
        s = mfma32<kBf16>(ka[k % (kAheadK + 1)], qf[k], s);
      }
      f32x4_t ks[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) ks[q] = *reinterpret_cast<const f32x4_t *>(sc + 8 * q + 4 * hf);
      __builtin_amdgcn_sched_barrier(0);
      // Cache rows of the image's two groups of 16.
      const int t0 = walk.image(i) * kKeys, r0 = win.real(t0), r1 = win.real(t0 + 16);
      const bool full = there == 0xFFFFFFFFu && r1 + 15 <= at_lo &&
                        (int64_t(min(r0, r1)) > int64_t(at_hi) - p.r.window || r1 + 15 < p.r.sinks);
      float x[16];
      float tmax = -__builtin_inff();
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = s[e] * ks[e >> 2][e & 3];
      if (!full) {
        // Bit k: row k of the image is there and this lane's query row sees it.
        auto below = [](int64_t end) { return (1u << min(max(end, int64_t(0)), int64_t(16))) - 1u; };
        auto seen16 = [&](int r) {
          return below(int64_t(at) + 1 - r) & (~below(int64_t(at) + 1 - p.r.window - r) | below(int64_t(p.r.sinks) - r));
        };
        const uint32_t seen = ((seen16(r0) | (seen16(r1) << 16)) & there) >> (4 * hf);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = (seen >> (8 * (e >> 2) + (e & 3))) & 1u ? x[e] : -__builtin_inff();
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) tmax = fmaxf(tmax, x[e]);
      tmax = max_of_halves(tmax);
      if (kApart || __any(tmax > r + room)) {
        // Every row whose P has outgrown 2^kTop moves (rows that moved alone came to move O^T
        // again and again: 8192 rows within 2048 took 2 % longer).
        float ty;  // of logit + log2 of V's scale, rounded up
        if (!kApart && even) {
          ty = tmax + (kMost - room);
        } else {
          ty = -__builtin_inff();
          int own = kKeys;  // opaque: loads shared with those below would be held across
          asm volatile("" : "+v"(own));
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4_t vsc = *reinterpret_cast<const f32x4_t *>(sc + own + 8 * q + 4 * hf);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (vsc[j] != 0.f) ty = fmaxf(ty, x[4 * q + j] + float(__builtin_amdgcn_frexp_expf(vsc[j])));
          }
          ty = max_of_halves(ty);
        }
        float r_new = fmaxf(r, ty - kTop);
        if constexpr (kApart) {
          const float m_new = fmaxf(m, tmax);
          r_new = fmaxf(r_new, m_new - 126.f);
          l *= __builtin_amdgcn_exp2f(m - m_new);
          m = m_new;
        }
        if (!__all(r == r_new || r == kNone)) {
          const float alpha = __builtin_amdgcn_exp2f(r - r_new);
          if constexpr (!kApart) l *= alpha;
#pragma unroll
          for (int db = 0; db < kDB; ++db) oacc[db] *= alpha;
        }
        r = r_new;
      }
      const float ref = kApart ? m : r;
      u32x4 pf[2], pr[2];
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4_t vsc = *reinterpret_cast<const f32x4_t *>(sc + kKeys + 8 * q + 4 * hf);
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float pw = __builtin_amdgcn_exp2f(x[4 * q + j] - ref);
          sum += pw;
          w[j] = pw * vsc[j];
          if constexpr (kApart) w[j] *= __builtin_amdgcn_exp2f(m - r);
        }
        pf[q >> 1][2 * (q & 1)] = pack_f16(w[0], w[1]);
        pf[q >> 1][2 * (q & 1) + 1] = pack_f16(w[2], w[3]);
        if constexpr (kRest) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const f16x2_t high = __builtin_bit_cast(f16x2_t, uint32_t(pf[q >> 1][2 * (q & 1) + j]));
            pr[q >> 1][2 * (q & 1) + j] = pack_f16(w[2 * j] - float(high[0]), w[2 * j + 1] - float(high[1]));  // exact
          }
        }
      }
      l += sum;
      u32x4 va[kAheadV + 1];
#pragma unroll
      for (int k = 0; k < kAheadV; ++k) va[k] = vf[64 * k];
#pragma unroll
      for (int k = 0; k < 2 * kDB; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        if (k + kAheadV < 2 * kDB) va[(k + kAheadV) % (kAheadV + 1)] = vf[64 * (k + kAheadV)];
        oacc[k >> 1] = mfma32<false>(va[k % (kAheadV + 1)], pf[k & 1], oacc[k >> 1]);
        if constexpr (kRest) oacc[k >> 1] = mfma32<false>(va[k % (kAheadV + 1)], pr[k & 1], oacc[k >> 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  bool apart = false;
  for (int i = t_begin + lane; i < t_end; i += kWave)
    apart |= reinterpret_cast<const float *>(img + size_t(walk.image(i)) * kImg + frag_bytes(kD))[2 * kKeys + 2] ==
             -__builtin_inff();
  apart = __any(apart);  // of the whole workgroup: the images are the same
  float inv;
  if (apart) {
    images_of(std::true_type{});
    l = sum_of_halves(l);
    inv = l != 0.f ? 1.f / l : 0.f;
    const float back = __builtin_amdgcn_exp2f(r - m);
#pragma unroll
    for (int db = 0; db < kDB; ++db) oacc[db] = oacc[db] * inv * back;  // in this order it stays in range
    inv = 1.f;
  } else {
    images_of(std::false_type{});
    l = sum_of_halves(l);
    inv = l != 0.f ? 1.f / l : 0.f;
  }
  if (odd_seen) {
    // Infinities and NaN of V lie as zeros in the images: the rows that see them get them
    // here.  (In the loop above this would hold a second copy of O.)
#pragma unroll 1
    for (int i = t_begin; i < t_end; ++i) {
      const int t0 = walk.image(i) * kKeys, r0 = win.real(t0), r1 = win.real(t0 + 16);
      uint32_t left = __builtin_amdgcn_readfirstlane(
          reinterpret_cast<const uint32_t *>(img + size_t(walk.image(i)) * kImg + frag_bytes(kD))[2 * kKeys + 1]);
#pragma unroll 1
      for (; left; left &= left - 1) {
        const int key = __builtin_ctz(left);
        const int real = (key < 16 ? r0 : r1 - 16) + key, col = real / p.r.block_size;
        const int64_t blk = int64_t((static_cast<const BtT *>(p.r.block_table) + size_t(b) * p.r.bt_stride)[col]);
        const uint8_t *vr = p.r.value_cache + ((blk * p.r.block_size + (real - col * p.r.block_size)) * p.r.hkv + h) * (kD + 4);
        const float vsc = *reinterpret_cast<const float *>(vr + kD);
        const bool vis = window_sees(p.r, at, real);
#pragma unroll
        for (int db = 0; db < kDB; ++db)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(vr + 32 * db + 8 * q + 4 * hf);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              // A finite code counts as one, zero or minus one: beside a scale that is not finite that is enough.
              const uint32_t c = (w >> (8 * j)) & 0xFFu, c7 = c & 0x7Fu;
              const float size = c == 0x80u ? __builtin_nanf("") : c7 == 0x6Fu ? __builtin_inff() : c7 ? 1.f : 0.f;
              const float v = (c & 0x80u ? -size : size) * vsc;
              if (vis && !(fabsf(v) < __builtin_inff())) oacc[db][4 * q + j] += v;
            }
          }
      }
    }
  }
  auto answer = [&](int db, int q) {
    return f32x4_t{oacc[db][4 * q] * inv, oacc[db][4 * q + 1] * inv, oacc[db][4 * q + 2] * inv, oacc[db][4 * q + 3] * inv};
  };
  lds_barrier();  // every wavefront is done with the images: their place takes the rows
  if (whole) {
    if (at_lo <= at_hi)
      store_rows<kD, kBf16>(smem + wave * kRowsLds<kD>, static_cast<uint16_t *>(p.r.out), answer, [&](int i) {
        const int row = wave * 32 + i, in_tile = int(__umulhi(2u * uint32_t(row), p.r.group_magic)), tok = tok0 + in_tile;
        return tok < tok_end ? (int64_t(begin + tok) * p.r.hq + h * p.r.group + (row - in_tile * p.r.group)) * kD : int64_t(-1);
      });
  } else {
    // As the registers hold it: 1 KiB for each of the wavefront's quads of dims.
    const size_t rows = size_t(part) * kRows + wave * 32;
    if (hf == 0) {
      // l in [1/2, 1): r may lie far below or above the logits.
      const int e = __builtin_amdgcn_frexp_expf(l);
      p.part_ml[2 * (rows + n)] = (apart ? m : r) + float(e);
      p.part_ml[2 * (rows + n) + 1] = __builtin_amdgcn_ldexpf(l, -e);
    }
    f32x4_t *o = reinterpret_cast<f32x4_t *>(p.part_o + rows * kD) + lane;
#pragma unroll
    for (int db = 0; db < kDB; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q) o[64 * (4 * db + q)] = answer(db, q);
  }
  }
}

// Joins the parts of items that lie in several runs: M = max m_s, out = sum_s 2^(m_s - M)
// l_s o_s / sum_s 2^(m_s - M) l_s, o_s a part's own attention.  Per run a workgroup for
// every 32 rows takes the item that reaches into it from the one before, if that is
// where it begins; a wavefront takes a quarter of the dims.  The workgroups behind them
// give the rows of items without images their zeros.  Bound by the parts' bytes: 130 MB of
// FP32 for 8192 rows of 16 heads of 256, 40 us (22 for 4 x 512).
template <int kD, bool kBf16>
__global__ __launch_bounds__(kThreads) void window_join_kernel(const WindowParams p) {
  constexpr int kQuads = kD / 32;  // quads of dims of a wavefront
  constexpr int kRows = rows_of(kD), kBlocks = kRows / 32;
  __shared__ __attribute__((aligned(16))) uint8_t rows_lds[kRowsLds<kD>];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, hf = lane >> 5;
  const int items = *p.plan_items, images = p.plan[items], workers = min(p.workers, images);
  if (int(blockIdx.x) >= p.workers * kBlocks) {
    const int i0 = (int(blockIdx.x) - p.workers * kBlocks) * kThreads;
    for (int item = i0; item < min(i0 + kThreads, items); ++item) {
      if (p.plan[item + 1] > p.plan[item]) continue;
      const int4 it = p.items[2 * item];
      const int begin = p.items[2 * item + 1].x, count = p.items[2 * item + 1].y;
      const int words = p.r.group * (kD / 2), rows = min(p.tokens, count - it.w);
      for (int i = tid; i < rows * words; i += kThreads)
        static_cast<u32_a2 *>(p.r.out)[(size_t(begin + it.w + i / words) * p.r.hq + it.z * p.r.group) * (kD / 2) + i % words] = 0;
    }
    return;
  }
  const int w = int(blockIdx.x) / kBlocks, block = int(blockIdx.x) % kBlocks;
  if (w == 0 || w >= workers) return;  // uniform, as what follows
  const int at = run_begin(images, w, workers), item = p.plan_first[w];
  const int lo = p.plan[item], hi = p.plan[item + 1] - kStart;
  if (lo == at || hi <= at || run_begin(images, w - 1, workers) > lo) return;
  const int w0 = w - 1, w1 = int((int64_t(hi) * workers - 1) / images);
  const bool ends = run_begin(images, w1 + 1, workers) <= hi + kStart;  // else w1's run goes on with other items
  const int4 it = p.items[2 * item];
  const int begin = p.items[2 * item + 1].x, count = p.items[2 * item + 1].y;
  auto rows_of_part = [&](int s) { return size_t(2 * s + (s < w1 || ends ? 1 : 0)) * kRows + block * 32; };
  float m = kNone;
  for (int s = w0; s <= w1; ++s) m = fmaxf(m, p.part_ml[2 * (rows_of_part(s) + n)]);
  float total = 0.f;
  f32x4_t acc[kQuads];
#pragma unroll
  for (int k = 0; k < kQuads; ++k) acc[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int s0 = w0; s0 <= w1; s0 += 2) {
    float f[2];
    f32x4_t v[2][kQuads];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int s = min(s0 + i, w1);
      const f32x4_t *o = reinterpret_cast<const f32x4_t *>(p.part_o + rows_of_part(s) * kD) + 64 * kQuads * wave + lane;
#pragma unroll
      for (int k = 0; k < kQuads; ++k) v[i][k] = o[64 * k];
      const float ms = p.part_ml[2 * (rows_of_part(s) + n)], ls = p.part_ml[2 * (rows_of_part(s) + n) + 1];
      // A part that saw nothing has l = 0; one with a NaN logit l = NaN, whatever its maximum.
      f[i] = s0 + i <= w1 && ls != 0.f ? __builtin_amdgcn_exp2f(ms - m) * ls : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      total += f[i];
#pragma unroll
      for (int k = 0; k < kQuads; ++k) acc[k] += f[i] != 0.f ? f[i] * v[i][k] : f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  const float inv = total != 0.f ? 1.f / total : 0.f;
#pragma unroll
  for (int k = 0; k < kQuads; ++k) {
    const int quad = kQuads * wave + k;  // dims 8 quad + 4 hf + [0, 4)
    *reinterpret_cast<u32x2 *>(rows_lds + n * (2 * kD + 16) + 16 * quad + 8 * hf) =
        u32x2{pack_out<kBf16>(acc[k][0] * inv, acc[k][1] * inv), pack_out<kBf16>(acc[k][2] * inv, acc[k][3] * inv)};
  }
  __syncthreads();
  for (int i = tid; i < 32 * (kD / 8); i += kThreads) {
    const int in = i / (kD / 8), piece = i % (kD / 8), row = block * 32 + in;
    const int in_tile = int(__umulhi(2u * uint32_t(row), p.r.group_magic)), tok = it.w + in_tile;
    if (in_tile < p.tokens && tok < count)
      *reinterpret_cast<u32x4_a2 *>(static_cast<uint16_t *>(p.r.out) +
                                    (size_t(begin + tok) * p.r.hq + it.z * p.r.group + (row - in_tile * p.r.group)) * kD + 8 * piece) =
          *reinterpret_cast<const u32x4 *>(rows_lds + in * (2 * kD + 16) + 16 * piece);
  }
}

// ------------------------------------------------------------- host side

// Requests of more (token, head) rows per KV head than this run on images: kOnlyRows for a
// call's only request, which cannot fill the GPU with its images' items, kLongRows for one of
// several.  Images against the other kernels, us, 8 KV heads of 128, groups of 4, 16-row pages
// (the one shape that both were measured at):
//   requests, window   256 rows     384        512        768
//   1 of 1024          60 vs 27   61 vs 26   49 vs 30   50 vs 40
//   1 of 4096          64 vs 35   69 vs 41   60 vs 46   63 vs 69
//   4 of 4096          70 vs 64   78 vs 92   85 vs 105  107 vs 198
//   8 of 1024          62 vs 46              77 vs 104
//   16 of 256          63 vs 53   70 vs 94   87 vs 120  111 vs 235
//   32 of 1024        182 vs 168            238 vs 356
constexpr int64_t kLongRows = 256, kOnlyRows = 512;
// Image bytes of a pass; requests that do not fit wait for the next one.
constexpr int64_t kImageBytes = int64_t(512) << 20;

struct WindowPlan {
  int64_t long_rows;   // 0: the only request, whatever its length
  int64_t requests;    // that can be long
  int64_t slots, tiles, tokens, items, workers;
  bool others;         // short requests may be among them
  size_t images, parts_o, parts_ml, plan, rows;  // bytes
  size_t total() const { return std::max(rows, images + parts_o + parts_ml + plan); }
};

// Up to 256 query heads per KV head: an item holds a token's at least, and so does kLongRows.
// 2 x 1024 rows within 2048 under 64 heads of 128 and one KV head take 221 us so and 4890 on
// the kernels of few rows, under 128 heads 376 and 9770.
bool image_shape(int64_t d, int64_t dv, int64_t group, int64_t block_size) {
  return (d == 64 || d == 128 || d == 256) && dv == d && block_size % 16 == 0 && group <= 256;
}
static_assert(rows_of(64) >= 256 && rows_of(128) >= 256 && rows_of(256) >= 256);

WindowPlan plan_window(int64_t batch, int64_t heads, int64_t hkv, int64_t d, int64_t dv, int64_t block_size,
                       int64_t total_q, int64_t max_query, int64_t max_len, int64_t window, int64_t sinks) {
  WindowPlan pl{};
  const int64_t group = heads / hkv;
  pl.others = true;
  int64_t row_queries = max_query;
  if (image_shape(d, dv, group, block_size) && max_query * group > (batch > 1 ? kLongRows : kOnlyRows) && max_len > 0) {
    pl.long_rows = batch > 1 ? kLongRows : 0;
    pl.others = batch > 1;
    pl.requests = std::min(batch, batch > 1 ? total_q / (kLongRows / group + 1) : int64_t(1));
    row_queries = kLongRows / group;
  }
  if (pl.requests > 0) {
    const int64_t seen = rows_bound(max_len, max_query, window, sinks);
    pl.tiles = (seen + kKeys - 1) / kKeys;
    const int64_t per_slot = hkv * pl.tiles * img_bytes(int(d));
    pl.slots = std::max<int64_t>(1, std::min({pl.requests, kImageBytes / per_slot, int64_t(kMaxSlots)}));
    pl.tokens = rows_of(int(d)) / group;
    // At most: every request's rows in whole items.
    pl.items = hkv * (pl.slots * std::min((max_query + pl.tokens - 1) / pl.tokens, total_q / pl.tokens + 1));
    if (batch > 1) pl.items = std::min(pl.items, hkv * (total_q / pl.tokens + pl.slots));
    pl.workers = 256 * groups_per_cu(int(d));
    pl.images = size_t(pl.slots) * per_slot;
    pl.parts_o = size_t(2 * pl.workers) * rows_of(int(d)) * d * sizeof(float);
    pl.parts_ml = size_t(2 * pl.workers) * rows_of(int(d)) * 2 * sizeof(float);
    pl.plan = size_t(pl.items) * 2 * sizeof(int4) + size_t(pl.items + 2 + pl.workers) * sizeof(int32_t);
  }
  if (pl.others)
    pl.rows = row_workspace(batch, total_q, heads, hkv, d, dv, block_size, row_queries,
                            rows_bound(max_len, row_queries, window, sinks), false);
  return pl;
}

template <int kD, bool kBf16, typename BtT>
int launch_images(const char *name, WindowParams p, const WindowPlan &pl, hipStream_t s) {
  constexpr int kTiles = kThreads / kD;
  // The images, and the rows in their place.
  constexpr size_t kSmem = std::max(kStages * size_t(img_bytes(kD)), size_t(waves_of(kD)) * kRowsLds<kD>);
  if (const int st = reserve_dynamic_lds(reinterpret_cast<const void *>(&window_attention_kernel<kD, kBf16, BtT>), kSmem,
                                         name))
    return st;
  const int64_t groups = int64_t(p.slots) * ((p.tiles + kTiles - 1) / kTiles);
  for (p.first_slot = 0; p.first_slot < pl.requests; p.first_slot += p.slots) {
    window_image_kernel<kD, kBf16, BtT><<<unsigned((groups + 7) / 8 * 8 * p.r.hkv + 8), kThreads, 0, s>>>(p);
    window_attention_kernel<kD, kBf16, BtT><<<unsigned(p.workers), 64 * waves_of(kD), kSmem, s>>>(p);
    window_join_kernel<kD, kBf16>
        <<<unsigned(p.workers * (rows_of(kD) / 32) + (pl.items + kThreads - 1) / kThreads), kThreads, 0, s>>>(p);
    if (const int st = check_launch(name)) return st;
  }
  return HIF8_OK;
}

template <bool kBf16, typename BtT>
int launch_images_of(const char *name, const WindowParams &p, const WindowPlan &pl, hipStream_t s) {
  if (p.r.d == 64) return launch_images<64, kBf16, BtT>(name, p, pl, s);
  if (p.r.d == 128) return launch_images<128, kBf16, BtT>(name, p, pl, s);
  return launch_images<256, kBf16, BtT>(name, p, pl, s);
}

}  // namespace
}  // namespace hif8

using namespace hif8;

extern "C" size_t hif8_window_attention_workspace_size(int64_t batch, int64_t num_heads, int64_t num_kv_heads,
                                                       int64_t head_size, int64_t head_size_v, int64_t block_size,
                                                       int64_t total_query_tokens, int64_t max_query_len,
                                                       int64_t max_seq_len, int64_t window, int64_t sinks) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_size <= 0 || head_size_v <= 0 || block_size <= 0 ||
      total_query_tokens <= 0 || max_query_len <= 0 || max_seq_len < 0 || window <= 0 || sinks < 0 ||
      num_heads % num_kv_heads)
    return 0;
  window = std::min<int64_t>(window, 0x7FFFFFFF), sinks = std::min<int64_t>(sinks, 0x7FFFFFFF);
  return plan_window(batch, num_heads, num_kv_heads, head_size, head_size_v, block_size, total_query_tokens,
                     max_query_len, max_seq_len, window, sinks)
      .total();
}

extern "C" int hif8_window_attention(const void *query, int q_dtype, const uint8_t *key_cache,
                                     const uint8_t *value_cache, int64_t num_blocks, int64_t block_size,
                                     int64_t num_kv_heads, int64_t head_size, int64_t head_size_v,
                                     const void *block_table, int block_table_dtype, int64_t max_blocks_per_seq,
                                     const int32_t *query_start_loc, const int32_t *seq_lens, int64_t batch,
                                     int64_t num_heads, int64_t total_query_tokens, int64_t max_query_len,
                                     int64_t max_seq_len, int64_t window, int64_t sinks, float scale, void *out,
                                     void *workspace, size_t workspace_bytes, hif8_stream_t stream) {
  static const char *kName = "hif8_window_attention";
  clear_error();
  if (window <= 0 || sinks < 0)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: window must be positive and sinks not negative", kName);
  if (max_query_len < 0) return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions must be positive", kName);
  if (batch > 0 && total_query_tokens > 0) {
    if (max_query_len == 0)
      return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: max_query_len must cover the query rows", kName);
    if (!query_start_loc && (max_query_len != 1 || total_query_tokens != batch))
      return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: without query_start_loc every request has one query row", kName);
    if (max_query_len > 0x7FFFFFFF)
      return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", kName);
  }
  // Past the lengths' range a window or a count of first rows means the same.
  window = std::min<int64_t>(window, 0x7FFFFFFF), sinks = std::min<int64_t>(sinks, 0x7FFFFFFF);
  const RowArgs a{query, q_dtype, key_cache, value_cache, num_blocks, block_size, num_kv_heads, head_size, head_size_v,
                  block_table, block_table_dtype, max_blocks_per_seq, query_start_loc, seq_lens, nullptr, 0, batch,
                  num_heads, total_query_tokens, max_query_len, max_seq_len, scale, out, nullptr, 0, 0, 1, workspace,
                  workspace_bytes, stream, window, sinks, 0};
  if (const int st = check_row_args(kName, a)) return st;
  if (batch == 0 || total_query_tokens == 0) return HIF8_OK;
  const size_t need = hif8_window_attention_workspace_size(batch, num_heads, num_kv_heads, head_size, head_size_v,
                                                           block_size, total_query_tokens, max_query_len, max_seq_len,
                                                           window, sinks);
  if (!workspace || workspace_bytes < need)
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes required (got %zu)", kName, need,
                workspace_bytes);
  const WindowPlan pl = plan_window(batch, num_heads, num_kv_heads, head_size, head_size_v, block_size,
                                    total_query_tokens, max_query_len, max_seq_len, window, sinks);
  if (pl.requests == 0) return row_attention(kName, a);
  if (!aligned(workspace, 16))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned", kName);
  if (pl.items > 0x1FFFFF || pl.items * (pl.tiles + kStart) > 0x7FFFFFFF || pl.slots * num_kv_heads * (pl.tiles + 8) > 0xFFFFFF)  // threads of a launch
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: dimensions too large", kName);
  const int64_t group = num_heads / num_kv_heads;
  if (pl.others) {
    RowArgs few = a;
    few.max_query = kLongRows / group;
    few.long_rows = kLongRows;
    if (const int st = row_attention(kName, few)) return st;
  }
  WindowParams p{};
  p.r.query = query;
  p.r.key_cache = key_cache;
  p.r.value_cache = value_cache;
  p.r.block_table = block_table;
  p.r.start_loc = query_start_loc;
  p.r.lens = seq_lens;
  p.r.out = out;
  p.r.bt_stride = max_blocks_per_seq;
  p.r.num_blocks = num_blocks;
  p.r.block_size = int(block_size);
  p.r.hkv = int(num_kv_heads);
  p.r.hq = int(num_heads);
  p.r.group = int(group);
  p.r.group_magic = uint32_t(((int64_t(1) << 31) + group - 1) / group);
  p.r.d = p.r.dv = int(head_size);
  p.r.batch = int(batch);
  p.r.total_q = int(total_query_tokens);
  p.r.max_len = int(max_seq_len);
  p.r.scale_log2 = scale * 1.4426950408889634f;
  p.r.window = int(window);
  p.r.sinks = int(sinks);
  p.r.most_rows = int(rows_bound(max_seq_len, max_query_len, window, sinks));
  p.r.long_rows = int(pl.long_rows);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  p.img = ws;
  p.part_o = reinterpret_cast<float *>(ws + pl.images);
  p.part_ml = reinterpret_cast<float *>(ws + pl.images + pl.parts_o);
  p.tiles = int(pl.tiles);
  p.slots = int(pl.slots);
  p.tokens = int(pl.tokens);
  p.items = reinterpret_cast<int4 *>(ws + pl.images + pl.parts_o + pl.parts_ml);
  p.plan = reinterpret_cast<int32_t *>(p.items + 2 * pl.items);
  p.plan_items = p.plan + pl.items + 1;
  p.plan_first = p.plan_items + 1;
  p.most_items = int(pl.items);
  p.workers = int(pl.workers);
  p.zero_rest = pl.others ? 0 : 1;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool i64 = block_table_dtype == HIF8_INDEX_INT64;
  if (q_dtype == HIF8_DTYPE_BF16)
    return i64 ? launch_images_of<true, int64_t>(kName, p, pl, s)
               : launch_images_of<true, int32_t>(kName, p, pl, s);
  return i64 ? launch_images_of<false, int64_t>(kName, p, pl, s)
             : launch_images_of<false, int32_t>(kName, p, pl, s);
}
