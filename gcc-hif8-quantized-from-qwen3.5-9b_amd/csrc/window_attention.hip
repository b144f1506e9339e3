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
//   * window_attention_kernel: a workgroup of four wavefronts owns (request, KV
//     head, 128 (token, head) rows), 32 rows a wavefront, and walks the images of
//     the rows it sees.  Per image S^T = K Q^T and O^T += V^T P^T on
//     v_mfma_f32_32x32x16, a softmax with a running maximum between them.
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
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;  // four wavefronts
constexpr int kRows = 128;     // (token, head) rows of a workgroup, 32 a wavefront
constexpr int kKeys = 32;      // cached rows of an image
constexpr int kMaxSplits = 64;

// An image: K fragments [D / 16], V fragments [D / 32][2], then K's scales (times the
// softmax scale, base 2) [32], V's [32], and two words: rows that are there, rows whose V
// holds an infinity or NaN.
constexpr int frag_bytes(int d) { return 2 * kKeys * d * 2; }
constexpr int img_bytes(int d) { return (frag_bytes(d) + 8 * kKeys + 16 + 1023) / 1024 * 1024; }

struct WindowParams {
  RowAttnParams r;       // request split, lengths, table, caches, window
  uint8_t *img;          // [slots][hkv][tiles]
  float *part_o;         // [slots][hkv][q_tiles][splits][kRows][D]
  float *part_ml;        // [slots][hkv][q_tiles][splits][kRows][2]
  int tiles;             // images per (slot, KV head)
  int slots, first_slot; // requests of this pass; slot s holds the (first_slot + s)-th long request
  int tokens, q_tiles, splits;  // tokens of a workgroup, workgroups of the longest request, parts of its rows
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

// ------------------------------------------------------------------ images

// A workgroup per (slot, KV head, kThreads / D * 32 rows): threads take 16 codes of a K
// row, and 4 codes of eight V rows each.  Bound by the bytes (4 of image and 1 of cache
// per element).  The KV heads of one tile, whose rows share cache lines, have block ids
// equal modulo 8: one XCD.
template <int kD, bool kBf16, typename BtT>
__global__ __launch_bounds__(kThreads) void window_image_kernel(const WindowParams p) {
  constexpr int kTiles = kThreads / kD;         // images of a workgroup
  constexpr int kChunks = kD / 16;              // 16-code chunks of a row
  constexpr int kPerTile = kThreads / kTiles;   // threads of an image
  constexpr int kLoads = kKeys * kChunks / kPerTile;
  static_assert(kPerTile == kD && kD % 64 == 0, "a wavefront works on one image");
  __shared__ uint32_t dec[256];  // the query's type below, fp16 (0 where not finite) above
  __shared__ uint32_t odd[kTiles];
  const int tid = threadIdx.x;
  const int xcd = int(blockIdx.x) & 7, rest = int(blockIdx.x) >> 3;
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
    if (tid < kTiles) odd[tid] = 0;
  }
  const int tile = first + tid / kPerTile, at = tid % kPerTile;
  const BtT *bt = static_cast<const BtT *>(p.r.block_table) + size_t(b) * p.r.bt_stride;
  const int64_t rec = int64_t(p.r.hkv) * (kD + 4);
  // Offset of this KV head's row `key` of the image, or -1.
  auto offset_of = [&](int key) -> int64_t {
    const int t = tile * kKeys + key;
    if (t >= win.rows) return -1;
    const int real = win.real(t), col = real / p.r.block_size;
    const int64_t blk = int64_t(bt[col]);
    if (blk < 0 || blk >= p.r.num_blocks) return -1;
    return (blk * p.r.block_size + (real - col * p.r.block_size)) * rec + int64_t(h) * (kD + 4);
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
    if (bad) atomicOr(&odd[tid / kPerTile], bad);
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
      if (!finite) atomicOr(&odd[tid / kPerTile], 1u << at);
    }
    const uint64_t seen = __ballot(there);  // the image's first wavefront
    if (at == 0) reinterpret_cast<uint32_t *>(im + frag_bytes(kD))[2 * kKeys] = uint32_t(seen);
  }
  __syncthreads();
  if (mine && at == 0) reinterpret_cast<uint32_t *>(im + frag_bytes(kD))[2 * kKeys + 1] = odd[tid / kPerTile];
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

// Weights are 2^(x - m + kBias - e), m a maximum of the row that moves once a logit passes
// it by kLazy, 2^e the power of two above the largest of V's scales (held within 2^+-96, so
// that sums of weights stay in range): P = weight * V's scale stays below 2^14 and starts
// high in fp16's range, so that small weights keep their bits.
constexpr float kBias = 6.f, kLazy = 8.f;

template <int kD, bool kBf16, typename BtT>
__global__ __launch_bounds__(kThreads, kD == 256 ? 2 : 3) void window_attention_kernel(const WindowParams p) {
  constexpr int kQS = kD / 16;   // MFMA steps over the head dims
  constexpr int kDB = kD / 32;   // 32-dim blocks of O^T
  constexpr int kImg = img_bytes(kD);
  constexpr int kCopies = kImg / 1024;
  constexpr int kAhead = 2;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];  // two images
  __shared__ int top;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, hf = lane >> 5;
  // Neighbouring query tiles of one KV head see nearly the same images: they run on
  // one XCD, one after the other.
  const int items = p.slots * p.r.hkv * p.q_tiles * p.splits;
  const int per_xcd = (items + 7) / 8;
  const int item = (int(blockIdx.x) & 7) * per_xcd + (int(blockIdx.x) >> 3);
  if ((int(blockIdx.x) >> 3) >= per_xcd || item >= items) return;  // padding block (uniform)
  const int split = item % p.splits, qt = (item / p.splits) % p.q_tiles;
  const int sh = item / (p.splits * p.q_tiles);
  const int slot = sh / p.r.hkv, h = sh - slot * p.r.hkv;
  const int b = long_request(p.r, p.first_slot + slot);
  int begin = 0, count = 0;
  if (b >= 0) request_rows(p.r, b, begin, count);
  const int tok0 = qt * p.tokens;
  if (p.zero_rest && split == 0) {  // rows of the query outside the only request
    for (int i = tid; i < p.tokens * p.r.group * (kD / 2); i += kThreads) {
      const int row = tok0 + i / (p.r.group * (kD / 2)), in_row = i % (p.r.group * (kD / 2));
      if (row < p.r.total_q && (row < begin || row - begin >= count))
        reinterpret_cast<uint32_t *>(p.r.out)[(size_t(row) * p.r.hq + h * p.r.group) * (kD / 2) + in_row] = 0;
    }
  }
  if (b < 0 || tok0 >= count) return;  // uniform
  const int len = clamp_rows(p.r.lens[b], p.r.max_len);
  const WindowRows win = window_rows(p.r, len, count);
  const int first_at = len - count;  // position of the request's first query row
  const int tok_end = min(tok0 + p.tokens, count);

  // The images that this workgroup's rows see: those of the first rows, and from the one
  // on in which its first row's window begins.
  const int last_t = min(win.rows, max(0, first_at + tok_end - win.skip));
  const int tiles_end = (last_t + kKeys - 1) / kKeys;
  const int low_t = int(max(int64_t(first_at) + tok0 + 1 - p.r.window, int64_t(win.skip))) - win.skip;
  const int sink_tiles = (min(p.r.sinks, last_t) + kKeys - 1) / kKeys;
  const int near = max(low_t / kKeys, sink_tiles);
  const int total = sink_tiles + max(tiles_end - near, 0);
  const int t_begin = int(int64_t(total) * split / p.splits), t_end = int(int64_t(total) * (split + 1) / p.splits);
  auto image_of = [&](int i) { return i < sink_tiles ? i : i - sink_tiles + near; };

  // This lane's query row: column n of the wavefront's 32.
  const int row = wave * 32 + n;
  const int tok = tok0 + int(__umulhi(2u * uint32_t(row), p.r.group_magic));
  const int in_group = row - (tok - tok0) * p.r.group;
  const bool ok = tok < tok_end;
  const int at = ok ? first_at + tok : -1;
  const int qhead = h * p.r.group + (ok ? in_group : 0);
  const size_t out_row = (size_t(begin + (ok ? tok : 0)) * p.r.hq + qhead) * kD;
  // Positions of the wavefront's rows (it may have none).
  const int at_lo = first_at + tok0 + int(__umulhi(2u * uint32_t(wave * 32), p.r.group_magic));
  const int at_hi = min(first_at + tok0 + int(__umulhi(2u * uint32_t(wave * 32 + 31), p.r.group_magic)), first_at + tok_end - 1);

  const uint8_t *img = p.img + (size_t(slot) * p.r.hkv + h) * p.tiles * kImg;
  const uint32_t lds0 = lds_address(smem);
  auto copy = [&](int i, int stage) {
    const uint8_t *src = img + size_t(image_of(i)) * kImg + 16 * lane;
    for (int j = wave; j < kCopies; j += kThreads / kWave) dma16(src + 1024 * j, lds0 + uint32_t(stage) * kImg + 1024u * j);
  };
  u32x4 qf[kQS];  // lane: dims 16 i + 8 hf + [0, 8) of row n
  {
    const uint16_t *q = static_cast<const uint16_t *>(p.r.query) + out_row + 8 * hf;
#pragma unroll
    for (int i = 0; i < kQS; ++i) qf[i] = *reinterpret_cast<const u32x4 *>(q + 16 * i);
  }
  if (t_begin < t_end) copy(t_begin, 0);
  // The power of two of the largest of V's scales.
  if (tid == 0) top = 0;
  __syncthreads();
  {
    float most = 0.f;
    for (int i = t_begin * kKeys + tid; i < t_end * kKeys; i += kThreads) {
      const uint8_t *im = img + size_t(image_of(i / kKeys)) * kImg + frag_bytes(kD);
      most = fmaxf(most, fabsf(reinterpret_cast<const float *>(im)[kKeys + i % kKeys]));
    }
    atomicMax(&top, int(__float_as_uint(most)));
  }
  __syncthreads();
  const float largest = __uint_as_float(uint32_t(__builtin_amdgcn_readfirstlane(top)));
  const float base = kBias - float(min(max(largest > 0.f ? int(__builtin_amdgcn_frexp_expf(largest)) : 0, -96), 96));

  f32x16_t oacc[kDB];
#pragma unroll
  for (int db = 0; db < kDB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) oacc[db][e] = 0.f;
  float m = -__builtin_inff(), l = 0.f;
  uint32_t odd_seen = 0;

  for (int i = t_begin; i < t_end; ++i) {
    const int stage = (i - t_begin) & 1;
    wait_vmcnt<0>();  // this wavefront's part of image i
    lds_barrier();    // every wavefront's; and all are done with the other stage
    if (i + 1 < t_end) copy(i + 1, stage ^ 1);
    if (at_lo > at_hi) continue;  // a wavefront without rows (uniform)
    const uint8_t *im = smem + stage * kImg;
    const u32x4 *kf = reinterpret_cast<const u32x4 *>(im) + lane;
    const u32x4 *vf = reinterpret_cast<const u32x4 *>(im + frag_bytes(kD) / 2) + lane;
    const float *sc = reinterpret_cast<const float *>(im + frag_bytes(kD));
    const uint32_t there = __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint32_t *>(sc)[2 * kKeys]);
    odd_seen |= __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint32_t *>(sc)[2 * kKeys + 1]);
    // S^T: element e is key 8 (e / 4) + 4 hf + e % 4 of row n.
    f32x16_t s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
    // Fragments are read kAhead steps before their products, no earlier: more would spill.
    u32x4 ka[2][kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) ka[0][k] = kf[64 * k];
#pragma unroll
    for (int k0 = 0; k0 < kQS; k0 += kAhead) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (k0 + kAhead < kQS) ka[(k0 / kAhead + 1) & 1][k] = kf[64 * (k0 + kAhead + k)];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) s = mfma32<kBf16>(ka[(k0 / kAhead) & 1][k], qf[k0 + k], s);
    }
    __builtin_amdgcn_sched_barrier(0);
    // Cache rows of the image's two groups of 16.
    const int t0 = image_of(i) * kKeys, r0 = win.real(t0), r1 = win.real(t0 + 16);
    const bool full = there == 0xFFFFFFFFu && r1 + 15 <= at_lo && (int64_t(min(r0, r1)) > int64_t(at_hi) - p.r.window ||
                                                                   r1 + 15 < p.r.sinks);
    float x[16];
    float tmax = -__builtin_inff();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4_t ks = *reinterpret_cast<const f32x4_t *>(sc + 8 * q + 4 * hf);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * q + j] = s[4 * q + j] * ks[j];
    }
    if (!full) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = 8 * q + 4 * hf + j, real = (q < 2 ? r0 : r1 - 16) + key;
          const bool vis = bool((there >> key) & 1u) & window_sees(p.r, at, real);
          x[4 * q + j] = vis ? x[4 * q + j] : -__builtin_inff();
        }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) tmax = fmaxf(tmax, x[e]);
    tmax = max_of_halves(tmax);
    if (__any(tmax > m + kLazy)) {
      const bool grow = tmax > m + kLazy;  // also the first logit of a row: m is -infinity
      const float m_new = grow ? tmax : m;
      const float alpha = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
      if (!__all(!grow || m == -__builtin_inff())) {
        l *= alpha;
#pragma unroll
        for (int db = 0; db < kDB; ++db) oacc[db] *= alpha;
      }
      m = m_new;
    }
    const float ref = m == -__builtin_inff() ? 0.f : m - base;
    u32x4 pf[2];
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
      }
      pf[q >> 1][2 * (q & 1)] = pack_f16(w[0], w[1]);
      pf[q >> 1][2 * (q & 1) + 1] = pack_f16(w[2], w[3]);
    }
    l += sum;
    u32x4 va[2][2];
    va[0][0] = vf[0], va[0][1] = vf[64];
#pragma unroll
    for (int db = 0; db < kDB; ++db) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int st = 0; st < 2; ++st)
        if (db + 1 < kDB) va[(db + 1) & 1][st] = vf[64 * (2 * db + 2 + st)];
#pragma unroll
      for (int st = 0; st < 2; ++st) oacc[db] = mfma32<false>(va[db & 1][st], pf[st], oacc[db]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if (at_lo > at_hi) return;
  if (odd_seen) {
    // Infinities and NaN of V lie as zeros in the images: the rows that see them get them
    // here.  (In the loop above this would hold a second copy of O.)
#pragma unroll 1
    for (int i = t_begin; i < t_end; ++i) {
      const int t0 = image_of(i) * kKeys, r0 = win.real(t0), r1 = win.real(t0 + 16);
      uint32_t left = __builtin_amdgcn_readfirstlane(
          reinterpret_cast<const uint32_t *>(img + size_t(image_of(i)) * kImg + frag_bytes(kD))[2 * kKeys + 1]);
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
  l = sum_of_halves(l);
  if (!ok) return;
  const float inv = l != 0.f ? 1.f / l : 0.f;
  if (p.splits == 1) {
    uint16_t *o = static_cast<uint16_t *>(p.r.out) + out_row + 4 * hf;
#pragma unroll
    for (int db = 0; db < kDB; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x16_t &a = oacc[db];
        *reinterpret_cast<u32x2 *>(o + 32 * db + 8 * q) =
            u32x2{pack_out<kBf16>(a[4 * q] * inv, a[4 * q + 1] * inv),
                  pack_out<kBf16>(a[4 * q + 2] * inv, a[4 * q + 3] * inv)};
      }
    return;
  }
  const size_t part = size_t(item) * kRows + row;
  if (hf == 0) {
    p.part_ml[2 * part] = m;
    p.part_ml[2 * part + 1] = l;
  }
  if (l == 0.f) return;  // saw nothing: its outputs are not read
  float *o = p.part_o + part * kD + 4 * hf;
#pragma unroll
  for (int db = 0; db < kDB; ++db)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x16_t &a = oacc[db];
      *reinterpret_cast<f32x4_t *>(o + 32 * db + 8 * q) =
          f32x4_t{a[4 * q] * inv, a[4 * q + 1] * inv, a[4 * q + 2] * inv, a[4 * q + 3] * inv};
    }
}

// Joins the parts of every row: M = max m_s, out = sum_s 2^(m_s - M) l_s o_s / sum_s
// 2^(m_s - M) l_s, o_s a part's own attention.  A wavefront per row, four dims a lane.
template <int kD, bool kBf16>
__global__ __launch_bounds__(kThreads) void window_join_kernel(const WindowParams p) {
  const int item = int(blockIdx.x), lane = threadIdx.x & 63;  // (slot, KV head, query tile)
  const int row = int(blockIdx.y) * (kThreads / kWave) + (threadIdx.x >> 6);
  const int qt = item % p.q_tiles, sh = item / p.q_tiles, slot = sh / p.r.hkv, h = sh - slot * p.r.hkv;
  const int b = long_request(p.r, p.first_slot + slot);
  if (b < 0) return;  // uniform
  int begin, count;
  request_rows(p.r, b, begin, count);
  const int in_tile = int(__umulhi(2u * uint32_t(row), p.r.group_magic)), tok = qt * p.tokens + in_tile;
  if (in_tile >= p.tokens || tok >= count) return;  // uniform
  const size_t base = size_t(item) * p.splits * kRows + row;
  const bool have = lane < p.splits;
  const float ms = have ? p.part_ml[2 * (base + size_t(have ? lane : 0) * kRows)] : -__builtin_inff();
  const float ls = have ? p.part_ml[2 * (base + size_t(have ? lane : 0) * kRows) + 1] : 0.f;
  const float mx = wave_max(ms);
  // A part that saw nothing has l = 0; one with a NaN logit l = NaN, whatever its maximum.
  const float w = ls != 0.f ? __builtin_amdgcn_exp2f(ms - (mx == -__builtin_inff() ? 0.f : mx)) * ls : 0.f;
  const float total = wave_sum(w);
  const float inv = total != 0.f ? 1.f / total : 0.f;
  f32x4_t acc{0.f, 0.f, 0.f, 0.f};
  const bool dims = 4 * lane < kD;
  for (int s0 = 0; s0 < p.splits; s0 += 8) {
    float ws[8];
    f32x4_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ws[j] = s0 + j < p.splits ? __shfl(w, s0 + j, kWave) : 0.f;
      v[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (dims && ws[j] != 0.f)
        v[j] = *reinterpret_cast<const f32x4_t *>(p.part_o + (base + size_t(s0 + j) * kRows) * kD + 4 * lane);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) acc += ws[j] * inv * v[j];
  }
  if (!dims) return;
  uint16_t *o = static_cast<uint16_t *>(p.r.out) +
                (size_t(begin + tok) * p.r.hq + h * p.r.group + (row - in_tile * p.r.group)) * kD + 4 * lane;
  *reinterpret_cast<u32x2 *>(o) = u32x2{pack_out<kBf16>(acc[0], acc[1]), pack_out<kBf16>(acc[2], acc[3])};
}

// ------------------------------------------------------------- host side

// Requests of more (token, head) rows per KV head than this run on images.
constexpr int64_t kLongRows = 128;
// Image bytes of a pass; requests that do not fit wait for the next one.
constexpr int64_t kImageBytes = int64_t(512) << 20;

struct WindowPlan {
  int64_t long_rows;   // 0: the only request, whatever its length
  int64_t requests;    // that can be long
  int64_t slots, tiles, tokens, q_tiles, splits;
  bool others;         // short requests may be among them
  size_t images, parts_o, parts_ml, rows;  // bytes
  size_t total() const { return std::max(rows, images + parts_o + parts_ml); }
};

bool image_shape(int64_t d, int64_t dv, int64_t group, int64_t block_size) {
  return (d == 64 || d == 128 || d == 256) && dv == d && block_size % 16 == 0 && group <= 32;
}

WindowPlan plan_window(int64_t batch, int64_t heads, int64_t hkv, int64_t d, int64_t dv, int64_t block_size,
                       int64_t total_q, int64_t max_query, int64_t max_len, int64_t window, int64_t sinks) {
  WindowPlan pl{};
  const int64_t group = heads / hkv;
  pl.others = true;
  int64_t row_queries = max_query;
  if (image_shape(d, dv, group, block_size) && max_query * group > kLongRows && max_len > 0) {
    pl.long_rows = batch > 1 ? kLongRows : 0;
    pl.others = batch > 1;
    pl.requests = std::min(batch, batch > 1 ? total_q / (kLongRows / group + 1) : int64_t(1));
    row_queries = kLongRows / group;
  }
  if (pl.requests > 0) {
    const int64_t seen = rows_bound(max_len, max_query, window, sinks);
    pl.tiles = (seen + kKeys - 1) / kKeys;
    const int64_t per_slot = hkv * pl.tiles * img_bytes(int(d));
    pl.slots = std::max<int64_t>(1, std::min(pl.requests, kImageBytes / per_slot));
    pl.tokens = kRows / group;
    pl.q_tiles = ((batch > 1 ? max_query : std::max(max_query, total_q)) + pl.tokens - 1) / pl.tokens;
    // Two workgroups a CU, parts of at least eight images.
    const int64_t items = pl.slots * hkv * pl.q_tiles;
    const int64_t walk = std::min(pl.tiles, (rows_bound(max_len, pl.tokens, window, sinks) + kKeys - 1) / kKeys + 1);
    pl.splits = std::max<int64_t>(1, std::min({512 / items, walk / 8, int64_t(kMaxSplits)}));
    pl.images = size_t(pl.slots) * per_slot;
    if (pl.splits > 1) {
      pl.parts_o = size_t(items) * pl.splits * kRows * d * sizeof(float);
      pl.parts_ml = size_t(items) * pl.splits * kRows * 2 * sizeof(float);
    }
  }
  if (pl.others)
    pl.rows = row_workspace(batch, total_q, heads, hkv, d, dv, block_size, row_queries,
                            rows_bound(max_len, row_queries, window, sinks), false);
  return pl;
}

template <int kD, bool kBf16, typename BtT>
int launch_images(const char *name, WindowParams p, int64_t requests, hipStream_t s) {
  constexpr int kTiles = kThreads / kD;
  constexpr size_t kSmem = 2 * size_t(img_bytes(kD));
  if (const int st = reserve_dynamic_lds(reinterpret_cast<const void *>(&window_attention_kernel<kD, kBf16, BtT>), kSmem,
                                         name))
    return st;
  const int64_t groups = int64_t(p.slots) * ((p.tiles + kTiles - 1) / kTiles);
  const int64_t items = int64_t(p.slots) * p.r.hkv * p.q_tiles;
  for (p.first_slot = 0; p.first_slot < requests; p.first_slot += p.slots) {
    window_image_kernel<kD, kBf16, BtT><<<unsigned((groups + 7) / 8 * 8 * p.r.hkv), kThreads, 0, s>>>(p);
    window_attention_kernel<kD, kBf16, BtT>
        <<<unsigned((items * p.splits + 7) / 8 * 8), kThreads, kSmem, s>>>(p);
    if (p.splits > 1)
      window_join_kernel<kD, kBf16><<<dim3(unsigned(items), kRows / (kThreads / kWave)), kThreads, 0, s>>>(p);
    if (const int st = check_launch(name)) return st;
  }
  return HIF8_OK;
}

template <bool kBf16, typename BtT>
int launch_images_of(const char *name, const WindowParams &p, int64_t requests, hipStream_t s) {
  if (p.r.d == 64) return launch_images<64, kBf16, BtT>(name, p, requests, s);
  if (p.r.d == 128) return launch_images<128, kBf16, BtT>(name, p, requests, s);
  return launch_images<256, kBf16, BtT>(name, p, requests, s);
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
  const WindowPlan pl = plan_window(batch, num_heads, num_kv_heads, head_size, head_size_v, block_size,
                                    total_query_tokens, max_query_len, max_seq_len, window, sinks);
  // Bytes for either: the query's alignment, which also decides, is not known here.
  return std::max(pl.total(), row_workspace(batch, total_query_tokens, num_heads, num_kv_heads, head_size, head_size_v,
                                            block_size, max_query_len,
                                            rows_bound(max_seq_len, max_query_len, window, sinks), false));
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
  if (pl.requests == 0 || !aligned(query, 16) || !aligned(out, 16)) return row_attention(kName, a);
  if (!aligned(workspace, 16))
    return fail(HIF8_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned", kName);
  const int64_t items = pl.slots * num_kv_heads * pl.q_tiles;
  if (items * pl.splits > 0xFFFFFF || pl.slots * num_kv_heads * (pl.tiles + 8) > 0xFFFFFF)  // threads of a launch
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
  p.q_tiles = int(pl.q_tiles);
  p.splits = int(pl.splits);
  p.zero_rest = pl.others ? 0 : 1;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool i64 = block_table_dtype == HIF8_INDEX_INT64;
  if (q_dtype == HIF8_DTYPE_BF16)
    return i64 ? launch_images_of<true, int64_t>(kName, p, pl.requests, s)
               : launch_images_of<true, int32_t>(kName, p, pl.requests, s);
  return i64 ? launch_images_of<false, int64_t>(kName, p, pl.requests, s)
             : launch_images_of<false, int32_t>(kName, p, pl.requests, s);
}
