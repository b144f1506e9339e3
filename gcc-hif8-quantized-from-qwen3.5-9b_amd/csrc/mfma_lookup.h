// HiF8 codes into MFMA operands through a lookup table in LDS, for gfx950.
//
// The table holds one 32-bit entry per code - its bf16 (or fp16) value below,
// its fp16 value above - once per lane: entry c of lane i lies at byte
// 256 c + 4 i, so the 64 lanes of a lookup read 64 different banks whatever
// their codes are, and an address is one byte permutation of the code word.
// Every HiF8 value is exact in bf16 and in fp16.
#pragma once

#include "hif8_common.h"

namespace hif8 {

constexpr int kLookupBytes = 256 * 256;

typedef uint32_t lk_u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 lk_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 lk_f16x8 __attribute__((ext_vector_type(8)));
typedef float lk_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short lk_u16x2 __attribute__((ext_vector_type(2)));

// Fills the table, with 256 words of LDS for the entries before they are spread
// (256 threads work one out each: loading them took longer than a short call's
// attention).  The caller synchronises afterwards.
template <bool kBf16Low, int kThreads>
__device__ __forceinline__ void fill_lookup(uint32_t *table, uint32_t *entries, int tid) {
  if (tid < 256) {
    const uint32_t f = decode_bits(uint32_t(tid));
    const uint32_t h = float_to_f16_bits(__uint_as_float(f));  // exact
    entries[tid] = (kBf16Low ? f >> 16 : h) | (h << 16);
  }
  lds_barrier();
#pragma unroll
  for (int i = 0; i < 4096 / kThreads; ++i) {
    const uint32_t v = entries[(tid >> 4) + kThreads / 16 * i];
    reinterpret_cast<lk_u32x4 *>(table)[tid + kThreads * i] = lk_u32x4{v, v, v, v};
  }
}

// One 16-bit table value: code = byte kByte of w; kHigh picks the entry's upper
// half.  lane4 = 4 * lane, the low byte of the offset (the code is the high one);
// table = the table's LDS address.
template <int kByte, bool kHigh>
__device__ __forceinline__ uint16_t look(uint32_t w, uint32_t lane4, uint32_t table) {
  typedef const __attribute__((address_space(3))) uint16_t lds_u16;
  const uint32_t at = __builtin_amdgcn_perm(w, lane4, 0x0c0c0000u | uint32_t((4 + kByte) << 8));
  return *reinterpret_cast<lds_u16 *>(at + table + (kHigh ? 2u : 0u));
}

// Eight codes of two words -> eight 16-bit values in order.
template <bool kHigh>
__device__ __forceinline__ lk_u32x4 look8(uint32_t w0, uint32_t w1, uint32_t lane4, uint32_t table) {
  lk_u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, lk_u16x2{look<0, kHigh>(w0, lane4, table), look<1, kHigh>(w0, lane4, table)});
  r[1] = __builtin_bit_cast(uint32_t, lk_u16x2{look<2, kHigh>(w0, lane4, table), look<3, kHigh>(w0, lane4, table)});
  r[2] = __builtin_bit_cast(uint32_t, lk_u16x2{look<0, kHigh>(w1, lane4, table), look<1, kHigh>(w1, lane4, table)});
  r[3] = __builtin_bit_cast(uint32_t, lk_u16x2{look<2, kHigh>(w1, lane4, table), look<3, kHigh>(w1, lane4, table)});
  return r;
}

// Byte kByte of each of eight words -> eight 16-bit values.
template <int kByte, bool kHigh>
__device__ __forceinline__ lk_u32x4 look_column(const uint32_t *w, uint32_t lane4, uint32_t table) {
  lk_u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = __builtin_bit_cast(uint32_t, lk_u16x2{look<kByte, kHigh>(w[2 * i], lane4, table),
                                                 look<kByte, kHigh>(w[2 * i + 1], lane4, table)});
  return r;
}

template <bool kBf16>
__device__ __forceinline__ lk_f32x4 mfma_16x16x32(lk_u32x4 a, lk_u32x4 b, lk_f32x4 c) {
  if constexpr (kBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lk_bf16x8, a), __builtin_bit_cast(lk_bf16x8, b),
                                                   c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(lk_f16x8, a), __builtin_bit_cast(lk_f16x8, b), c,
                                                  0, 0, 0);
}

// The other lanes' values of the same column (lane % 16): the row swaps of gfx950
// leave x of lanes 16 (or 32) apart side by side, without a trip through LDS.
__device__ __forceinline__ float max_over_groups(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const float y = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float sum_over_groups(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const float y = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Sum over the 16 lanes of a group (lane / 16), in all of them: rotations within
// the row of 16, an addition each, where shuffles go through LDS.
template <int kBy>
__device__ __forceinline__ float rotated(float x) {
  return __uint_as_float(uint32_t(__builtin_amdgcn_update_dpp(0, int(__float_as_uint(x)), 0x120 + kBy, 0xF, 0xF, false)));
}
__device__ __forceinline__ float sum_over_columns(float x) {
  x += rotated<8>(x);
  x += rotated<4>(x);
  x += rotated<2>(x);
  return x + rotated<1>(x);
}

// Inclusive sum over the lanes of a wavefront: shifts within rows of 16, then the
// rows' last lanes handed on to the rows behind.
__device__ __forceinline__ int wave_prefix(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
}

// Bit 7 of each byte: it is no infinity (0x6F, 0xEF) and no NaN (0x80).  The other bits
// mean nothing; words are joined by `and`.
__device__ __forceinline__ uint32_t finite_bytes(uint32_t w) {
  const uint32_t size = w & 0x7F7F7F7Fu;
  return ((size ^ 0x6F6F6F6Fu) + 0x7F7F7F7Fu) & ((size + 0x7F7F7F7Fu) | ~w);
}

// True when some byte of w is an infinity (0x6F, 0xEF) or NaN (0x80); may also
// be true next to such a byte, never false on one.
__device__ __forceinline__ bool some_not_finite(uint32_t w) {
  const uint32_t inf = (w & 0x7F7F7F7Fu) ^ 0x6F6F6F6Fu, nan = w ^ 0x80808080u;
  return (((inf - 0x01010101u) & ~inf) | ((nan - 0x01010101u) & ~nan)) & 0x80808080u;
}

}  // namespace hif8
