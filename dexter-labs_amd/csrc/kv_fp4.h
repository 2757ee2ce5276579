// A KV cache's pages in 4 bits on gfx950: the format, and reading it.
//
// A row of a head is D codes of 4 bits and D / 32 scale bytes. A code is a sign
// and an E2M1 number (0, 0.5, 1, 1.5, 2, 3, 4 or 6), two to a byte, the earlier
// element in the low half; 32 consecutive ones (a block) share the scale
// 2^(byte - 127), a byte of 255 makes them NaN. It is the format that this
// hardware converts by itself: one instruction gives two values of bf16 or f16
// with their scale, and a code has 2 significant bits, so the values are exact in
// either type: reading rounds nothing.
//
// The scale is 2^e for the least e with every magnitude of the block at most
// 7 * 2^e, so that the rounding to 6, the largest code, is off by at most the
// half step 2^e that any code above 4 may be off by. Relative to the values' norm,
// of normal data: 0.112. e keeps to [-127, 125] for bf16 and [-23, 13] for f16, where
// all of a block's values are numbers of that type.
//
// A pool is bytes [2, P, H, R * (D / 2 + D / 32)]: of each page and head first the
// codes of its R rows, then their scales. Heads come before rows, unlike in a
// 16-bit pool: a head's 16 rows, the least that lies in one page, are then 1 KB of
// codes in one piece (D 128), where a row alone would be half of a cache line.
#pragma once

#include "dx_common.h"

namespace dx {
namespace {

template <typename T> struct Fp4Range;
template <> struct Fp4Range<bf16_t> { static constexpr int lo = 0, hi = 125 + 127; };
template <> struct Fp4Range<f16_t> { static constexpr int lo = 127 - 23, hi = 13 + 127; };

// The scale of a byte, as the conversions take it: the bits of 2^(byte - 127), of which
// they use the exponent (0 is 2^-127, 255 NaN).
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes to eight values.
template <typename T> __device__ __forceinline__ u32x4 fp4_values(uint32_t codes, float scale);
template <> __device__ __forceinline__ u32x4 fp4_values<bf16_t>(uint32_t codes, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
}
template <> __device__ __forceinline__ u32x4 fp4_values<f16_t>(uint32_t codes, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3))};
}

// From the codes of a page's row `in_page` to its scale bytes.
template <int D>
__device__ __forceinline__ uint64_t fp4_scales_behind(int page_rows, uint32_t in_page) {
  return uint64_t(uint32_t(page_rows)) * (D / 2) - uint64_t(in_page) * (D / 2 - D / 32);
}

}  // namespace

// Bytes of a row of a head, and whether a head dim has the format.
constexpr int64_t fp4_row_bytes(int64_t D) { return D / 2 + D / 32; }

}  // namespace dx
