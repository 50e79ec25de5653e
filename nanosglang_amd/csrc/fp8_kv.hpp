// The 8-bit KV pool: what its writers and readers share.
//
// A layer's pool holds e4m3 codes [num_pages, page_size, num_kv_heads,
// head_dim] for K and for V, and one power-of-two scale per (token, KV head) of
// each, as an E8M0 byte e (value 2^(e - 127)) in kv_scale [num_pages,
// num_kv_heads, 2, page_size] (K's bytes, then V's): a head's 2 P bytes of a
// page lie together, so that a reader of one head touches no other head's.
//
// A row x is stored with the smallest e >= 1 for which max |x| <= 448 *
// 2^(e - 127) (448: e4m3's largest value) and codes rne(x * 2^(127 - e)).  The
// scale is a power of two because a code times it is then exact in bf16 (four
// significant bits): gfx950's v_cvt_scalef32_pk_bf16_fp8 does the
// dequantisation within the conversion to bf16 that the MFMA operand needs
// anyway, with no rounding of its own, and one byte a row is 1 / 128 of the
// codes at head dim 128.  A row with a NaN or an infinity, or a value that e4m3
// would round to 2^128 (from 1.9375 * 2^127 on), has e = 255: it reads back as
// NaN.  Its V codes are zero, so that a probability of zero on such a
// row (a masked position of a tile) adds nothing instead of 0 * NaN.
#pragma once

#include "common.hpp"

namespace nsg {

typedef uint32_t fp8_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t fp8_u32x4 __attribute__((ext_vector_type(4)));
typedef short fp8_s16x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kE8M0NaN = 255;

// E8M0 byte as the fp32 scale (255: infinity, which the conversions below
// turn into NaN for every code).
__device__ __forceinline__ float e8m0_scale(uint32_t e) { return __uint_as_float(e << 23); }

// The byte of a row whose largest |x| has the fp32 bits `amax` (as an
// unsigned integer, so NaN orders above infinity and is not lost): amax = 1.m
// * 2^(E - 127) needs 2^(E - 8 - 127) if 1.m <= 1.75 (448 = 1.75 * 2^8), else
// twice that.
__device__ __forceinline__ uint32_t e8m0_of(uint32_t amax) {
  if (amax >= 0x7f780000u) return kE8M0NaN;
  const int e = (int)((amax + 0x1fffffu) >> 23) - 8;
  return e < 1 ? 1u : (uint32_t)e;
}

// Four bf16 values (two packed pairs) over `scale`, rounded to e4m3.
__device__ __forceinline__ uint32_t to_fp8x4(uint32_t lo, uint32_t hi, float scale) {
  fp8_s16x2 o = {0, 0};
  o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, __builtin_bit_cast(bf16x2_t, lo), scale, false);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, __builtin_bit_cast(bf16x2_t, hi), scale, true);
  return __builtin_bit_cast(uint32_t, o);
}

// Four codes times `scale` as two packed bf16 pairs (exact).
__device__ __forceinline__ fp8_u32x2 from_fp8x4(uint32_t codes, float scale) {
  return fp8_u32x2{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true))};
}

// Offset of a row's scale byte: token slot `slot`, KV head h, which = 0 (K) or 1 (V).
__device__ __forceinline__ int64_t scale_at(int64_t slot, int log2P, int Hkv, int h, int which) {
  const int64_t page = slot >> log2P;
  return (((page * Hkv + h) * 2 + which) << log2P) + (slot & ((1 << log2P) - 1));
}

}  // namespace nsg
