// The MXFP4 format on gfx950: blocks of 32 e2m1 codes along k (levels 0, .5,
// 1, 1.5, 2, 3, 4, 6 and a sign; the low nibble of a byte is the even k) and one
// e8m0 scale byte s a block; a code stands for level * 2^(s - 127), s = 255 for NaN.
//
// The conversions below and the scaled matrix instruction take such codes and
// bytes as they are. Checked against their definitions on gfx950: the
// conversion to e2m1 rounds to nearest even and saturates at 6 (every bf16
// value at ten scales, every tie and its fp32 neighbours), the conversion to
// bf16 is exact for scale bytes 0..252 (bf16 subnormals included) and gives
// NaN for 255; above 252 the levels past bf16's range become infinite.
#pragma once

#include "common.h"

namespace lf {
namespace mx {

constexpr int kBlock = 32;  // values per scale

// The fp32 whose exponent field is the scale byte: the conversions read nothing else of it.
__device__ __forceinline__ float scale_f32(uint32_t byte) { return __uint_as_float(byte << 23); }

// The two values of byte kSel of eight packed codes, times the scale, as a bf16 pair.
template <int kSel>
__device__ __forceinline__ uint32_t decode2(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, kSel));
}

// 32 packed codes as an operand of the scaled matrix instructions (of 4-bit operands they read four registers).
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ i32x8 operand(const u32x4& codes) {
  const i32x4 v = __builtin_bit_cast(i32x4, codes);
  return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
}

// Eight packed codes as eight bf16 values.
__device__ __forceinline__ u32x4 decode8(uint32_t codes, float scale) {
  return u32x4{decode2<0>(codes, scale), decode2<1>(codes, scale), decode2<2>(codes, scale), decode2<3>(codes, scale)};
}

// The scale byte of a block whose largest magnitude has these fp32 bits:
// floor(log2) - 2 (6 = 1.5 * 2^2 is the largest level), biased by 127, not
// below 0; 255 for infinity and NaN.
__device__ __forceinline__ uint32_t scale_byte(uint32_t magnitude) {
  const uint32_t e = magnitude >> 23;
  return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}

// v without its first `bytes` (0 .. 16), zeros behind.
__device__ __forceinline__ u32x4 drop_bytes(u32x4 v, int bytes) {
  if (bytes & 16) v = u32x4{0u, 0u, 0u, 0u};
  v = bytes & 8 ? u32x4{v.z, v.w, 0u, 0u} : v;
  v = bytes & 4 ? u32x4{v.y, v.z, v.w, 0u} : v;
  const int b = bytes & 3;
  return u32x4{__builtin_amdgcn_alignbyte(v.y, v.x, b), __builtin_amdgcn_alignbyte(v.z, v.y, b),
               __builtin_amdgcn_alignbyte(v.w, v.z, b), __builtin_amdgcn_alignbyte(0u, v.w, b)};
}

}  // namespace mx
}  // namespace lf
