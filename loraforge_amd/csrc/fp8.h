// The FP8 format on gfx950: e4m3 codes (OCP: a sign, values 0 .. 448, 0x7f and
// 0xff NaN, no infinity) with one fp32 scale for every 128 values of a row
// (activations) or every 128 x 128 block of a matrix (weights); the last block of a
// dimension may be shorter. A code stands for its value times the scale.
//
// The conversions used here were checked on gfx950 against their definitions: e4m3 to
// bf16 is exact for all codes (a bf16 holds every e4m3 value), fp32 to e4m3 rounds to
// nearest even.
//
// The 8-bit matrix instructions (v_mfma_*_f8f6f4, and the older v_mfma_*_fp8_fp8 alike) align
// eight products of consecutive k to the one of largest exponent and drop what lies
// more than 13 bits below it; across the eights they keep 24 bits. Found with single
// products: 2^16 + 2^3 - 2^16 is exact within eight, 2^16 + 2^2 - 2^16 gives 0. It is
// the price of their rate, four times that of bf16's. Eight products lose up to 7 x 2^-13 of
// their largest (seven just below the cut, of one sign). Measured on sums of 128 products, 64 rows x 4096
// weights, of the sum of magnitudes: values of N(0, 1) 2^-15.8 at most and 2^-18.9 in the root mean square, with one
// channel in 64 eight times as large 2^-14.3 and 2^-18.2, beside a result that is
// rounded to bf16, 2^-9 of it. Products with bf16 x are exact in fp32.
#pragma once

#include "common.h"

namespace lf {
namespace fp8 {

constexpr int kBlock = 128;  // values of a row, and rows of a weight, per scale
constexpr float kMax = 448.0f;

__host__ __device__ __forceinline__ constexpr int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

typedef int i32x8 __attribute__((ext_vector_type(8)));

// 32 codes as an operand of v_mfma_f32_16x16x128_f8f6f4 and 32x32x64.
__device__ __forceinline__ i32x8 operand(const u32x4& a, const u32x4& b) {
  return __builtin_shufflevector(__builtin_bit_cast(int __attribute__((ext_vector_type(4))), a),
                                 __builtin_bit_cast(int __attribute__((ext_vector_type(4))), b), 0, 1, 2, 3, 4, 5, 6, 7);
}

// 16 x 16 products over 128 k (of which lane quarter q holds 32), from zero: no scales.
__device__ __forceinline__ f32x4 mfma16(const i32x8& a, const i32x8& b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// Two codes of a word (the low or high half) as a bf16 pair.
template <bool kHigh>
__device__ __forceinline__ uint32_t decode2(uint32_t codes) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, kHigh));
}
// Eight codes as eight bf16 values.
__device__ __forceinline__ u32x4 decode8(uint32_t lo, uint32_t hi) {
  return u32x4{decode2<false>(lo), decode2<true>(lo), decode2<false>(hi), decode2<true>(hi)};
}

}  // namespace fp8
}  // namespace lf
