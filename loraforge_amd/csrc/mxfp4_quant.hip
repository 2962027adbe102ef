// MXFP4 quantisation and its inverse.
//
// Each block of 32 values along k: m = max |x|, scale 2^E with E = floor(log2 m) - 2
// (clamped at -127), code = e2m1 nearest to x 2^-E, ties to even, saturated at 6. The
// division by a power of two is exact, so codes do not depend on how they are computed.
// HBM-bound: 2 or 4 bytes read and 17/32 written an element, and 17/32 read and 2
// written on the way back: 24576 x 4096 in bf16 37-57 us (4.5-6.9 TB/s: the input, used again, may be in the
// memory-side cache), in fp32 86 us (5.3 TB/s), and 37.7 back (6.7 TB/s; a copy reaches 5.1), 4096 x 4096
// 8.2 us. Seven rows take 2.2 us each way: one load's latency.
#include "mxfp4.h"
#include "../../include/loraforge_amd.h"

namespace lf {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint32_t max4(uint32_t v) {
  v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0xB1, 0xf, 0xf, true)));  // quad_perm 1 0 3 2
  return max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x4E, 0xf, 0xf, true)));  // quad_perm 2 3 0 1
}

// Eight values of a block: the four lanes of a quad hold it whole.
template <class T>
struct Eight;

template <>
struct Eight<uint16_t> {
  uint4 v;
  __device__ __forceinline__ void load(const uint16_t* p) { v = *reinterpret_cast<const uint4*>(p); }
  // (bf16 magnitudes order as their bits do: the two halves of a pair are compared as integers.)
  __device__ __forceinline__ uint32_t magnitude() const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t hi = 0, lo = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hi = max(hi, w[i] & 0x7fff0000u);
      lo = max(lo, (w[i] << 16) & 0x7fff0000u);
    }
    return max(hi, lo);
  }
  __device__ __forceinline__ uint32_t encode(float scale) const {
    const bf16x2 a = __builtin_bit_cast(bf16x2, v.x), b = __builtin_bit_cast(bf16x2, v.y);
    const bf16x2 c = __builtin_bit_cast(bf16x2, v.z), d = __builtin_bit_cast(bf16x2, v.w);
    uint32_t q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, a, scale, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, b, scale, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, c, scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, d, scale, 3);
  }
};

template <>
struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ uint32_t magnitude() const {
    const float w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(w[i]) & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ uint32_t encode(float scale) const {
    uint32_t q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a.x, a.y, scale, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, a.z, a.w, scale, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, b.x, b.y, scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, b.z, b.w, scale, 3);
  }
};

// One quad of lanes per block, one block per quad and step. A block that holds
// infinity or NaN gets scale 255 (NaN) and zero codes.
template <class T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const T* x, int64_t blocks, int64_t row_blocks,
                                                            int64_t stride, uint32_t* codes, uint8_t* scales) {
  const int part = threadIdx.x & 3;
  const bool flat = stride == row_blocks * mx::kBlock;
  for (int64_t b = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 2; b < blocks; b += int64_t(gridDim.x) * (kThreads / 4)) {
    const int64_t row = flat ? 0 : b / row_blocks;
    Eight<T> v;
    v.load(x + row * stride + (b - row * row_blocks) * mx::kBlock + part * 8);
    const uint32_t byte = mx::scale_byte(max4(v.magnitude()));
    codes[b * 4 + part] = byte == 255u ? 0u : v.encode(mx::scale_f32(byte));
    if (part == 0) scales[b] = uint8_t(byte);
  }
}

// Eight codes per lane: 4 bytes read, 16 written.
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint32_t* codes, const uint8_t* scales, int64_t words,
                                                              u32x4* out) {
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < words; i += int64_t(gridDim.x) * kThreads)
    out[i] = mx::decode8(codes[i], mx::scale_f32(scales[i >> 2]));
}

unsigned blocks_for(int64_t items) {
  const int64_t want = (items + kThreads - 1) / kThreads;
  return unsigned(want < 8192 ? want : 8192);
}

}  // namespace
}  // namespace lf

extern "C" int lf_mxfp4_quantize(const void* x, int32_t fp32, int64_t rows, int64_t k, int64_t x_stride, uint8_t* codes,
                                 uint8_t* scales, void* stream) {
  LF_REQUIRE(rows >= 0 && k > 0 && k % lf::mx::kBlock == 0, "k must be a positive multiple of 32");
  LF_REQUIRE(x_stride >= k, "x_stride must cover k values");
  if (rows == 0) return lf::kOk;
  LF_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr, "null pointer argument");
  LF_REQUIRE(lf::aligned16(x) && x_stride % (fp32 ? 4 : 8) == 0, "x rows must be 16-byte aligned");
  LF_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 4 == 0, "codes must be 4-byte aligned");
  const int64_t row_blocks = k / lf::mx::kBlock, blocks = rows * row_blocks;
  if (rows == 1) x_stride = k;
  const dim3 grid(lf::blocks_for(blocks * 4)), threads(lf::kThreads);
  auto s = static_cast<hipStream_t>(stream);
  auto* words = reinterpret_cast<uint32_t*>(codes);
  if (fp32)
    hipLaunchKernelGGL(lf::quantize_kernel<float>, grid, threads, 0, s, static_cast<const float*>(x), blocks, row_blocks,
                       x_stride, words, scales);
  else
    hipLaunchKernelGGL(lf::quantize_kernel<uint16_t>, grid, threads, 0, s, static_cast<const uint16_t*>(x), blocks,
                       row_blocks, x_stride, words, scales);
  LF_HIP(hipGetLastError());
  return lf::kOk;
}

extern "C" int lf_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t blocks, uint16_t* out, void* stream) {
  LF_REQUIRE(blocks >= 0, "blocks must be non-negative");
  if (blocks == 0) return lf::kOk;
  LF_REQUIRE(codes != nullptr && scales != nullptr && out != nullptr, "null pointer argument");
  LF_REQUIRE(lf::aligned16(out) && reinterpret_cast<uintptr_t>(codes) % 4 == 0,
             "out must be 16-byte and codes 4-byte aligned");
  const int64_t words = blocks * 4;
  hipLaunchKernelGGL(lf::dequantize_kernel, dim3(lf::blocks_for(words)), dim3(lf::kThreads), 0,
                     static_cast<hipStream_t>(stream), reinterpret_cast<const uint32_t*>(codes), scales, words,
                     reinterpret_cast<lf::u32x4*>(out));
  LF_HIP(hipGetLastError());
  return lf::kOk;
}
