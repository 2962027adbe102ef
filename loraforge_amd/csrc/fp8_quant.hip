// FP8 quantisation and its inverse.
//
// Of each block (128 values of a row, or 128 x 128 of a matrix): A = max(max |x|, 2^-100),
// scale = fp32(A / 448), code = e4m3 nearest to 448 x / A, ties to even. With the bf16 x =
// X 2^i and A = B 2^j (X, B below 2^8) the quotient is a tie only where it is a fraction of
// few bits, and else at least 2^-13 of itself away from one; the division below is exact in
// the first case and right to 2^-23 in the second, so that the codes are those of
// the formula in real numbers.
//
// HBM-bound: 2 bytes read and 1 written an element, and 1 read and 2 written on the way back. 24576 x 4096 in blocks
// 67 us (4.5 TB/s), back 51 (5.9); 8192 rows of 4096 23 (4.4), 5 rows 2.8 each way, which is a launch.
#include "fp8.h"
#include "../../include/loraforge_amd.h"

namespace lf {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kLeast = (127u - 100u) << 23;  // 2^-100

// What a block with this largest magnitude (fp32 bits) multiplies its values with and
// divides them by: 448 x / A = (x factor) / divisor, with the divisor in [1, 2).
struct Block {
  float factor, divisor, inverse, scale;
  bool finite;

  __device__ __forceinline__ explicit Block(uint32_t magnitude) {
    finite = magnitude < 0x7f800000u;
    const uint32_t a = max(magnitude, kLeast);
    const uint32_t e = a >> 23;  // biased
    factor = __uint_as_float(((262u - e) << 23) | 0x600000u);  // 1.75 * 2^8 * 2^(127 - e)
    divisor = __uint_as_float((a & 0x7fffffu) | 0x3f800000u);
    inverse = __builtin_amdgcn_rcpf(divisor);
    inverse = fmaf(fmaf(-divisor, inverse, 1.0f), inverse, inverse);
    scale = finite ? __uint_as_float(a) / fp8::kMax : __builtin_nanf("");
  }
  __device__ __forceinline__ float quotient(float x) const {
    const float n = x * factor, q = n * inverse;
    return fmaf(fmaf(-q, divisor, n), inverse, q);
  }
  // Codes of four bf16 values.
  __device__ __forceinline__ uint32_t encode4(uint32_t a, uint32_t b) const {
    if (!finite) return 0u;
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(bf16_lo(a)), quotient(bf16_hi(a)), 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(quotient(bf16_lo(b)), quotient(bf16_hi(b)), v, true));
  }
};

// Largest magnitude of eight bf16 values, as fp32 bits (magnitudes order as their bits do).
__device__ __forceinline__ uint32_t magnitude8(const u32x4& v) {
  uint32_t hi = 0, lo = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi = max(hi, v[i] & 0x7fff0000u);
    lo = max(lo, (v[i] << 16) & 0x7fff0000u);
  }
  return max(hi, lo);
}

template <int kCtrl>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  return max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), kCtrl, 0xf, 0xf, true)));
}
// The maximum over a row of 16 lanes, by rotations.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
  return max_dpp<0x121>(max_dpp<0x122>(max_dpp<0x124>(max_dpp<0x128>(v))));
}

// How a grid of kThreads-sized workgroups covers rows x chunks of eight values: `lanes`
// (a power of two) chunks of a row beside each other, strips of them in x, rows in y.
struct Cover {
  int chunks, lanes, rows;  // chunks of a row; lanes of a row; rows of a workgroup
};

// Scales of 128 values of a row: 16 lanes a block, 16 bytes a lane.
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const uint16_t* x, int64_t rows, int64_t k, int64_t stride,
                                                                 Cover g, uint8_t* codes, float* scales) {
  const int lane = threadIdx.x & (g.lanes - 1), in_row = threadIdx.x / g.lanes;
  const int chunk = blockIdx.x * g.lanes + lane;
  const bool in = chunk < g.chunks;
  const int64_t blocks = fp8::blocks_of(k);
  for (int64_t row = int64_t(blockIdx.y) * g.rows + in_row; row < rows; row += int64_t(gridDim.y) * g.rows) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if (in) v = *reinterpret_cast<const u32x4*>(x + row * stride + int64_t(chunk) * 8);
    const Block b(max16(magnitude8(v)));
    if (in) {
      *reinterpret_cast<uint2*>(codes + row * k + int64_t(chunk) * 8) = make_uint2(b.encode4(v[0], v[1]), b.encode4(v[2], v[3]));
      if (chunk % 16 == 0) scales[row * blocks + chunk / 16] = b.scale;
    }
  }
}

// Scales of 128 x 128 blocks: a workgroup a block, 16 lanes a row, eight rows a thread.
__global__ __launch_bounds__(kThreads) void quantize_blocks_kernel(const uint16_t* x, int64_t rows, int64_t k, int64_t stride,
                                                                   int64_t row_blocks, int64_t all, uint8_t* codes, float* scales) {
  __shared__ uint32_t most[2][kThreads / 64];
  constexpr int kPer = fp8::kBlock / 16;
  const int64_t at = int64_t(blockIdx.x) * fp8::kBlock + (threadIdx.x & 15) * 8;
  for (int64_t b = blockIdx.y, turn = 0; b < all; b += gridDim.y, turn ^= 1) {
    const int64_t matrix = b / row_blocks, first = (b - matrix * row_blocks) * fp8::kBlock;
    const int left = int(rows - first < fp8::kBlock ? rows - first : fp8::kBlock);
    const int64_t row0 = matrix * rows + first;
    u32x4 v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = 16 * i + int(threadIdx.x >> 4);
      v[i] = u32x4{0u, 0u, 0u, 0u};
      if (r < left && at < k) v[i] = *reinterpret_cast<const u32x4*>(x + (row0 + r) * stride + at);
    }
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine = max(mine, magnitude8(v[i]));
    mine = max16(mine);
    mine = max(mine, uint32_t(__shfl_xor(int(mine), 16, 64)));
    mine = max(mine, uint32_t(__shfl_xor(int(mine), 32, 64)));
    // (Two places in turn: who is still behind the last barrier reads the other one.)
    if ((threadIdx.x & 63) == 0) most[turn][threadIdx.x >> 6] = mine;
    __syncthreads();
    const Block q(max(max(most[turn][0], most[turn][1]), max(most[turn][2], most[turn][3])));
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = 16 * i + int(threadIdx.x >> 4);
      if (r < left && at < k)
        *reinterpret_cast<uint2*>(codes + (row0 + r) * k + at) = make_uint2(q.encode4(v[i][0], v[i][1]), q.encode4(v[i][2], v[i][3]));
    }
    if (threadIdx.x == 0) scales[b * gridDim.x + blockIdx.x] = q.scale;
  }
}

// Eight codes a lane: 8 bytes read, 16 written. A scale for `scale_rows` rows of each matrix of `rows` rows.
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint8_t* codes, const float* scales, int64_t all_rows, int64_t rows,
                                                              int64_t k, int32_t scale_rows, Cover g, uint16_t* out) {
  const int lane = threadIdx.x & (g.lanes - 1), in_row = threadIdx.x / g.lanes;
  const int chunk = blockIdx.x * g.lanes + lane;
  if (chunk >= g.chunks) return;
  const int64_t blocks = fp8::blocks_of(k), row_blocks = (rows + scale_rows - 1) / scale_rows;
  for (int64_t row = int64_t(blockIdx.y) * g.rows + in_row; row < all_rows; row += int64_t(gridDim.y) * g.rows) {
    int64_t scale_row = row;
    if (scale_rows != 1) {
      const int64_t matrix = row / rows;
      scale_row = matrix * row_blocks + (row - matrix * rows) / fp8::kBlock;
    }
    const float scale = scales[scale_row * blocks + chunk / 16];
    const uint2 c = *reinterpret_cast<const uint2*>(codes + row * k + int64_t(chunk) * 8);
    const uint32_t word[2] = {c.x, c.y};
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(int(word[i]), false), b = __builtin_amdgcn_cvt_pk_f32_fp8(int(word[i]), true);
      o[2 * i] = pack_bf16x2(a[0] * scale, a[1] * scale);
      o[2 * i + 1] = pack_bf16x2(b[0] * scale, b[1] * scale);
    }
    *reinterpret_cast<u32x4*>(out + row * k + int64_t(chunk) * 8) = o;
  }
}

Cover cover(int64_t k, dim3& grid, int64_t rows) {
  Cover g;
  g.chunks = int(k / 8);
  g.lanes = 16;
  while (g.lanes < g.chunks && g.lanes < kThreads) g.lanes *= 2;
  g.rows = kThreads / g.lanes;
  const int64_t strips = (g.chunks + g.lanes - 1) / g.lanes, want = (rows + g.rows - 1) / g.rows;
  const int64_t most = 16384 / strips > 1 ? 16384 / strips : 1;  // (each workgroup then takes several rows)
  grid = dim3(unsigned(strips), unsigned(want < most ? want : most));
  return g;
}

}  // namespace
}  // namespace lf

extern "C" int lf_fp8_quantize(const uint16_t* x, int64_t matrices, int64_t rows, int64_t k, int64_t x_stride, int32_t scale_rows,
                               uint8_t* codes, float* scales, void* stream) {
  LF_REQUIRE(matrices >= 0 && rows >= 0 && k > 0 && k % 16 == 0 && k < (int64_t(1) << 31), "k must be a positive multiple of 16");
  LF_REQUIRE(scale_rows == 1 || scale_rows == lf::fp8::kBlock, "a scale covers 1 or 128 rows");
  LF_REQUIRE(rows < (int64_t(1) << 31) && matrices < (int64_t(1) << 31), "sizes must fit signed int32 indexing");
  LF_REQUIRE(x_stride >= k, "x_stride must cover k values");
  if (rows == 0 || matrices == 0) return lf::kOk;
  LF_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr, "null pointer argument");
  LF_REQUIRE(lf::aligned16(x) && x_stride % 8 == 0, "x rows must be 16-byte aligned");
  LF_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 8 == 0, "codes must be 8-byte aligned");
  auto s = static_cast<hipStream_t>(stream);
  if (scale_rows == 1) {
    dim3 grid;
    const lf::Cover g = lf::cover(k, grid, matrices * rows);
    hipLaunchKernelGGL(lf::quantize_rows_kernel, grid, dim3(lf::kThreads), 0, s, x, matrices * rows, k, x_stride, g, codes, scales);
  } else {
    const int64_t row_blocks = lf::fp8::blocks_of(rows), all = matrices * row_blocks;
    hipLaunchKernelGGL(lf::quantize_blocks_kernel, dim3(unsigned(lf::fp8::blocks_of(k)), unsigned(all < 65535 ? all : 65535)),
                       dim3(lf::kThreads), 0, s, x, rows, k, x_stride, row_blocks, all, codes, scales);
  }
  LF_HIP(hipGetLastError());
  return lf::kOk;
}

extern "C" int lf_fp8_dequantize(const uint8_t* codes, const float* scales, int64_t matrices, int64_t rows, int64_t k,
                                 int32_t scale_rows, uint16_t* out, void* stream) {
  LF_REQUIRE(matrices >= 0 && rows >= 0 && k > 0 && k % 16 == 0 && k < (int64_t(1) << 31), "k must be a positive multiple of 16");
  LF_REQUIRE(scale_rows == 1 || scale_rows == lf::fp8::kBlock, "a scale covers 1 or 128 rows");
  LF_REQUIRE(rows < (int64_t(1) << 31) && matrices < (int64_t(1) << 31), "sizes must fit signed int32 indexing");
  if (rows == 0 || matrices == 0) return lf::kOk;
  LF_REQUIRE(codes != nullptr && scales != nullptr && out != nullptr, "null pointer argument");
  LF_REQUIRE(lf::aligned16(out) && reinterpret_cast<uintptr_t>(codes) % 8 == 0, "out must be 16-byte and codes 8-byte aligned");
  dim3 grid;
  const lf::Cover g = lf::cover(k, grid, matrices * rows);
  hipLaunchKernelGGL(lf::dequantize_kernel, grid, dim3(lf::kThreads), 0, static_cast<hipStream_t>(stream), codes, scales,
                     matrices * rows, rows, k, scale_rows, g, out);
  LF_HIP(hipGetLastError());
  return lf::kOk;
}
