// Parameters of the products with bf16 or MXFP4 weights, dense and grouped by
// expert (expert_stream.hip, expert_tile.h), and what both kernels share.
//
// Rows offsets[e] .. offsets[e + 1] of the product belong to expert e: row p is
// x[tokens[p]] (x[p] without tokens) times the transpose of w[e]. The dense
// product is that of one expert with all rows. Segment bounds and token
// indexes come from device memory; both are clamped to the buffers.
#pragma once

#include "mxfp4.h"

namespace lf {
namespace expert {

struct Params {
  const char* x;       // bf16 [x_rows, k], or packed codes
  int64_t x_row;       // bytes from row to row
  const uint8_t* xs;   // scale bytes [x_rows, k / 32] of packed x
  const char* w;       // bf16 or packed [experts, n, k]
  const uint8_t* ws;   // scale bytes [experts, n, k / 32] of packed w
  const uint16_t* bias;    // [experts, n] or null
  const int32_t* offsets;  // [experts + 1], null: one expert with all rows
  const int32_t* tokens;   // [rows] or null
  uint16_t* y;
  int64_t y_stride;
  int rows, x_rows, n, k, experts;
  int width;   // output columns: n, or n / 2 with SwiGLU
  int y_vec;   // rows of y are 16-byte aligned
  int swiglu;  // w rows [gate | up]: y = silu(gate) * up
};

// Zeros that lanes past the end of k load instead of what follows the row.
__device__ const u32x4 kZeros = {0u, 0u, 0u, 0u};

struct Segment {
  int expert, begin, end;
};

// Bounds of expert e's rows.
__device__ __forceinline__ Segment segment_of(const Params& p, int e) {
  if (!p.offsets) return {0, 0, p.rows};
  const int begin = min(max(p.offsets[e], 0), p.rows);
  return {e, begin, min(max(p.offsets[e + 1], begin), p.rows)};
}

// Searches the experts in order, 64 at a time, for the one that holds item
// `index`, where expert e has count(segment) items; `index` becomes the item's
// number within it. Uniform; an index past the last item finds an empty segment.
template <class Count>
__device__ __forceinline__ Segment find_segment(const Params& p, int& index, Count&& count) {
  if (!p.offsets) return index < count(Segment{0, 0, p.rows}) ? Segment{0, 0, p.rows} : Segment{0, 0, 0};
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < p.experts; base += 64) {
    Segment s{0, 0, 0};
    if (base + lane < p.experts) s = segment_of(p, base + lane);
    const int mine = count(s);
    int sum = mine;  // inclusive sums over the lanes
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(sum, d, 64);
      if (lane >= d) sum += up;
    }
    const uint64_t past = __ballot(sum > index);
    if (past) {
      const int at = __builtin_ctzll(past);
      index -= __builtin_amdgcn_readlane(sum - mine, at);
      return {__builtin_amdgcn_readlane(s.expert, at), __builtin_amdgcn_readlane(s.begin, at),
              __builtin_amdgcn_readlane(s.end, at)};
    }
    index -= __builtin_amdgcn_readlane(sum, 63);
  }
  return {0, 0, 0};
}

// Row of x behind row `pos` of the product.
__device__ __forceinline__ int64_t x_row_of(const Params& p, int pos) {
  return p.tokens ? min(max(p.tokens[pos], 0), p.x_rows - 1) : pos;
}

// SwiGLU in fp32: g / (1 + e^-g) * u from the hardware exp2 and reciprocal (1 ulp
// each). The rounding of the exponent is worth |g| 2^-24 of the result, little beside the
// rounding to bf16 that follows; past g = -87.3 the reciprocal gives 0 where |silu(g)| is below
// 1e-36, as the quotient in 32 bits does past -88.7. A third of the instructions of a correctly
// rounded quotient (a 256 x 256 tile's epilogue 21.9k -> 12.5k cycles). Silu itself is not
// rounded to bf16 here, as silu_times does for the paths that follow a reference which does.
__device__ __forceinline__ float silu_mul_f32(float g, float u) {
  const float e = __builtin_amdgcn_exp2f(g * -1.44269504088896341f);
  return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

// `part`: rows per workgroup (16, 32 or 64); `groups`: 16-row groups of weight rows (1 or 2).
int launch_stream(const Params& p, int part, int groups, hipStream_t stream);
int launch_rows(const Params& p, hipStream_t stream);
// Tiles of at most `cap` rows x `columns` weight rows (one translation unit per pair of types).
int launch_tiles_bf16(const Params& p, int cap, int columns, hipStream_t stream);
int launch_tiles_mxw(const Params& p, int cap, int columns, hipStream_t stream);
int launch_tiles_mx(const Params& p, int cap, int columns, hipStream_t stream);

}  // namespace expert
}  // namespace lf
