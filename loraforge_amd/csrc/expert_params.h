// Parameters of the products with bf16, MXFP4 or FP8 weights, dense and grouped by
// expert (expert_stream.hip, expert_rows.hip, expert_tile.h), and what the kernels share.
//
// Rows offsets[e] .. offsets[e + 1] of the product belong to expert e: row p is
// x[tokens[p]] (x[p] without tokens) times the transpose of w[e]. The dense
// product is that of one expert with all rows. Segment bounds and token
// indexes come from device memory; both are clamped to the buffers.
#pragma once

#include "fp8.h"
#include "mxfp4.h"
#include "../../include/loraforge_amd.h"

namespace lf {
namespace expert {

// Rows held as pairs: a value of 32 bits as the sum of two of bf16 (17 bits or more of it), so that a product's
// result keeps them into the next one. Row r of such an x is rows 2 r and 2 r + 1, two rows of the product.
enum Pair : int {
  kSingle,  // y bf16
  kSplit,   // y: bf16 pairs, rows 2 r and 2 r + 1 of y (of a product with SwiGLU)
  kJoin,    // x: pairs (`rows` and `x_rows` count both), y: fp32, one row for each pair (without)
};

// Types of an operand.
enum Type : int { kBf16, kMxfp4, kFp8 };

struct Params {
  const char* x;       // bf16 [x_rows, k], or codes
  int64_t x_row;       // bytes from row to row
  const uint8_t* xs;   // scale bytes [x_rows, k / 32] of MXFP4 x
  const char* w;       // bf16 or codes [experts, n, k]
  const uint8_t* ws;   // scale bytes [experts, n, k / 32] of MXFP4 w
  const float* xs8;    // scales [x_rows, k / 128 rounded up] of FP8 x
  const float* ws8;    // scales [experts, n / 128, k / 128, both rounded up] of FP8 w
  const uint16_t* bias;    // [experts, n] or null
  const int32_t* offsets;  // [experts + 1], null: one expert with all rows
  const int32_t* tokens;   // [rows] or null
  uint16_t* y;
  int64_t y_stride;
  int rows, x_rows, n, k, experts;
  int width;   // output columns: n, or n / 2 with SwiGLU
  int y_vec;   // rows of y are 16-byte aligned
  int swiglu;  // w rows [gate | up]: y = silu(gate) * up
  int pair;    // Pair
};

// Zeros that lanes past the end of k load instead of what follows the row.
__device__ const u32x4 kZeros = {0u, 0u, 0u, 0u};

struct Segment {
  int expert, begin, end;
};

// Bounds of expert e's rows.
__device__ __forceinline__ Segment segment_of(const Params& p, int e) {
  if (!p.offsets) return {0, 0, p.rows};
  const int twice = p.pair == kJoin ? 1 : 0;
  const int begin = min(max(p.offsets[e] << twice, 0), p.rows);
  return {e, begin, min(max(p.offsets[e + 1] << twice, begin), p.rows)};
}

// Inclusive sums over the lanes of a wave: within rows of 16 lanes, then the rows' totals.
__device__ __forceinline__ int scan_lanes(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15 to rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31 to rows 2 and 3
  return v;
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
    const int sum = scan_lanes(mine);
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

// Scales of the 128-row block that holds row `row` of expert e's FP8 weight, one for each 128 k.
__device__ __forceinline__ const float* fp8_scales(const Params& p, int e, int row) {
  return p.ws8 + (int64_t(e) * fp8::blocks_of(p.n) + row / fp8::kBlock) * fp8::blocks_of(p.k);
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

// A value as a pair: the nearest bf16, and the nearest to what that leaves (nothing where it is not finite).
__device__ __forceinline__ void split_pair(float v, uint16_t& high, uint16_t& low) {
  high = uint16_t(f32_to_bf16(v));
  const float rest = v - bf16_to_f32(high);
  low = (high & 0x7f80u) == 0x7f80u ? uint16_t(0) : uint16_t(f32_to_bf16(rest));
}

// A product of a pair from those of its halves. Where the high half's is not finite it stands for both: beside an infinite
// weight the low half's is NaN or of either sign.
__device__ __forceinline__ float join_pair(float high, float low) {
  return __builtin_fabsf(high) < __builtin_huge_valf() ? high + low : high;
}

// `part`: rows per workgroup (16, 32 or 64); `groups`: 16-row groups of weight rows (1 or 2).
int launch_stream(const Params& p, int part, int groups, hipStream_t stream);
int launch_rows(const Params& p, hipStream_t stream);
// Tiles of at most `cap` rows x `columns` weight rows (one translation unit per pair of types).
int launch_tiles_bf16(const Params& p, int cap, int columns, hipStream_t stream);
int launch_tiles_mxw(const Params& p, int cap, int columns, hipStream_t stream);
int launch_tiles_mx(const Params& p, int cap, int columns, hipStream_t stream);
int launch_tiles_fp8(const Params& p, int cap, int columns, hipStream_t stream);  // (fp8_tile.h: both operands FP8)
int launch_tiles_w8(const Params& p, int cap, int columns, hipStream_t stream);   // bf16 x, FP8 weights
// A product that leaves or takes pairs (expert_linear.hip).
int launch_pairs(const lf_expert_product& a, Pair pair, hipStream_t stream);
// lf_combine_experts of contiguous fp32 rows (expert_routing.hip).
int combine_f32(const float* rows, int64_t num_rows, const int32_t* positions, const float* weights, int64_t tokens, int32_t top,
                int64_t n, const uint16_t* base, int64_t base_stride, uint16_t* y, int64_t y_stride, hipStream_t stream);

}  // namespace expert
}  // namespace lf
