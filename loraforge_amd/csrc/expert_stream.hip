// Products of few rows with large weights (decode): every weight byte is read
// once and multiplied by the handful of rows of its expert, so the kernel is
// bound by HBM, at the smallest sizes by latency.
//
// A workgroup owns 16 kF weight rows of one expert over the whole of k, and up to 64 of
// the expert's rows (16 or 32 where that leaves CUs idle: the weights then come from L2 again); its
// eight waves take every eighth step of 128 k, so that together they read 512
// (MXFP4) or 2048 (bf16) consecutive bytes of a row. Weights go from memory
// straight into the operand layout of the matrix instructions (nobody else
// needs them): v_mfma_f32_16x16x32_bf16 on MXFP4 or FP8 weights decoded in registers
// or on bf16 ones, v_mfma_scale_f32_16x16x128_f8f6f4 where x is MXFP4 too, its form without
// scales where both are FP8. The weight is the A operand, 16 rows of x the B operand. The order of k
// within a step is free as long as both operands agree on it: with MXFP4 and FP8 weights
// lane quarter q holds block q of the step (32 k, one MXFP4 scale), else 8 k of each. An FP8
// scale is that of a whole step: a step's products are summed from zero and added
// to the sums times x's and the weight's scale, in fp32.
// The waves' partial sums meet in LDS, in a fixed order.
// FP8 weights: a row of 4096 x 4096 5.8 us (16.8 MB, 2.9 TB/s: a launch, two loads' latency, as a wave asks for its four
// steps in pairs, the join); 24 tokens over 64
// experts, top 4, 4096 x 4096 with SwiGLU 136-149 (727 MB fetched, 4.9-5.3 TB/s; a wave for 16 weight rows 158).
#include "expert_params.h"

namespace lf {
namespace expert {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kStep = 128;   // k per step
constexpr int kRowTiles = 4;  // most 16-row tiles of a pass


__device__ __forceinline__ u32x4 load16(const char* p) { return *reinterpret_cast<const u32x4*>(p); }

// Weight row of the workgroup's local row r (SwiGLU: the first half are gate
// rows, the second the up rows of the same columns).
template <int kF>
__device__ __forceinline__ int weight_row(const Params& p, int block, int r) {
  if (!p.swiglu) return min(block * 16 * kF + r, p.n - 1);
  const int column = min(block * 8 * kF + (r & (8 * kF - 1)), p.width - 1);
  return column + (r >= 8 * kF ? p.width : 0);
}

// What one step needs of kN operand rows of a lane.
template <int kType, int kN>
struct Rows {
  u32x4 v[kN][kType == kMxfp4 ? 1 : kType == kFp8 ? 2 : 4];
  uint32_t scale[kType == kBf16 ? 1 : kN];  // a byte, or a float's bits
};

struct RowPtr {
  const char* v;
  const uint8_t* s;   // MXFP4
  const float* s8;    // FP8: of the rows that the lane's sums belong to
};

// kBlocked: a lane's k of a step is block q (else 8 k of each block).
template <int kType, bool kBlocked, int kN>
__device__ __forceinline__ void load_rows(const Params& p, const RowPtr (&row)[kN], int step, int q, Rows<kType, kN>& r) {
  const int k0 = step * kStep;
  const bool whole = k0 + kStep <= p.k;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    if constexpr (kType == kFp8) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int at = k0 + 32 * q + 16 * j;
        r.v[i][j] = load16(whole || at < p.k ? row[i].v + at : reinterpret_cast<const char*>(&kZeros));
      }
      r.scale[i] = __float_as_uint(row[i].s8[step]);
    } else if constexpr (kType == kMxfp4) {
      const int block = k0 / mx::kBlock + q;
      const bool in = whole || block < p.k / mx::kBlock;
      r.v[i][0] = load16(in ? row[i].v + block * 16 : reinterpret_cast<const char*>(&kZeros));
      r.scale[i] = *(in ? row[i].s + block : reinterpret_cast<const uint8_t*>(&kZeros));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = k0 + (kBlocked ? 32 * q + 8 * j : 32 * j + 8 * q);
        r.v[i][j] = load16(whole || at < p.k ? row[i].v + at * 2 : reinterpret_cast<const char*>(&kZeros));
      }
    }
  }
}

template <int kX, int kW, int kF, int kT>
__device__ __forceinline__ void contract(const Rows<kW, kF>& w, const Rows<kX, kT>& x, f32x4 (&acc)[kF][kT]) {
#pragma unroll
  for (int f = 0; f < kF; ++f) {
    if constexpr (kW == kFp8) {
      f32x4 sum[kT];
      if constexpr (kX == kFp8) {
#pragma unroll
        for (int t = 0; t < kT; ++t) sum[t] = fp8::mfma16(fp8::operand(w.v[f][0], w.v[f][1]), fp8::operand(x.v[t][0], x.v[t][1]));
      } else {
#pragma unroll
        for (int t = 0; t < kT; ++t) sum[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 codes = w.v[f][j >> 1];
          const bf16x8 a = __builtin_bit_cast(bf16x8, fp8::decode8(codes[j % 2 * 2], codes[j % 2 * 2 + 1]));
#pragma unroll
          for (int t = 0; t < kT; ++t) sum[t] = lf::mfma16(a, __builtin_bit_cast(bf16x8, x.v[t][j]), sum[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        const float s = __uint_as_float(w.scale[f]) * (kX == kFp8 ? __uint_as_float(x.scale[kX == kFp8 ? t : 0]) : 1.0f);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[f][t][e] = fmaf(s, sum[t][e], acc[f][t][e]);
      }
    } else if constexpr (kX == kMxfp4) {
#pragma unroll
      for (int t = 0; t < kT; ++t)
        acc[f][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx::operand(w.v[f][0]), mx::operand(x.v[t][0]), acc[f][t],
                                                                     4, 4, 0, w.scale[f], 0, x.scale[t]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 a;
        if constexpr (kW == kMxfp4)
          a = mx::decode8(w.v[f][0][j], mx::scale_f32(w.scale[f]));
        else
          a = w.v[f][j];
#pragma unroll
        for (int t = 0; t < kT; ++t)
          acc[f][t] = mfma16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, x.v[t][j]), acc[f][t]);
      }
    }
  }
}

// Rows first .. first + 16 kT - 1 (below the segment's end) of the workgroup's columns.
template <int kX, int kW, int kF, int kT>
__device__ __forceinline__ void stream_rows(const Params& p, const Segment& seg, int first, int block, float* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & 15, q = lane >> 4;
  const int64_t w_row = kW == kMxfp4 ? p.k / 2 : kW == kFp8 ? p.k : int64_t(p.k) * 2;
  const int blocks = p.k / mx::kBlock;
  RowPtr w[kF], x[kT];
#pragma unroll
  for (int f = 0; f < kF; ++f) {
    const int64_t row = int64_t(seg.expert) * p.n + weight_row<kF>(p, block, 16 * f + c);
    w[f] = {p.w + row * w_row, kW == kMxfp4 ? p.ws + row * blocks : nullptr,
            kW == kFp8 ? fp8_scales(p, seg.expert, weight_row<kF>(p, block, 16 * f + 4 * q)) : nullptr};
  }
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    const int64_t row = x_row_of(p, min(first + 16 * t + c, seg.end - 1));
    x[t] = {p.x + row * p.x_row, kX == kMxfp4 ? p.xs + row * blocks : nullptr,
            kX == kFp8 ? p.xs8 + row * fp8::blocks_of(p.k) : nullptr};
  }
  f32x4 acc[kF][kT];
#pragma unroll
  for (int f = 0; f < kF; ++f)
#pragma unroll
    for (int t = 0; t < kT; ++t) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Steps requested together: as many as fit 128 registers, two workgroups a CU (an
  // MXFP4 row takes nine with its scale and addresses, an FP8 one thirteen).
  constexpr int kRegsOf[3] = {16, 9, 13};
  constexpr int kRegs = kRegsOf[kW] * kF + kRegsOf[kX] * kT;
  constexpr int kDepth = kRegs <= 18 ? 4 : kRegs <= 36 ? 2 : 1;
  const int steps = (p.k + kStep - 1) / kStep;
  for (int s = wave; s < steps; s += kDepth * kWaves) {
    Rows<kW, kF> wr[kDepth];
    Rows<kX, kT> xr[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (d && s + d * kWaves >= steps) break;
      load_rows<kW, kW != kBf16, kF>(p, w, s + d * kWaves, q, wr[d]);
      load_rows<kX, kW != kBf16, kT>(p, x, s + d * kWaves, q, xr[d]);
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (d && s + d * kWaves >= steps) break;
      contract<kX, kW, kF, kT>(wr[d], xr[d], acc);
    }
  }

  // Partial sums as [wave][feature tile][row tile][row][feature].
#pragma unroll
  for (int f = 0; f < kF; ++f)
#pragma unroll
    for (int t = 0; t < kT; ++t)
      *reinterpret_cast<f32x4*>(red + ((wave * kF + f) * kT + t) * 256 + c * 16 + 4 * q) = acc[f][t];
  __syncthreads();
  const uint16_t* bias = p.bias ? p.bias + int64_t(seg.expert) * p.n : nullptr;
  auto total = [&](int r, int row) {  // local weight row r, row of the pass
    float sum = 0.f;
    const float* at = red + ((r >> 4) * kT + (row >> 4)) * 256 + (row & 15) * 16 + (r & 15);
#pragma unroll
    for (int v = 0; v < kWaves; ++v) sum += at[v * kF * kT * 256];
    return bias ? sum + bf16_to_f32(bias[weight_row<kF>(p, block, r)]) : sum;
  };
  const int columns = p.swiglu ? 8 * kF : 16 * kF;
  const int shift = p.swiglu ? 3 : 4;
  for (int i = threadIdx.x; i < columns * 16 * kT; i += kThreads) {
    const int r = (i & (columns - 1)), row = (i >> shift) / kF;
    const int n = block * columns + r;
    if (first + row >= seg.end || n >= p.width) continue;
    if (p.pair == kJoin) {  // (a pair's rows are in one pass)
      if (!(row & 1)) reinterpret_cast<float*>(p.y)[int64_t((first + row) >> 1) * p.y_stride + n] = join_pair(total(r, row), total(r, row + 1));
      continue;
    }
    const float v = p.swiglu ? silu_mul_f32(total(r, row), total(r + 8 * kF, row)) : total(r, row);
    if (p.pair == kSplit) {
      uint16_t* y = p.y + int64_t(first + row) * 2 * p.y_stride + n;
      split_pair(v, y[0], y[p.y_stride]);
    } else {
      p.y[int64_t(first + row) * p.y_stride + n] = uint16_t(f32_to_bf16(v));
    }
  }
}

// Rows of a pass. (32 weight rows in FP8 beside 64 rows, whose products of a step are summed apart from the sums so far, take
// more than the 128 registers of a wave: passes of 32 then.)
template <int kW, int kF>
constexpr int kMostRows = kW == kFp8 && kF == 2 ? 32 : 64;

// Grid: column blocks x passes of `part` rows (16, 32 or 64) of the experts (y, then z).
// (A loop over passes in the kernel takes its registers past 128, into scratch.)
template <int kX, int kW, int kF>
__global__ __launch_bounds__(kThreads, 4) void stream_kernel(Params p, int part) {
  __shared__ float red[kWaves * kF * kRowTiles * 256];
  int index = int(blockIdx.z * gridDim.y + blockIdx.y);
  Segment seg = find_segment(p, index, [&](const Segment& s) { return (s.end - s.begin + part - 1) / part; });
  if (seg.end <= seg.begin) return;
  seg.begin += index * part;
  seg.end = min(seg.end, seg.begin + part);
  const int rows = seg.end - seg.begin;
  if (rows <= 16) {
    stream_rows<kX, kW, kF, 1>(p, seg, seg.begin, blockIdx.x, red);
  } else if (rows <= 32) {
    stream_rows<kX, kW, kF, 2>(p, seg, seg.begin, blockIdx.x, red);
  } else if constexpr (kMostRows<kW, kF> > 32) {
    stream_rows<kX, kW, kF, 4>(p, seg, seg.begin, blockIdx.x, red);
  }
}

template <int kX, int kW>
int launch_types(const Params& p, int part, int groups, hipStream_t stream) {
  if (groups == 2 && part > kMostRows<kW, 2>) part = kMostRows<kW, 2>;
  // At most: a pass more than whole ones for every expert that has a row.
  const int64_t used = p.offsets ? (p.experts < p.rows ? p.experts : p.rows) : 1;
  const int64_t passes = (p.rows + used * (part - 1)) / part;
  constexpr int64_t kMostY = 65535;
  const int64_t columns = (p.swiglu ? 8 : 16) * groups;
  const dim3 grid(unsigned((p.width + columns - 1) / columns), unsigned(passes < kMostY ? passes : kMostY),
                  unsigned((passes + kMostY - 1) / kMostY)),
      threads(kThreads);
  if (groups == 2)
    hipLaunchKernelGGL((stream_kernel<kX, kW, 2>), grid, threads, 0, stream, p, part);
  else
    hipLaunchKernelGGL((stream_kernel<kX, kW, 1>), grid, threads, 0, stream, p, part);
  LF_HIP(hipGetLastError());
  return kOk;
}

}  // namespace

int launch_stream(const Params& p, int part, int groups, hipStream_t stream) {
  if (p.ws8)
    return p.xs8 ? launch_types<kFp8, kFp8>(p, part, groups, stream) : launch_types<kBf16, kFp8>(p, part, groups, stream);
  if (p.xs) return launch_types<kMxfp4, kMxfp4>(p, part, groups, stream);
  return p.ws ? launch_types<kBf16, kMxfp4>(p, part, groups, stream) : launch_types<kBf16, kBf16>(p, part, groups, stream);
}

}  // namespace expert
}  // namespace lf
