// Products of few rows with large weights (decode): every weight byte is read
// once and multiplied by the handful of rows of its expert, so the kernel is
// bound by HBM, at the smallest sizes by latency.
//
// A workgroup owns 16 kF weight rows of one expert over the whole of k, and up to 64 of
// the expert's rows (16 or 32 where that leaves CUs idle: the weights then come from L2 again); its
// eight waves take every eighth step of 128 k, so that together they read 512
// (MXFP4) or 2048 (bf16) consecutive bytes of a row. Weights go from memory
// straight into the operand layout of the matrix instructions (nobody else
// needs them): v_mfma_f32_16x16x32_bf16 on MXFP4 weights decoded in registers
// or on bf16 ones, v_mfma_scale_f32_16x16x128_f8f6f4 where x is MXFP4 too.
// The weight is the A operand, 16 rows of x the B operand. The order of k
// within a step is free as long as both operands agree on it: with MXFP4 weights
// lane quarter q holds block q of the step (32 k, one scale), else 8 k of each.
// The waves' partial sums meet in LDS, in a fixed order.
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
template <bool kMx, int kN>
struct Rows {
  u32x4 v[kN][kMx ? 1 : 4];
  uint32_t scale[kMx ? kN : 1];
};

struct RowPtr {
  const char* v;
  const uint8_t* s;
};

// kBlocked: a lane's k of a step is block q (else 8 k of each block).
template <bool kMx, bool kBlocked, int kN>
__device__ __forceinline__ void load_rows(const Params& p, const RowPtr (&row)[kN], int step, int q, Rows<kMx, kN>& r) {
  const int k0 = step * kStep;
  const bool whole = k0 + kStep <= p.k;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    if constexpr (kMx) {
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

template <bool kXMx, bool kWMx, int kF, int kT>
__device__ __forceinline__ void contract(const Rows<kWMx, kF>& w, const Rows<kXMx, kT>& x, f32x4 (&acc)[kF][kT]) {
#pragma unroll
  for (int f = 0; f < kF; ++f) {
    if constexpr (kXMx) {
#pragma unroll
      for (int t = 0; t < kT; ++t)
        acc[f][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx::operand(w.v[f][0]), mx::operand(x.v[t][0]), acc[f][t],
                                                                     4, 4, 0, w.scale[f], 0, x.scale[t]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 a;
        if constexpr (kWMx)
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
template <bool kXMx, bool kWMx, int kF, int kT>
__device__ __forceinline__ void stream_rows(const Params& p, const Segment& seg, int first, int block, float* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = lane & 15, q = lane >> 4;
  const int64_t w_row = kWMx ? p.k / 2 : int64_t(p.k) * 2;
  const int blocks = p.k / mx::kBlock;
  RowPtr w[kF], x[kT];
#pragma unroll
  for (int f = 0; f < kF; ++f) {
    const int64_t row = int64_t(seg.expert) * p.n + weight_row<kF>(p, block, 16 * f + c);
    w[f] = {p.w + row * w_row, kWMx ? p.ws + row * blocks : nullptr};
  }
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    const int64_t row = x_row_of(p, min(first + 16 * t + c, seg.end - 1));
    x[t] = {p.x + row * p.x_row, kXMx ? p.xs + row * blocks : nullptr};
  }
  f32x4 acc[kF][kT];
#pragma unroll
  for (int f = 0; f < kF; ++f)
#pragma unroll
    for (int t = 0; t < kT; ++t) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Steps requested together: as many as fit 128 registers, two workgroups a CU (an
  // MXFP4 row takes nine with its scale and addresses).
  constexpr int kRegs = (kWMx ? 9 : 16) * kF + (kXMx ? 9 : 16) * kT;
  constexpr int kDepth = kRegs <= 18 ? 4 : kRegs <= 36 ? 2 : 1;
  const int steps = (p.k + kStep - 1) / kStep;
  for (int s = wave; s < steps; s += kDepth * kWaves) {
    Rows<kWMx, kF> wr[kDepth];
    Rows<kXMx, kT> xr[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (d && s + d * kWaves >= steps) break;
      load_rows<kWMx, kWMx, kF>(p, w, s + d * kWaves, q, wr[d]);
      load_rows<kXMx, kWMx, kT>(p, x, s + d * kWaves, q, xr[d]);
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (d && s + d * kWaves >= steps) break;
      contract<kXMx, kWMx, kF, kT>(wr[d], xr[d], acc);
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
    const float v = p.swiglu ? silu_mul_f32(total(r, row), total(r + 8 * kF, row)) : total(r, row);
    p.y[int64_t(first + row) * p.y_stride + n] = uint16_t(f32_to_bf16(v));
  }
}

// Grid: column blocks x passes of `part` rows (16, 32 or 64) of the experts (y, then z).
// (A loop over passes in the kernel takes its registers past 128, into scratch.)
template <bool kXMx, bool kWMx, int kF>
__global__ __launch_bounds__(kThreads, 4) void stream_kernel(Params p, int part) {
  __shared__ float red[kWaves * kF * kRowTiles * 256];
  int index = int(blockIdx.z * gridDim.y + blockIdx.y);
  Segment seg = find_segment(p, index, [&](const Segment& s) { return (s.end - s.begin + part - 1) / part; });
  if (seg.end <= seg.begin) return;
  seg.begin += index * part;
  seg.end = min(seg.end, seg.begin + part);
  const int rows = seg.end - seg.begin;
  if (rows <= 16) {
    stream_rows<kXMx, kWMx, kF, 1>(p, seg, seg.begin, blockIdx.x, red);
  } else if (rows <= 32) {
    stream_rows<kXMx, kWMx, kF, 2>(p, seg, seg.begin, blockIdx.x, red);
  } else {
    stream_rows<kXMx, kWMx, kF, 4>(p, seg, seg.begin, blockIdx.x, red);
  }
}

template <bool kXMx, bool kWMx>
int launch_types(const Params& p, int part, int groups, hipStream_t stream) {
  // At most: a pass more than whole ones for every expert that has a row.
  const int64_t used = p.offsets ? (p.experts < p.rows ? p.experts : p.rows) : 1;
  const int64_t passes = (p.rows + used * (part - 1)) / part;
  constexpr int64_t kMostY = 65535;
  const int64_t columns = (p.swiglu ? 8 : 16) * groups;
  const dim3 grid(unsigned((p.width + columns - 1) / columns), unsigned(passes < kMostY ? passes : kMostY),
                  unsigned((passes + kMostY - 1) / kMostY)),
      threads(kThreads);
  if (groups == 2)
    hipLaunchKernelGGL((stream_kernel<kXMx, kWMx, 2>), grid, threads, 0, stream, p, part);
  else
    hipLaunchKernelGGL((stream_kernel<kXMx, kWMx, 1>), grid, threads, 0, stream, p, part);
  LF_HIP(hipGetLastError());
  return kOk;
}

}  // namespace

int launch_stream(const Params& p, int part, int groups, hipStream_t stream) {
  if (p.xs) return launch_types<true, true>(p, part, groups, stream);
  return p.ws ? launch_types<false, true>(p, part, groups, stream) : launch_types<false, false>(p, part, groups, stream);
}

}  // namespace expert
}  // namespace lf
