// Products of a few rows each with many weights (a decode batch over its
// experts): bound by HBM, which has to be kept busy from many workgroups.
//
// A wave owns 16 weight rows over the whole of k, so no sums cross waves; the eight
// waves of a workgroup share the rows of x. Both go through LDS by direct copies of
// whole 128-byte row pieces: fragments loaded straight into the operand layout
// (16 rows, one per lane) take the address unit 64 cycles a load, four times a copy's, and
// bounded the kernel that splits k over its waves (expert_stream.hip) at 3.9 TB/s (24
// tokens over 64 experts, top 4, 4096 x 4096 with SwiGLU: 114 us); this one takes 72, with
// MXFP4 x as well (72-73 with its quantisation).
//
// Each wave streams its weights through a ring of three stages (16 rows x 128 bytes:
// 256 k in MXFP4, 64 in bf16) without meeting the others; x comes in chunks of 8 KiB
// for all waves, two buffers, one barrier a chunk. v_mfma_f32_16x16x32_bf16 (MXFP4
// weights decoded in registers), v_mfma_scale_f32_16x16x128_f8f6f4 where x is MXFP4
// too; the weight is the A operand, up to 16 rows of x the B operand. Lane quarter q
// takes units (of 16 bytes) 2 q and 2 q + 1 of a stage, so its two scales are neighbours.
#include "expert_params.h"
#include "lds_pipeline.h"

namespace lf {
namespace expert {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kRing = 3;
constexpr int kSlot = 16 * 128;       // bytes of a wave's stage
constexpr int kXBytes = 8192;         // bytes of an x chunk
constexpr int kScaleStages = 8;       // stages per unit of scales (2048 k, 64 bytes of a row)
constexpr int kScaleUnit = 16 * 64;   // bytes of a unit of 16 rows


// LDS accesses of the stage loop, each block with its own wait: the compiler would
// wait for every copy in flight before an LDS access of its own.
__device__ __forceinline__ void lds_write16(uint32_t at, const u32x4& v) {
  asm volatile("ds_write_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" ::"v"(at), "v"(v) : "memory");
}
__device__ __forceinline__ uint32_t lds_scales(uint32_t at) {
  uint32_t v;
  asm volatile("ds_read_u16 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(at) : "memory");
  return v;
}
__device__ __forceinline__ void lds_four(u32x4 (&v)[4], const uint32_t (&at)[4], uint32_t base) {
  asm volatile(
      "ds_read_b128 %0, %4\n\t"
      "ds_read_b128 %1, %5\n\t"
      "ds_read_b128 %2, %6\n\t"
      "ds_read_b128 %3, %7\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
      : "v"(at[0] + base), "v"(at[1] + base), "v"(at[2] + base), "v"(at[3] + base)
      : "memory");
}
__device__ __forceinline__ void lds_two(u32x4 (&v)[2], uint32_t a, uint32_t b) {
  asm volatile(
      "ds_read_b128 %0, %2\n\t"
      "ds_read_b128 %1, %3\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1])
      : "v"(a), "v"(b)
      : "memory");
}

// Scales of 64 blocks (2048 k) of 16 rows: lane 4 r + i loads bytes 16 i .. of row
// r's, at any alignment and not past the row (k >= 512), and puts them in place with
// zeros past the end of k (the codes are zero there).
struct ScaleLoad {
  const uint8_t* row;
  u32x4 v;
  int skip;

  __device__ __forceinline__ void load(int unit, int blocks) {
    typedef u32x4 u32x4u __attribute__((aligned(1)));
    const int want = 64 * unit + 16 * (threadIdx.x & 3), from = min(want, blocks - 16);
    skip = min(want - from, 16);
    v = *reinterpret_cast<const u32x4u*>(row + from);
  }
  __device__ __forceinline__ void store(uint32_t area) const { lds_write16(area + (threadIdx.x & 63) * 16, mx::drop_bytes(v, skip)); }
};

template <bool kXMx, bool kWMx>
struct Rows {
  static constexpr int kXStage = kWMx && !kXMx ? 512 : 128;  // bytes of an x row per stage

  // Rows first .. first + 15 of the segment, 128 weight rows of block `block`.
  static __device__ __forceinline__ void run(const Params& p, const Segment& seg, int first, int block, char* lds) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, q = lane >> 4;
    const int count = min(16, seg.end - first);
    const int shift = count <= 4 ? 2 : count <= 8 ? 3 : 4;  // rows of an x chunk, rounded up: 4, 8 or 16
    const int x_piece = kXBytes >> shift;                   // bytes of a row in a chunk
    const int chunk_stages = x_piece / kXStage;
    const int row_bytes_x = kXMx ? p.k / 2 : p.k * 2, row_bytes_w = kWMx ? p.k / 2 : p.k * 2;
    const int stages = (row_bytes_w + 127) / 128, blocks = p.k / mx::kBlock;
    const char* zeros = reinterpret_cast<const char*>(&kZeros);
    char* xbuf = lds;
    char* ring = lds + 2 * kXBytes + wave * kRing * kSlot;
    char* scale_area = lds + 2 * kXBytes + kWaves * kRing * kSlot + wave * kScaleUnit * (kXMx ? 2 : 1);

    // Weight row r of the wave: a column each, or (SwiGLU) gate rows 0 .. 7 and up rows 8 .. 15 of eight columns.
    const int column0 = block * (p.swiglu ? 64 : 128) + wave * (p.swiglu ? 8 : 16);
    auto weight_row = [&](int r) {
      const int64_t base = int64_t(seg.expert) * p.n;
      if (!p.swiglu) return base + min(column0 + r, p.n - 1);
      return base + min(column0 + (r & 7), p.width - 1) + (r >= 8 ? p.width : 0);
    };
    auto x_row = [&](int r) { return x_row_of(p, first + min(r, count - 1)); };

    // Copies: eight rows of a stage each, unit u of row r at u ^ (r & 7). x: a KiB a wave and chunk.
    const int r8 = lane >> 3, wat = ((lane & 7) ^ r8) * 16;
    const char* wsrc[2] = {p.w + weight_row(r8) * row_bytes_w + wat, p.w + weight_row(8 + r8) * row_bytes_w + wat};
    const int xo = wave * 1024 + lane * 16, xr = xo >> (13 - shift), xu = (xo & (x_piece - 1)) >> 4;
    const int xat = ((xu & ~7) | ((xu ^ xr) & 7)) * 16;
    const char* xsrc = p.x + x_row(xr) * p.x_row + xat;
    auto copy_w = [&](int st) {
      const bool in = st * 128 + wat < row_bytes_w;
      char* slot = ring + st % kRing * kSlot;
      copy16(in ? wsrc[0] + st * 128 : zeros, slot);
      copy16(in ? wsrc[1] + st * 128 : zeros, slot + 1024);
    };
    auto copy_x = [&](int ch) {
      const bool in = ch * x_piece + xat < row_bytes_x;
      copy16(in ? xsrc + int64_t(ch) * x_piece : zeros, xbuf + (ch & 1) * kXBytes + wave * 1024);
    };
    ScaleLoad ws, xs;
    if constexpr (kWMx) {
      ws.row = p.ws + weight_row(lane >> 2) * blocks;
      ws.load(0, blocks);
    }
    if constexpr (kXMx) {
      xs.row = p.xs + x_row(lane >> 2) * blocks;
      xs.load(0, blocks);
    }
    copy_x(0);
    copy_w(0);
    copy_w(1);

    // Reads: units 2 q and 2 q + 1 of weight row c, and what they meet of x row c.
    const uint32_t ring_at = lds_addr(ring), x_at = lds_addr(xbuf), scale_at = lds_addr(scale_area);
    const uint32_t wread[2] = {uint32_t(c * 128 + ((2 * q) ^ (c & 7)) * 16), uint32_t(c * 128 + ((2 * q + 1) ^ (c & 7)) * 16)};
    const int xc = min(c, count - 1);
    uint32_t xread[2][4];  // [unit][8 k of it], of MXFP4 and bf16-beside-bf16 x only [unit][0]
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        xread[s][j] = uint32_t(xc * x_piece + (((kXStage == 512 ? 4 * (2 * q + s) + j : 2 * q + s) ^ (xc & 7)) * 16));
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int st = 0; st < stages; ++st) {
      // Stage st has arrived, and the x chunk that starts with it (copied before it).
      wait_vm<2>();
      if (kWMx && st % kScaleStages == 0) {
        ws.store(scale_at);
        ws.load(st / kScaleStages + 1, blocks);
        if constexpr (kXMx) {
          xs.store(scale_at + kScaleUnit);
          xs.load(st / kScaleStages + 1, blocks);
        }
      }
      if (st % chunk_stages == 0) {
        barrier_only();
        copy_x(st / chunk_stages + 1);
      }
      copy_w(st + 2);  // (its slot's reads are done)
      const uint32_t slot = ring_at + st % kRing * kSlot;
      const uint32_t x_base = x_at + (st / chunk_stages & 1) * kXBytes + st % chunk_stages * kXStage;
      uint32_t wscale = 0, xscale = 0;
      if constexpr (kWMx) wscale = lds_scales(scale_at + c * 64 + st % kScaleStages * 8 + 2 * q);
      if constexpr (kXMx) xscale = lds_scales(scale_at + kScaleUnit + xc * 64 + st % kScaleStages * 8 + 2 * q);
      if constexpr (kXStage == 512) {
        u32x4 w[2];
        lds_two(w, slot + wread[0], slot + wread[1]);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          u32x4 x[4];
          lds_four(x, xread[s], x_base);
          const float scale = mx::scale_f32(s == 0 ? wscale & 0xffu : wscale >> 8);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc = mfma16(vec_bf16x8(mx::decode8(w[s][j], scale)), vec_bf16x8(x[j]), acc);
        }
      } else {
        u32x4 v[4];
        const uint32_t at[4] = {slot + wread[0], slot + wread[1], x_base + xread[0][0], x_base + xread[1][0]};
        lds_four(v, at, 0);
        if constexpr (kXMx) {
          acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx::operand(v[0]), mx::operand(v[2]), acc, 4, 4, 0, wscale, 0, xscale);
          acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx::operand(v[1]), mx::operand(v[3]), acc, 4, 4, 1, wscale, 1, xscale);
        } else {
          acc = mfma16(vec_bf16x8(v[0]), vec_bf16x8(v[2]), acc);
          acc = mfma16(vec_bf16x8(v[1]), vec_bf16x8(v[3]), acc);
        }
      }
    }

    // acc[e]: weight row 4 q + e, x row c.
    const uint16_t* bias = p.bias ? p.bias + int64_t(seg.expert) * p.n : nullptr;
    const int column = column0 + (p.swiglu ? 4 * (q & 1) : 4 * q);
    float out[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = min(column + e, p.width - 1) + (p.swiglu && q >= 2 ? p.width : 0);
      out[e] = acc[e] + (bias ? bf16_to_f32(bias[at]) : 0.f);
      if (p.swiglu) out[e] = silu_mul_f32(out[e], __shfl_xor(out[e], 32, 64));  // (lanes of gate rows: the others' are not stored)
    }
    // Copies for stages past the end are on their way, and other waves still read x.
    wait_vm<0>();
    barrier_only();
    if (c >= count || (p.swiglu && q >= 2)) return;
    uint16_t* y = p.y + int64_t(first + c) * p.y_stride + column;
    if (p.y_vec && column + 4 <= p.width) {
      *reinterpret_cast<u32x2*>(y) = u32x2{pack_bf16x2(out[0], out[1]), pack_bf16x2(out[2], out[3])};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (column + e < p.width) y[e] = uint16_t(f32_to_bf16(out[e]));
    }
  }
};

// Grid: blocks of 128 weight rows x experts that have rows.
template <bool kXMx, bool kWMx>
__global__ __launch_bounds__(kThreads, 4) void rows_kernel(Params p) {
  extern __shared__ char lds[];
  int index = blockIdx.y;
  const Segment seg = find_segment(p, index, [](const Segment& s) { return s.end > s.begin ? 1 : 0; });
  for (int first = seg.begin; first < seg.end; first += 16) Rows<kXMx, kWMx>::run(p, seg, first, blockIdx.x, lds);
}

template <bool kXMx, bool kWMx>
int launch_types(const Params& p, hipStream_t stream) {
  const int segments = p.offsets ? (p.experts < p.rows ? p.experts : p.rows) : 1;
  const int columns = p.swiglu ? 64 : 128;
  const dim3 grid(unsigned((p.width + columns - 1) / columns), unsigned(segments));
  const unsigned lds = 2 * kXBytes + kWaves * (kRing * kSlot + kScaleUnit * (kXMx ? 2 : 1));
  hipLaunchKernelGGL((rows_kernel<kXMx, kWMx>), grid, dim3(kThreads), lds, stream, p);
  LF_HIP(hipGetLastError());
  return kOk;
}

}  // namespace

int launch_rows(const Params& p, hipStream_t stream) {
  if (p.xs) return launch_types<true, true>(p, stream);
  return p.ws ? launch_types<false, true>(p, stream) : launch_types<false, false>(p, stream);
}

}  // namespace expert
}  // namespace lf
