// Products of many rows (prefill): MFMA tiles of up to 256 rows x 64 kJ weight rows.
//
// Four waves, one per SIMD, in a 2 x 2 arrangement: a wave owns 32 kI rows x
// 32 kJ weight rows (v_mfma_f32_32x32x16_bf16, or v_mfma_scale_f32_32x32x64_f8f6f4
// where both operands are MXFP4; the weight is the A operand). Both operands
// go through LDS by direct copies, in stages of 128 bytes of every x row (64 k in
// bf16, 256 k in MXFP4); a ring of kSlots stages, the copies of a stage
// issued as soon as its slot is free. A stage is four sub-steps; the operands
// of a sub-step are read while the one before it is multiplied. MXFP4 weights
// beside bf16 x are decoded in registers (four conversions per eight weights,
// exact), so they cost a quarter of the copies and no pass of their own.
//
// The order of k within a stage is free as long as both operands agree: lane
// half h of sub-step s takes unit 4 h + s (16 bytes), so that an MXFP4 lane's
// blocks of a stage are consecutive and its scales one dword (byte s for
// sub-step s), and beside bf16 x a lane's 32 weights of a stage are one block.
//
// An expert's rows are cut into steps of 64, and those into as few tiles (of up to four)
// as can be, as even as can be, so that an expert costs what its rows need: the body
// is chosen by the tile's rows. (With tiles of one height, 300 rows ran as 384.)
//
// What bounds it, by clock stamps in a copy that records them. 4096 x 12288 x 4096, 768 tiles
// of 256 x 256, three a CU; a stage's 64 matrix instructions of 32 clocks are 2048 of its clocks:
//
//                clocks of a tile: start   loop              end     all      matrix  clock     product
//   bf16                           9.1k    150.9k (64 x 2358)  10.7k   170.7k   77 %    1.62 GHz  326-346 us
//   MXFP4 weights                  7.5k    185.2k (64 x 2894)  10.7k   203.4k   64 %    1.88 GHz  331-340 us
//   MXFP4 both                     7.1k    44.9k (16 x 2804)   10.9k   62.8k    52 %    1.65 GHz  111-112 us
//
// (Start: segment, addresses, first copies; end: the epilogue.) In bf16 the loop, which the matrix
// instructions fill to 87 %, at a clock that falls under load (2.4 GHz without): MXFP4 weights cost
// a fifth more clocks and the same time. 1.26 PFLOP/s (a library's product of 8192 cubed reaches 1.23).
// With MXFP4 on both sides the loop is a quarter as long and start and end are 29 % of
// a tile: 3.7 PFLOP/s. A workgroup takes all of a CU's LDS whatever its tile, so small
// tiles have nothing beside them to cover their LDS reads; few tiles leave CUs idle.
#pragma once

#include "expert_params.h"
#include "lds_pipeline.h"

namespace lf {
namespace expert {
namespace tile {

constexpr int kThreads = 256;
constexpr int kLds = 160 * 1024;
constexpr int kSubSteps = 4;
constexpr int kXRow = 128;  // bytes of an x row per stage

template <bool kXMx, bool kWMx, int kI, int kJ>
struct Shape {
  static constexpr bool kDecode = kWMx && !kXMx;           // MXFP4 weights for bf16 x
  static constexpr int kStageK = kXMx ? 256 : 64;
  static constexpr int kWRow = kDecode ? 32 : 128;         // bytes of a weight row per stage
  // (Whole copies of all waves: of 64 or 192 rows of 32 bytes 64 go twice.)
  static constexpr int kXBytes = 64 * kI * kXRow, kWBytes = (64 * kJ * kWRow + 4095) / 4096 * 4096;
  static constexpr int kStage = kXBytes + kWBytes;
  // (Deeper for small tiles of MXFP4 x, whose two stages a unit of scales are soon
  // through: 1024 tokens over 64 experts 4096 x 2048 in 64 x 128 tiles 165 -> 140 us;
  // bf16 x gains nothing, its small tiles wait for LDS reads.)
  static constexpr int kMost = kXMx && kI * kJ <= 3 ? 8 : 4;
  // Scales go through LDS in units. MXFP4 x: 16 bytes (two stages) of every x and weight
  // row; beside bf16 x a round of the ring, up to 8 bytes of every weight row, two buffers.
  // (A place for each thread's row, also where there are fewer rows:
  // a condition around the store costs more than the store, above all among matrix instructions.)
  static constexpr int kUnitBytes = kXMx ? 16 : 8;
  static constexpr int kXUnits = kThreads * 16;  // bytes
  static constexpr int kScaleBytes = kXMx ? 2 * kXUnits : kWMx ? 2 * kUnitBytes * kThreads : 0;
  static constexpr int kFit = (kLds - kScaleBytes) / kStage < kMost ? (kLds - kScaleBytes) / kStage : kMost;
  static constexpr int kSlots = kXMx ? kFit / 2 * 2 : kFit;
  static_assert(kSlots >= 2, "two stages have to fit");
  static constexpr int kXCopies = kXBytes / 4096, kWCopies = kWBytes / 4096;  // per wave
  static constexpr int kLoads = kXCopies + kWCopies;
};

// A lane's scales: with MXFP4 x its four blocks of every fragment row, beside bf16 x its one block.
struct Scales {
  u32x2 x[4], w[4];  // MXFP4 x: of both stages of a unit
};

// The operands of one sub-step.
template <int kI, int kJ>
struct Frags {
  u32x4 x[kI], w[kJ];
};

__device__ __forceinline__ void reads_done() { __builtin_amdgcn_s_waitcnt(0xC07F); }  // lgkmcnt(0), which the compiler sees
__device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0); }

// Bias, activation, rounding and stores. Each wave passes its sums through LDS of
// its own, two fragment rows (64 rows of the tile) at a time: acc[i][j][4 g + e] is
// row c of fragment row i and weight row 8 g + 4 h + e of fragment j, and in LDS a
// row's columns follow each other, so that eight lanes or more store whole cache
// lines and the code is short (an unrolled epilogue straight from the
// registers took longer to fetch than to run). For the same reason kPair (a Pair, or kAnyPair: as p.pair says) is a
// parameter: with the stores of its three forms beside each other 1024 rows of 11008 x 4096, MXFP4 both, took 41 us, and
// 33 without (rows of the last columns' tiles are stored a value at a time, and these tiles end last).
constexpr int kAnyPair = -1;
template <int kI, int kJ, bool kSwiglu, int kPair>
__device__ __forceinline__ void finish(const Params& p, const f32x16 (&acc)[kI][kJ], char* lds, int expert, int first, int count,
                                       int nt) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  constexpr int kRowBytes = 32 * kJ * 4 + 16;             // (padded: rows start at other banks)
  constexpr int kColumns = kSwiglu ? 16 * kJ : 32 * kJ;   // output columns of the wave
  constexpr int kParts = kColumns / 8;  // lanes that share a row (of kLanes, a power of two)
  constexpr int kLanes = kParts <= 2 ? 2 : kParts <= 4 ? 4 : kParts <= 8 ? 8 : 16, kRows = 64 / kLanes;
  char* mine = lds + wave * 64 * kRowBytes;
  const int wm = wave & 1, wn = wave >> 1, c = lane & 31;
  const bool idle = lane % kLanes >= kParts;
  const int part = idle ? 0 : lane % kLanes, in_row = lane / kLanes;
  // With SwiGLU eight columns are half of a fragment's gate values, their up values 16 on.
  const int local = kSwiglu ? part / 2 * 32 + part % 2 * 8 : part * 8;
  const int col = (nt * 2 + wn) * kColumns + part * 8;
  float add[8], add_up[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) add[e] = add_up[e] = 0.f;
  if (p.bias) {
    const uint16_t* bias = p.bias + int64_t(expert) * p.n;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = min(col + e, p.width - 1);
      add[e] = bf16_to_f32(bias[at]);
      if (kSwiglu) add_up[e] = bf16_to_f32(bias[at + p.width]);
    }
  }
  const bool vec = p.y_vec && col + 8 <= p.width;
  const int pair = kPair == kAnyPair ? p.pair : kPair;
  const bool all_vec = pair == kSingle && __ballot(!vec) == 0;
  // Eight output columns of staged row r.
  auto values = [&](int r, float (&out)[8]) {
    const f32x4* v = reinterpret_cast<const f32x4*>(mine + r * kRowBytes + local * 4);
    const f32x4 half[2] = {v[0], v[1]};
    f32x4 up[2];
    if (kSwiglu) up[0] = v[4], up[1] = v[5];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a = half[e >> 1][(e & 1) * 2] + add[2 * e], b = half[e >> 1][(e & 1) * 2 + 1] + add[2 * e + 1];
      if (kSwiglu) {
        a = silu_mul_f32(a, up[e >> 1][(e & 1) * 2] + add_up[2 * e]);
        b = silu_mul_f32(b, up[e >> 1][(e & 1) * 2 + 1] + add_up[2 * e + 1]);
      }
      out[2 * e] = a;
      out[2 * e + 1] = b;
    }
  };
  auto output = [&](int r) {
    float v[8];
    values(r, v);
    return u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
  };
#pragma unroll
  for (int two = 0; two < (kI + 1) / 2; ++two) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (2 * two + i < kI) {
            const f32x16& a = acc[2 * two + i][j];
            *reinterpret_cast<f32x4*>(mine + (32 * i + c) * kRowBytes + (32 * j + 8 * g + 4 * h) * 4) =
                f32x4{a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]};
          }
    const int staged = min(2, kI - 2 * two) * 32;
    auto place = [&](int r) { return (2 * two + (r >> 5)) * 64 + 32 * wm + (r & 31); };
    if (all_vec) {
      constexpr int kTogether = 32 / kRows < 4 ? 32 / kRows : 4;  // rows whose reads go out together
#pragma unroll 1
      for (int r0 = in_row; r0 < staged; r0 += kTogether * kRows) {
        u32x4 o[kTogether];
#pragma unroll
        for (int k = 0; k < kTogether; ++k) o[k] = output(r0 + k * kRows);
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
          const int row = place(r0 + k * kRows);
          if (row < count && !idle) *reinterpret_cast<u32x4*>(p.y + int64_t(first + row) * p.y_stride + col) = o[k];
        }
      }
    } else {
#pragma unroll 1
      for (int r = in_row; r < staged; r += kRows) {
        if (pair == kSingle) {
          const u32x4 o = output(r);
          uint16_t* y = p.y + int64_t(first + place(r)) * p.y_stride + col;
          if (place(r) >= count || idle) continue;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (col + e < p.width) y[e] = uint16_t(o[e >> 1] >> (16 * (e & 1)));
          continue;
        }
        const int64_t row = first + place(r);
        if (place(r) >= count || idle || (pair == kJoin && (r & 1))) continue;
        float v[8];
        values(r, v);
        if (pair == kJoin) {  // (a pair's rows are in one tile, one behind the other)
          float low[8];
          values(r + 1, low);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = join_pair(v[e], low[e]);
          float* y = reinterpret_cast<float*>(p.y) + (row >> 1) * p.y_stride + col;
          if (vec) {
            reinterpret_cast<f32x4*>(y)[0] = f32x4{v[0], v[1], v[2], v[3]};
            reinterpret_cast<f32x4*>(y)[1] = f32x4{v[4], v[5], v[6], v[7]};
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (col + e < p.width) y[e] = v[e];
          }
          continue;
        }
        uint16_t high[8], low[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) split_pair(v[e], high[e], low[e]);
        uint16_t* y = p.y + 2 * row * p.y_stride + col;
        if (vec) {
          *reinterpret_cast<u32x4*>(y) = __builtin_bit_cast(u32x4, high);
          *reinterpret_cast<u32x4*>(y + p.y_stride) = __builtin_bit_cast(u32x4, low);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (col + e < p.width) {
              y[e] = high[e];
              y[p.y_stride + e] = low[e];
            }
        }
      }
    }
  }
}

template <bool kXMx, bool kWMx, int kI, int kJ, int kPair>
struct Body {
  using S = Shape<kXMx, kWMx, kI, kJ>;
  const Params& p;
  int lane, wave, h;        // h: lane half
  int stages;
  // Copies: where the lane's 16-byte unit of each row that it copies is, and how
  // many bytes of the row are left from there on. bf16 x: addresses, with zeros in the
  // place of what lies past the end of k. MXFP4 x: row offsets (below 4 GiB) from a
  // common base; past the end the row's last unit again, as there both scale bytes are 0
  // and 2^-254 vanishes whatever the codes.
  const char* xsrc[kXMx ? 1 : S::kXCopies];
  const char* wsrc[kXMx ? 1 : S::kWCopies];
  uint32_t xrow[kXMx ? S::kXCopies : 1], wrow[kXMx ? S::kWCopies : 1];
  uint32_t at, row_last;
  const char* wfirst;
  int xleft, wleft;
  // Operand reads: byte offsets in a slot of sub-step s = 0, row of fragment 0.
  int xread, wread, xmask, wmask;
  // Scales: the rows this thread loads, their next unit, and where it reads fragment 0's.
  const uint8_t *xscale, *wscale;
  u32x4 xunit, wunit;
  int unit_skip, skips[2];
  int xsread, wsread;
  f32x16 acc[kI][kJ];

  __device__ __forceinline__ Body(const Params& p_) : p(p_) {}

  __device__ __forceinline__ int weight_row(int nt, int r) const {
    if (!p.swiglu) return min(nt * 64 * kJ + r, p.n - 1);
    // Half a fragment are gate rows, half up rows of the same columns.
    const int column = nt * 32 * kJ + r / 32 * 16 + r % 16;
    return min(column, p.width - 1) + (r / 16 % 2 ? p.width : 0);
  }

  // Copies of index first .. last - 1 of the next stage into a slot.
  __device__ __forceinline__ void copy(char* slot, int first, int last) {
    if constexpr (kXMx) {
      const uint32_t from = min(at, row_last);
#pragma unroll
      for (int d = 0; d < S::kXCopies; ++d)
        if (d >= first && d < last) copy16(p.x + (xrow[d] + from), slot + (d * 4 + wave) * 1024);
#pragma unroll
      for (int d = 0; d < S::kWCopies; ++d)
        if (d + S::kXCopies >= first && d + S::kXCopies < last)
          copy16(wfirst + (wrow[d] + from), slot + S::kXBytes + (d * 4 + wave) * 1024);
      if (first < last && last == S::kLoads) at += kXRow;
    } else {
      const char* zeros = reinterpret_cast<const char*>(&kZeros);
#pragma unroll
      for (int d = 0; d < S::kXCopies; ++d)
        if (d >= first && d < last) {
          copy16(xleft > 0 ? xsrc[d] : zeros, slot + (d * 4 + wave) * 1024);
          xsrc[d] += kXRow;
        }
#pragma unroll
      for (int d = 0; d < S::kWCopies; ++d)
        if (d + S::kXCopies >= first && d + S::kXCopies < last) {
          copy16(wleft > 0 ? wsrc[d] : zeros, slot + S::kXBytes + (d * 4 + wave) * 1024);
          wsrc[d] += S::kWRow;
        }
      if (first < last && last == S::kLoads) {
        xleft -= kXRow;
        wleft -= S::kWRow;
      }
    }
  }

  // Loads the scales of unit u (at any alignment): blocks 16 u .. of the thread's x
  // and weight row (k >= 512), or 2 kSlots u .. of its weight row (k >= 128). Nothing
  // past the row is read: towards its end the last bytes that can be, and
  // write_units moves them into place, with zeros past the end of k. No
  // branches: matrix instructions sink past them out of their order.
  // (MXFP4 x: every thread loads, so that each wave has as many loads on their way; kX, kW: which of them.)
  template <bool kX = true, bool kW = true>
  __device__ __forceinline__ void load_units(int u) {
    typedef u32x4 u32x4u __attribute__((aligned(1)));
    typedef uint32_t u32u __attribute__((aligned(1)));
    const int blocks = p.k / mx::kBlock;
    if constexpr (kXMx) {
      const int from = min(16 * u, blocks - 16);
      unit_skip = min(16 * u - from, 16);
      if constexpr (kX) xunit = *reinterpret_cast<const u32x4u*>(xscale + from);
      if constexpr (kW) wunit = *reinterpret_cast<const u32x4u*>(wscale + from);
    } else if constexpr (kWMx) {
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        const int want = 2 * S::kSlots * u + 4 * d, from = min(want, blocks - 4);
        wunit[d] = *reinterpret_cast<const u32u*>(wscale + from);
        skips[d] = min(want - from, 4);
      }
    }
  }
  template <bool kX = true, bool kW = true>
  __device__ __forceinline__ void write_units(char* scales, int u) const {
    char* to = scales + (kXMx ? 0 : (u & 1) * (S::kScaleBytes / 2)) + threadIdx.x * S::kUnitBytes;
    if constexpr (kXMx) {
      // (The two stages' dwords of a lane half side by side.)
      if constexpr (kX) {
        const u32x4 x = mx::drop_bytes(xunit, unit_skip);
        *reinterpret_cast<u32x4*>(to) = u32x4{x.x, x.z, x.y, x.w};
      }
      if constexpr (kW) {
        const u32x4 w = mx::drop_bytes(wunit, unit_skip);
        *reinterpret_cast<u32x4*>(to + S::kXUnits) = u32x4{w.x, w.z, w.y, w.w};
      }
    } else if constexpr (kWMx) {
      *reinterpret_cast<u32x2*>(to) =
          u32x2{uint32_t(uint64_t(wunit.x) >> (8 * skips[0])), uint32_t(uint64_t(wunit.y) >> (8 * skips[1]))};
    }
  }
  // Scales of a stage at place kPos of unit u. MXFP4 x: fragments first .. last - 1
  // (x, then weights) of both stages of the unit.
  template <int kPos>
  __device__ __forceinline__ void read_scales(const char* scales, int u, Scales& s, int first = 0, int last = kI + kJ) const {
    const char* from = scales + (kXMx ? 0 : (u & 1) * (S::kScaleBytes / 2));
    if constexpr (kXMx) {
#pragma unroll
      for (int i = 0; i < kI; ++i)
        if (i >= first && i < last) s.x[i] = *reinterpret_cast<const u32x2*>(from + xsread + i * 64 * 16);
#pragma unroll
      for (int j = 0; j < kJ; ++j)
        if (j + kI >= first && j + kI < last) s.w[j] = *reinterpret_cast<const u32x2*>(from + wsread + j * 32 * 16);
    } else if constexpr (kWMx) {
#pragma unroll
      for (int j = 0; j < kJ; ++j) s.w[j].x = *reinterpret_cast<const uint8_t*>(from + wsread + j * 32 * S::kUnitBytes + kPos * 2);
    }
  }

  // Operands first .. last - 1 of sub-step s: x fragments, then weight fragments.
  // (MXFP4 weights beside bf16 x are read once per stage.)
  static constexpr int kReads = kI + (S::kDecode ? 0 : kJ);
  __device__ __forceinline__ void read(const char* slot, int s, Frags<kI, kJ>& f, int first = 0, int last = kReads) const {
    const int unit = (4 * h + s) * 16;
#pragma unroll
    for (int i = 0; i < kI; ++i)
      if (i >= first && i < last) f.x[i] = *reinterpret_cast<const u32x4*>(slot + xread + i * 64 * kXRow + (unit ^ xmask));
    if constexpr (!S::kDecode) {
#pragma unroll
      for (int j = 0; j < kJ; ++j)
        if (j + kI >= first && j + kI < last)
          f.w[j] = *reinterpret_cast<const u32x4*>(slot + S::kXBytes + wread + j * 32 * kXRow + (unit ^ wmask));
    }
  }
  __device__ __forceinline__ void read_codes(const char* slot, u32x4 (&codes)[kJ]) const {
    if constexpr (S::kDecode) {
#pragma unroll
      for (int j = 0; j < kJ; ++j)
        codes[j] = *reinterpret_cast<const u32x4*>(slot + S::kXBytes + wread + j * 32 * S::kWRow + h * 16);
    }
  }

  template <int kPos, int kS>
  __device__ __forceinline__ void multiply(const Frags<kI, kJ>& f, const Scales& sc, int i, int j) {
    if constexpr (kXMx) {
      acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx::operand(f.w[j]), mx::operand(f.x[i]), acc[i][j], 4, 4, kS,
                                                                    int(sc.w[j][kPos & 1]), kS, int(sc.x[i][kPos & 1]));
    } else {
      acc[i][j] = mfma32(vec_bf16x8(f.w[j]), vec_bf16x8(f.x[i]), acc[i][j]);
    }
  }

  // One sub-step's kI kJ instructions, with `extra(n)` behind the n-th.
  template <int kPos, int kS, class Extra>
  __device__ __forceinline__ void sub_step(const Frags<kI, kJ>& f, const Scales& sc, Extra&& extra) {
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int i = 0; i < kI; ++i) {
        multiply<kPos, kS>(f, sc, i, j);
        extra(j * kI + i);
        pin();
      }
  }

  // Copies of a stage go out behind two sub-steps' instructions, half from the
  // sub-step on that frees their slot, half in the one after (all at once they
  // fill the memory pipe and hold the matrix instructions back: 8192 x 8192 x 8192
  // in bf16 8 % slower; over three or four sub-steps the last arrive too late).
  static constexpr int kFirst = S::kLoads / 2;
  // A sub-step's reads go out one behind each instruction where there are enough of them.
  static constexpr bool kSpread = kI * kJ >= kReads;

  // Stage kPos of round u, in `cur`; its first operands are in `f`, its scales in `sc`.
  // `next` holds the stage after it, and on return `f`, `sc` and `codes` are that
  // stage's. `prev` is the slot whose last reader was the stage before.
  template <int kPos>
  __device__ __forceinline__ void stage(char* prev, char* cur, const char* next, char* scales, int u,
                                        Frags<kI, kJ>& f, u32x4 (&codes)[kJ], Scales& sc) {
    constexpr int kM = kI * kJ;
    constexpr bool kLast = kPos == S::kSlots - 1;
    constexpr int kNext = kLast ? 0 : kPos + 1;
    const int u_next = kLast ? u + 1 : u;
    // Beside bf16 x, at the start of a unit the next one's scales, loaded a unit ago, go to the
    // other buffer (its last readers are behind the last barrier) and the loads of the one after it start.
    if constexpr (S::kDecode && kPos == 0) {
      write_units(scales, u + 1);
      load_units(u + 2);
      pin();
    }
    // MXFP4 x: a unit's scales are in registers from its first stage on, so the next one's,
    // written in its second stage behind the first one's barrier, take their place. With two slots
    // their loads go out behind the first stage's copies, apart (a load of 64 rows' scales takes
    // the address unit four times as long as a copy), else as soon as their registers are free.
    const int unit = u * (S::kSlots / 2) + kPos / 2;
    constexpr bool kLateLoads = kXMx && kPos % 2 == 0 && S::kSlots == 2;
    auto next_scales = [&](int n) {
      if constexpr (kXMx && kPos % 2 == 1) {
        if (n == 0) write_units<true, false>(scales, unit + 1);
        if (n == kM / 2) write_units<false, true>(scales, unit + 1);
        if (n == kM / 2 && S::kSlots > 2) load_units(unit + 2);
      }
      if constexpr (kLateLoads) {
        if (n == 0) load_units<true, false>(unit + 1);
        if (n == kM / 2) load_units<false, true>(unit + 1);
      }
    };
    Frags<kI, kJ> g;
    auto decode = [&](Frags<kI, kJ>& to, const u32x4 (&from)[kJ], const Scales& s, int sub, int n) {
      // Fragment j's conversions behind instruction j kI (all of them early enough for the next sub-step).
      if constexpr (S::kDecode)
        if (n % kI == 0) to.w[n / kI] = mx::decode8(from[n / kI][sub], mx::scale_f32(s.w[n / kI].x));
    };
    auto copies = [&](char* slot, int first, int last, int n) {
      copy(slot, first + n * (last - first) / kM, first + (n + 1) * (last - first) / kM);
    };
    // (Before each round of reads a wait for the last one, which has long arrived:
    // the compiler would otherwise wait behind the new reads, for them too.)
    auto reads = [&](const char* slot, int sub, Frags<kI, kJ>& to, int n) {
      if (kSpread) read(slot, sub, to, n, n + 1);
    };
    reads_done();
    if (!kSpread) read(cur, 1, g);
    pin();
    sub_step<kPos, 0>(f, sc, [&](int n) {
      reads(cur, 1, g, n);
      decode(g, codes, sc, 1, n);
      copies(prev, kFirst, S::kLoads, n);
    });
    reads_done();
    if (!kSpread) read(cur, 2, f);
    pin();
    sub_step<kPos, 1>(g, sc, [&](int n) {
      reads(cur, 2, f, n);
      decode(f, codes, sc, 2, n);
      next_scales(n);
    });
    reads_done();
    if (!kSpread) read(cur, 3, g);
    pin();
    sub_step<kPos, 2>(f, sc, [&](int n) {
      reads(cur, 3, g, n);
      decode(g, codes, sc, 3, n);
    });
    // Every wave has read all of `cur`, and `next` has arrived: at most the copies
    // of the stages after it, and the two loads of scales behind them, are still on their way.
    reads_done();
    wait_vm<(S::kSlots - 2) * S::kLoads + (kLateLoads ? 2 : 0)>();
    barrier_only();
    Scales su;
    if constexpr (S::kDecode) read_scales<kNext>(scales, u_next, su);
    u32x4 codes_next[kJ];
    read_codes(next, codes_next);
    if (!kSpread) read(next, 0, f);
    if constexpr (kXMx && kPos % 2 == 1 && !kSpread) read_scales<0>(scales, unit + 1, su);
    pin();
    sub_step<kPos, 3>(g, sc, [&](int n) {
      reads(next, 0, f, n);
      if constexpr (kXMx && kPos % 2 == 1 && kSpread) read_scales<0>(scales, unit + 1, su, n, n + 1);
      copies(cur, 0, kFirst, n);
      decode(f, codes_next, su, 0, n);
    });
    if constexpr (kXMx && kPos % 2 == 1) sc = su;
    if constexpr (S::kDecode) {
      sc = su;
#pragma unroll
      for (int j = 0; j < kJ; ++j) codes[j] = codes_next[j];
    }
  }

  // All stages. The slots are separate arguments so that the compiler knows
  // that reads of one do not depend on the copies into another (it would wait
  // for every copy in flight before each read).
  __device__ __forceinline__ void ring(char* __restrict__ s0, char* __restrict__ s1, char* __restrict__ s2,
                                       char* __restrict__ s3, char* __restrict__ s4, char* __restrict__ s5,
                                       char* __restrict__ s6, char* __restrict__ s7, char* __restrict__ scales) {
    constexpr int kN = S::kSlots;
    char* const slot[8] = {s0, s1, s2, s3, s4, s5, s6, s7};
    load_units(0);
    pin();
#pragma unroll
    for (int n = 0; n < kN - 1; ++n) copy(slot[n], 0, S::kLoads);
    copy(slot[kN - 1], 0, kFirst);
    pin();
    if constexpr (kWMx) write_units(scales, 0);
    if constexpr (!kXMx || S::kSlots > 2) load_units(1);
    wait_vm<(kN - 2) * S::kLoads + kFirst>();
    lds_barrier();
    Scales sc;
    read_scales<0>(scales, 0, sc);
    Frags<kI, kJ> f;
    u32x4 codes[kJ];
    read(s0, 0, f);
    read_codes(s0, codes);
    if constexpr (S::kDecode) {
#pragma unroll
      for (int j = 0; j < kJ; ++j) f.w[j] = mx::decode8(codes[j].x, mx::scale_f32(sc.w[j].x));
    }
    // (The larger tiles run whole rounds of the ring, stages past the end on zeros: with
    // more than one way out of the loop the compiler moves their sums through scratch.)
    constexpr bool kWhole = kI * kJ > 3;
    for (int st = 0, u = 0; st < stages; st += kN, ++u) {
#define LF_STAGE(n)                                                                                                  \
  if constexpr (kN > n) {                                                                                            \
    if (!kWhole && n > 0 && st + n >= stages) break;                                                                  \
    stage<n>(slot[(n + kN - 1) % kN], slot[n], slot[(n + 1) % kN], scales, u, f, codes, sc);                          \
  }
      LF_STAGE(0)
      LF_STAGE(1)
      LF_STAGE(2)
      LF_STAGE(3)
      LF_STAGE(4)
      LF_STAGE(5)
      LF_STAGE(6)
      LF_STAGE(7)
#undef LF_STAGE
    }
  }

  // The tile of `count` rows from `first` on, weight rows of column tile nt.
  __device__ __forceinline__ void run(char* lds, const Segment& seg, int first, int count, int nt) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    h = lane >> 5;
    const int wm = wave & 1, wn = wave >> 1, c = lane & 31;
    const int blocks = p.k / mx::kBlock;
    const int row_bytes_x = kXMx ? p.k / 2 : p.k * 2, row_bytes_w = kWMx ? p.k / 2 : p.k * 2;
    stages = (p.k + S::kStageK - 1) / S::kStageK;
    const int last = first + count - 1;

    // A copy covers eight rows of 128 bytes (of 32 bytes: 32 rows); row r's unit u
    // sits at u ^ (r / 2 % 8): two rows fill the 64 banks, and the 16 lanes of a pass of a
    // 16-byte read (which are not neighbours) then meet no bank twice. With r % 8 in its
    // place 40 % of the LDS cycles were conflicts.
    const int r8 = lane >> 3;
    const int xat = ((lane & 7) ^ ((wave & 1) * 4 + (r8 >> 1))) * 16;
    const int64_t w0 = int64_t(seg.expert) * p.n;
    const int wr = S::kWRow == 128 ? r8 : lane >> 1;
    const int wat = S::kWRow == 128 ? xat : (lane & 1) * 16;
#pragma unroll
    for (int d = 0; d < S::kXCopies; ++d) {
      const int64_t row = x_row_of(p, min(first + 8 * (d * 4 + wave) + r8, last));
      if constexpr (kXMx)
        xrow[d] = uint32_t(row * p.x_row);
      else
        xsrc[d] = p.x + row * p.x_row + xat;
    }
#pragma unroll
    for (int d = 0; d < S::kWCopies; ++d) {
      const int row = weight_row(nt, ((d * 4 + wave) * (1024 / S::kWRow) + wr) % (64 * kJ));
      if constexpr (kXMx)
        wrow[d] = uint32_t(row) * uint32_t(row_bytes_w);
      else
        wsrc[d] = p.w + (w0 + row) * row_bytes_w + wat;
    }
    wfirst = p.w + w0 * row_bytes_w;
    at = uint32_t(xat);
    row_last = uint32_t(row_bytes_x) - 16;
    xleft = row_bytes_x - xat;
    wleft = row_bytes_w - wat;

    xread = (32 * wm + c) * kXRow;  // fragment i: rows 64 i + 32 wm ..
    xmask = (c / 2 % 8) * 16;
    wread = (32 * kJ * wn + c) * S::kWRow;
    wmask = xmask;
    const int t = threadIdx.x;
    if constexpr (kXMx) {
      xscale = p.xs + x_row_of(p, min(first + t, last)) * blocks;
      xsread = (32 * wm + c) * 16 + 8 * h;
    }
    if constexpr (kWMx) {
      wscale = p.ws + (w0 + weight_row(nt, t % (64 * kJ))) * blocks;
      wsread = (kXMx ? S::kXUnits : 0) + (32 * kJ * wn + c) * S::kUnitBytes + (kXMx ? 8 : 1) * h;
    }
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    auto slot = [&](int n) { return lds + (n < S::kSlots ? n : 0) * S::kStage; };
    ring(slot(0), slot(1), slot(2), slot(3), slot(4), slot(5), slot(6), slot(7), lds + S::kSlots * S::kStage);

    // Copies of zeros for stages past the end are still on their way, and other
    // waves read their last operands.
    wait_vm<0>();
    lds_barrier();
    if (kPair == kSplit || (kPair == kSingle && p.swiglu))
      finish<kI, kJ, true, kPair>(p, acc, lds, seg.expert, first, count, nt);
    else
      finish<kI, kJ, false, kPair>(p, acc, lds, seg.expert, first, count, nt);
  }
};

// Where a workgroup's tile is. Tiles are numbered by expert, within an expert in
// groups of kGroup row tiles, column by column, and dealt to the XCDs (workgroup
// number modulo 8) in contiguous ranges: an XCD's workgroups share few row and
// column tiles at a time in its L2, and an expert's weights go to few XCDs.
constexpr int kGroup = 4;
constexpr int kXcds = 8;

__device__ __forceinline__ int tiles_of(const Segment& s, int cap) { return (s.end - s.begin + cap - 1) / cap; }

__device__ __forceinline__ int total_tiles(const Params& p, int cap) {
  if (!p.offsets) return (p.rows + cap - 1) / cap;
  int sum = 0;
  for (int e = threadIdx.x & 63; e < p.experts; e += 64) sum += tiles_of(segment_of(p, e), cap);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
  return __builtin_amdgcn_readfirstlane(sum);
}

struct Place {
  Segment seg;
  int first, count, nt;  // rows of the product, column tile; count 0: no tile
};

// The item of a workgroup among `items` of them, or -1.
__device__ __forceinline__ int item_of(int items) {
  const int share = (items + kXcds - 1) / kXcds, local = blockIdx.x / kXcds;
  const int index = int(blockIdx.x % kXcds) * share + local;
  return local < share && index < items ? index : -1;
}

// The workgroup's item and its expert, from bounds of up to 64 kPer experts that are loaded once. (Loaded twice, and added
// up by shuffles through LDS: 384 tokens of two choices among 32 experts, 1024 x 2048, 22.9 us, this way 22.0; 8192 tokens of
// four among 64, 4096 x 4096, MXFP4 420 and 413.)
template <int kPer>
__device__ __forceinline__ Segment find_once(const Params& p, int cap, int column_tiles, int& index) {
  const int lane = threadIdx.x & 63;
  Segment s[kPer];
  int sum[kPer], total = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) s[i] = segment_of(p, min(64 * i + lane, p.experts - 1));
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (64 * i + lane >= p.experts) s[i].end = s[i].begin;
    sum[i] = total + scan_lanes(tiles_of(s[i], cap));
    total = __builtin_amdgcn_readlane(sum[i], 63);
  }
  index = item_of(total * column_tiles);
  if (index < 0) return {0, 0, 0};
  Segment found{0, 0, 0};
  int at = index;
  bool open = true;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint64_t past = __ballot(sum[i] * column_tiles > index);
    if (open && past) {
      const int l = __builtin_ctzll(past);
      at = index - __builtin_amdgcn_readlane(sum[i] - tiles_of(s[i], cap), l) * column_tiles;
      found = {64 * i + l, __builtin_amdgcn_readlane(s[i].begin, l), __builtin_amdgcn_readlane(s[i].end, l)};
      open = false;
    }
  }
  index = at;
  return found;
}

__device__ __forceinline__ Place locate(const Params& p, int cap, int column_tiles) {
  int index;
  Segment seg;
  if (p.offsets && p.experts <= 256) {
    seg = p.experts <= 64 ? find_once<1>(p, cap, column_tiles, index) : find_once<4>(p, cap, column_tiles, index);
  } else {
    index = item_of(total_tiles(p, cap) * column_tiles);
    if (index >= 0) seg = find_segment(p, index, [&](const Segment& s) { return tiles_of(s, cap) * column_tiles; });
  }
  if (index < 0) return {{0, 0, 0}, 0, 0, 0};
  const int rows = seg.end - seg.begin, tiles = tiles_of(seg, cap);
  if (rows <= 0) return {{0, 0, 0}, 0, 0, 0};
  const int group = index / (kGroup * column_tiles), in_group = index - group * kGroup * column_tiles;
  const int group_tiles = min(kGroup, tiles - group * kGroup);
  const int mt = group * kGroup + in_group % group_tiles, nt = in_group / group_tiles;
  // 64-row steps of the expert, shared out evenly: the first tiles get one more.
  const int steps = (rows + 63) / 64, each = steps / tiles, more = steps - each * tiles;
  const int first = seg.begin + 64 * (mt * each + min(mt, more));
  return {seg, first, min(64 * (each + (mt < more)), seg.end - first), nt};
}

template <bool kXMx, bool kWMx, int kJ, int kPair>
__global__ __launch_bounds__(kThreads, 1) void tile_kernel(Params p, int cap, int column_tiles) {
  extern __shared__ char lds[];
  const auto [seg, first, count, nt] = locate(p, cap, column_tiles);
  if (count <= 0) return;
  switch ((count + 63) / 64) {
    case 1: Body<kXMx, kWMx, 1, kJ, kPair>(p).run(lds, seg, first, count, nt); break;
    case 2: Body<kXMx, kWMx, 2, kJ, kPair>(p).run(lds, seg, first, count, nt); break;
    case 3: Body<kXMx, kWMx, 3, kJ, kPair>(p).run(lds, seg, first, count, nt); break;
    default: Body<kXMx, kWMx, 4, kJ, kPair>(p).run(lds, seg, first, count, nt); break;
  }
}

// Launches tiles of at most `cap` rows (64, 128, 192 or 256) x 64 kJ weight rows.
template <int kJ>
int launch_kernel(void (*kernel)(Params, int, int), const Params& p, int cap, hipStream_t stream) {
  const int64_t columns = p.swiglu ? 32 * kJ : 64 * kJ;
  const int64_t column_tiles = (p.width + columns - 1) / columns;
  // At most: a tile more than whole ones for every expert that has a row.
  const int64_t used = p.offsets ? (p.experts < p.rows ? p.experts : p.rows) : 1;
  const int64_t row_tiles = (p.rows + used * (cap - 1)) / cap;
  LF_REQUIRE(row_tiles * column_tiles < (int64_t(1) << 30), "too many tiles");
  const unsigned grid = unsigned((row_tiles * column_tiles + kXcds - 1) / kXcds * kXcds);
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), kLds, stream, p, cap, int(column_tiles));
  LF_HIP(hipGetLastError());
  return kOk;
}
template <bool kXMx, bool kWMx, int kJ>
int launch(const Params& p, int cap, hipStream_t stream) {
  if constexpr (!kXMx) {
    if (p.pair == kSplit) return launch_kernel<kJ>(tile_kernel<kXMx, kWMx, kJ, kSplit>, p, cap, stream);
    if (p.pair == kJoin) return launch_kernel<kJ>(tile_kernel<kXMx, kWMx, kJ, kJoin>, p, cap, stream);
  }
  return launch_kernel<kJ>(tile_kernel<kXMx, kWMx, kJ, kSingle>, p, cap, stream);
}

}  // namespace tile
}  // namespace expert
}  // namespace lf
