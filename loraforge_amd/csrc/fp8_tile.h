// Products of many rows with FP8 weights: MFMA tiles of up to 256 rows x 64 kJ weight rows.
//
// Four waves, one per SIMD, 2 x 2: a wave owns 32 kI rows x 32 kJ weight rows. A stage is 128 k,
// one block of scales: for each of its kI kJ pairs of fragments a wave multiplies the
// block from zero (two v_mfma_f32_32x32x64_f8f6f4 where x is FP8, eight v_mfma_f32_32x32x16_bf16
// beside weights decoded in registers where it is bf16) into one of two registers sets T,
// and adds T times the block's scales to the pair's sums while the next pair is multiplied.
//
// The sums are operands of vector instructions, which reach 256 registers of a lane and not
// the other 256 (those hold the fragments): 192 of them are the most sums beside T, so tiles have
// at most 256 x 192 or 192 x 256. A scale is that of an x row (a lane) times that of 128 weight rows:
// one product a pair, and two with SwiGLU, where half a fragment's rows are gate rows and half up rows.
//
// Operands go through LDS by direct copies, rows of 128 bytes (of bf16 x 256), and so do the scales,
// a float a row and stage. Copies are buffer loads, which give zeros past the end of a buffer:
// a lane whose unit lies past the end of k, or a stage past it, asks for an address past every end.
// x fragments are held for a stage and replaced as the last weight fragment is done with each;
// weight fragments are read one ahead.
//
// What bounds it, by clock stamps in a copy that records them, 4096 x 12288 x 4096:
//
//                            tiles   clocks of a tile: start   loop              end     all     matrix  clock     product
//   FP8 both, 256 x 192      1024                      6.2k    73.1k (32 x 2284)  10.6k   89.9k   55 %    1.89 GHz  195-207 us
//   FP8 both, 192 x 256      1056                      6.4k    67.8k (32 x 2120)   8.4k   82.6k   59 %    1.91 GHz  219 (a fifth round)
//   bf16 x, 128 x 256        1536                      5.7k   111.2k (32 x 3475)   6.1k  123.0k   53 %    2.03 GHz  375-385
//
// (A library's product of the same codes with one scale for each row takes 173 us, with one in all 156, in bf16 281.) In the
// loop a stage's 24 pairs of matrix instructions are 1536 clocks; a pair's sixteen scaled additions, its share of reads, copies
// and scales are issued beside them, and what waits for what leaves a third unused. The clock falls with the work, from
// 2.4 GHz: 2.0 to 2.1 PFLOP/s. Beside bf16 x each wave decodes the weights that it multiplies, a conversion for two.
// Steps, 4096 x 12288 x 4096: weights streamed 1419 us, tiles 209, two barriers a stage and scales once a stage 195-207.
#pragma once

#include "expert_tile.h"

namespace lf {
namespace expert {
namespace tile8 {

using tile::kLds;
using tile::kThreads;
using tile::pin;
using tile::reads_done;

constexpr uint32_t kPast = 0x80000000u;  // past the end of every buffer here (they end below 2^31)
constexpr int kWRow = 128;

template <bool kX8, int kI, int kJ>
struct Shape {
  static constexpr int kXRow = kX8 ? 128 : 256;  // bytes of an x row per stage
  static constexpr int kXBytes = 64 * kI * kXRow, kWBytes = 64 * kJ * kWRow;
  static constexpr int kScaleBytes = (kX8 ? 2 : 1) * kThreads * 4;
  static constexpr int kStage = kXBytes + kWBytes + kScaleBytes;
  static constexpr int kSlots = 4 * kStage <= kLds ? 4 : 2;  // (even: two weight buffers and two T take turns over a round)
  static_assert(kSlots * kStage <= kLds, "two stages have to fit");
  static constexpr int kXCopies = kXBytes / 4096, kWCopies = kWBytes / 4096;  // per wave
  static constexpr int kLoads = kXCopies + kWCopies + (kX8 ? 2 : 1);
  static constexpr int kXUnits = kX8 ? 4 : 8;  // 16-byte units of an x fragment that a lane holds
};

// Sizes that fit LDS and registers.
constexpr int most_rows(bool x8, int columns) { return x8 ? (columns > 192 ? 192 : 256) : (columns > 192 ? 128 : 192); }

typedef __attribute__((address_space(3))) void* LdsPtr;
__device__ __forceinline__ void copy16(__amdgpu_buffer_rsrc_t r, char* lds, uint32_t at, uint32_t base) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsPtr)lds, 16, at, base, 0, 0);
}
__device__ __forceinline__ void copy4(__amdgpu_buffer_rsrc_t r, char* lds, uint32_t at, uint32_t base) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsPtr)lds, 4, at, base, 0, 0);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}

// The LDS of one stage: separate pointers, so that the compiler knows that reads of one slot do
// not wait for the copies into another.
struct Slot {
  char *x, *w, *s;
};

template <bool kX8, int kI, int kJ>
struct Body {
  using S = Shape<kX8, kI, kJ>;
  static constexpr int kPairs = kI * kJ;
  const Params& p;
  int lane, wave, h, stages, blocks;
  int plain_stages;  // first ones that need no checks
  // Copies: buffers, the lane's offset of each x row that it copies (its 16-byte unit added), of
  // its first weight row (the others a uniform step apart) and of its rows' scales.
  __amdgpu_buffer_rsrc_t xbuf, wbuf, xsbuf, wsbuf;
  uint32_t xrow[S::kXCopies], wrow, wstep, xsrow, wsrow;
  // (With 192 sums they are kept where vector instructions do not reach, and fetched for each copy: left to itself the
  // compiler moves ten times as many values to and fro.)
  static constexpr bool kFar = kI * kJ * 16 > (kX8 ? 160 : 112);
  int xunit, wunit;  // byte of the lane's unit in a stage's row
  // Operand reads: byte offsets in a slot of unit n of fragment 0, and of its scales.
  uint32_t xat[S::kXUnits], wat[4], xsat, wsat;
  f32x16 acc[kI][kJ];
  u32x4 x[kI][S::kXUnits], w[kX8 ? 2 : 1][4], wd[kX8 ? 1 : 8];
  // Weight scales of the gate (or all) and the up rows, two in turn: of a wave's rows where those lie in one
  // block of 128 each (all widths but 192), else of a fragment's. x rows' scales, in scale[i][0] until they are
  // multiplied with the weights'.
  static constexpr bool kOneBlock = kJ != 3;
  // (One kernel for all of bf16 x: the compiler finds no registers for 192 rows x 128 weight rows that store pairs alone.)
  static constexpr int kPair = kX8 ? kSingle : tile::kAnyPair;
  float sw[2][2], scale[kI][2];
  f32x16 t[2];
  float due[2];  // scales of the pair whose products wait in T

  __device__ __forceinline__ Body(const Params& p_) : p(p_) {}

  static __device__ __forceinline__ uint32_t far(uint32_t v) {
    if constexpr (kFar) asm volatile("v_accvgpr_write_b32 %0, %1" : "=a"(v) : "v"(v));
    return v;
  }
  static __device__ __forceinline__ uint32_t near(uint32_t v) {
    if constexpr (kFar) {
      uint32_t to;
      asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(to) : "a"(v));
      return to;
    }
    return v;
  }

  __device__ __forceinline__ int weight_row(int nt, int r) const {
    if (!p.swiglu) return min(nt * 64 * kJ + r, p.n - 1);
    const int column = nt * 32 * kJ + r / 32 * 16 + r % 16;
    return min(column, p.width - 1) + (r / 16 % 2 ? p.width : 0);
  }

  // A stage's copies in the order of their issue: x, its scales and the weight fragments that are read before the
  // stage's first barrier (kEarly of them), then the others. (Copies j and kJ + j are fragment j's, for both halves of the
  // tile. The weights' scales are read with each fragment where they are not one for all: with the late ones then.)
  static constexpr int kEarlyFrags = kJ >= 3 ? 2 : kJ == 2 ? 1 : 0;
  static constexpr int kEarly = kJ == 1 ? 0 : S::kXCopies + 2 * kEarlyFrags + (kX8 ? 1 : 0) + (kOneBlock ? 1 : 0);
  static constexpr int kLate = S::kLoads - kEarly;
  // Pair of the first of two weight fragments that begins with the first barrier and the read of the second fragment
  // (not the first pair: the barrier would wait for the reads behind the last stage).
  static constexpr int kRead = kI > 1 ? 1 : 0;

  // Copies first .. last - 1 of stage st into a slot. kChecked: any stage of any tile; else st is a whole stage of
  // k, and all of the tile's weight rows are there (their step is then part of the uniform offset).
  template <bool kChecked>
  __device__ __forceinline__ void copy(const Slot& to, int st, int first, int last) {
    if (first >= last) return;
    uint32_t xpast = 0, wpast = 0, spast = 0;
    int base = st;
    if constexpr (kChecked) {
      xpast = st * S::kXRow + xunit < (kX8 ? p.k : 2 * p.k) ? 0u : kPast;
      wpast = st * kWRow + wunit < p.k ? 0u : kPast;
      spast = st < blocks ? 0u : kPast;
      base = min(st, blocks - 1);  // (below every buffer's end, where the range check may subtract it)
    }
    int at = 0;
    auto now = [&]() {
      const bool in = at >= first && at < last;
      ++at;
      return in;
    };
    auto weights = [&](int d) {
      if (!now()) return;
      if constexpr (kChecked)
        copy16(wbuf, to.w + (d * 4 + wave) * 1024, (wrow | wpast) + d * wstep, base * kWRow);
      else
        copy16(wbuf, to.w + (d * 4 + wave) * 1024, wrow, base * kWRow + d * wstep);
    };
    auto weight_scales = [&]() {
      if (now()) copy4(wsbuf, to.s + wave * 256, wsrow | spast, base * 4);
    };
#pragma unroll
    for (int d = 0; d < S::kXCopies; ++d)
      if (now()) copy16(xbuf, to.x + (d * 4 + wave) * 1024, near(xrow[d]) | xpast, base * S::kXRow);
#pragma unroll
    for (int j = 0; j < kEarlyFrags; ++j) weights(j), weights(kJ + j);
    if constexpr (kX8)
      if (now()) copy4(xsbuf, to.s + kThreads * 4 + wave * 256, xsrow | spast, base * 4);
    weight_scales();
#pragma unroll
    for (int j = kEarlyFrags; j < kJ; ++j) weights(j), weights(kJ + j);
  }

  __device__ __forceinline__ void read_x(const Slot& from, int i) {
#pragma unroll
    for (int u = 0; u < S::kXUnits; ++u) x[i][u] = *reinterpret_cast<const u32x4*>(from.x + xat[u] + i * 64 * S::kXRow);
    if constexpr (kX8) scale[i][0] = *reinterpret_cast<const float*>(from.s + kThreads * 4 + xsat + i * 64 * 4);
  }
  __device__ __forceinline__ void read_ws(const Slot& from, int j, int b) {
    sw[b][0] = *reinterpret_cast<const float*>(from.s + wsat + j * 32 * 4);
    sw[b][1] = *reinterpret_cast<const float*>(from.s + wsat + j * 32 * 4 + 16 * 4);
  }
  // Weight fragment j into buffer b, and its scales.
  __device__ __forceinline__ void read_w(const Slot& from, int j, int b) {
#pragma unroll
    for (int u = 0; u < 4; ++u) w[kX8 ? b : 0][u] = *reinterpret_cast<const u32x4*>(from.w + wat[u] + j * 32 * kWRow);
    if constexpr (!kOneBlock) read_ws(from, j, b);
  }
  // Unit m (8 k of a lane) of the weight fragment that was read last.
  __device__ __forceinline__ void decode(int m) {
    if constexpr (!kX8) wd[m] = fp8::decode8(w[0][m / 2][m % 2 * 2], w[0][m / 2][m % 2 * 2 + 1]);
  }

  // Adds products first .. last - 1 that wait in a T to their sums.
  __device__ __forceinline__ void settle(f32x16& sums, const f32x16& from, int first, int last) {
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (r >= first && r < last) sums[r] = fmaf(due[r / 8], from[r], sums[r]);
  }

  // Stage st, at place kPos of a round: its x fragments, its first weight fragment and their scales are
  // read. `next` holds the stage after it. Two barriers: behind the first, x and the early weight fragments of
  // `cur` have been read by every wave, and their copies for the stage that comes into it go out; behind the second
  // (at the last weight fragment) the late ones. So a copy has a stage and a third or more until it is
  // waited for (with one barrier and all copies behind it they had two thirds on average: their latency,
  // some 2000 clocks under load, then bounded every tile: 4096 x 12288 x 4096 in 192 x 256 2340 clocks a stage).
  template <int kPos, bool kChecked>
  __device__ __forceinline__ void stage(const Slot& cur, const Slot& next, int st) {
    constexpr int kWBase = kPos * kJ, kTBase = kPos * kPairs;
    constexpr int kSteps = kX8 ? 2 : 8;
#pragma unroll
    for (int n = 0; n < kPairs; ++n) {
      const int j = n / kI, i = n % kI;
      const int b = (kWBase + j) & 1, tn = (kTBase + n) & 1;
      const bool last = j == kJ - 1;
      constexpr int kFirst = kJ == 2 ? kRead : (kEarlyFrags - 1) * kI, kLast = (kJ - 1) * kI;  // pairs that begin with a barrier
      if (kJ > 1 && n == kFirst) {
        // The late copies of `cur` have arrived.
        reads_done();
        wait_vm<(S::kSlots - 1) * S::kLoads>();
        barrier_only();
      }
      if (n == kLast) {
        // The early copies of `next` have arrived (and the first of the late ones, where those are the scales).
        reads_done();
        wait_vm<kJ == 1 ? (S::kSlots - 2) * S::kLoads : (S::kSlots - 1) * S::kLoads - (kOneBlock ? 0 : 1)>();
        barrier_only();
      }
      const int pi = n ? (n - 1) % kI : kI - 1, pj = n ? (n - 1) / kI : kJ - 1;  // the pair whose products wait
#pragma unroll
      for (int m = 0; m < kSteps; ++m) {
        pin();
        if constexpr (kX8) {
          const fp8::i32x8 a = fp8::operand(w[b][2 * m], w[b][2 * m + 1]), c = fp8::operand(x[i][2 * m], x[i][2 * m + 1]);
          if (m == 0)
            t[tn] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, c, f32x16{}, 0, 0, 0, 0, 0, 0);
          else
            t[tn] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, c, t[tn], 0, 0, 0, 0, 0, 0);
        } else {
          t[tn] = mfma32(vec_bf16x8(wd[m]), vec_bf16x8(x[i][m]), m == 0 ? f32x16{} : t[tn]);
        }
        pin();
        // (Reads and copies first: the products that wait are not there yet.)
        if (m == 0) {
          if (i == (kJ == 2 && !last ? kRead : 0)) {
            if (last)
              read_w(next, 0, (kWBase + kJ) & 1);
            else
              read_w(cur, j + 1, b ^ 1);
            if (kOneBlock && last) read_ws(next, 0, (kPos + 1) & 1);
          }
          constexpr int kOver = kLast - kFirst;  // pairs that the early copies are spread over
          if (last)
            copy<kChecked>(cur, st + S::kSlots, kEarly + i * kLate / kI, kEarly + (i + 1) * kLate / kI);
          else if (n >= kFirst)
            copy<kChecked>(cur, st + S::kSlots, (n - kFirst) * kEarly / kOver, (n - kFirst + 1) * kEarly / kOver);
          pin();
        }
        // (The next fragment's weights take the place of those that this pair, the fragment's last, is done with.)
        if (!kX8 && i == kI - 1 && m > 0) decode(m - 1);
        // A block's products are done some 12 clocks after its last instruction, so fewer of them are added at first.
        if constexpr (kX8)
          settle(acc[pi][pj], t[tn ^ 1], m ? 6 : 0, m ? 16 : 6);
        else if (m)
          settle(acc[pi][pj], t[tn ^ 1], (m - 1) * 16 / 7, m * 16 / 7);
      }
      if (!kX8 && i == kI - 1) decode(kSteps - 1);
      const int sb = kOneBlock ? kPos & 1 : b;
      if constexpr (kX8) {
        if (kOneBlock && j == 0) {
          scale[i][1] = scale[i][0] * sw[sb][1];
          scale[i][0] *= sw[sb][0];
        }
        due[0] = kOneBlock ? scale[i][0] : scale[i][0] * sw[sb][0];
        due[1] = kOneBlock ? scale[i][1] : scale[i][0] * sw[sb][1];
      } else {
        due[0] = sw[sb][0];
        due[1] = sw[sb][1];
      }
      if (last) read_x(next, i);
    }
  }

  template <bool kChecked>
  __device__ __forceinline__ void round(const Slot (&slot)[4], int st) {
    constexpr int kN = S::kSlots;
    stage<0, kChecked>(slot[0], slot[1], st);
    stage<1, kChecked>(slot[1], slot[2 % kN], st + 1);
    if constexpr (kN == 4) {
      stage<2, kChecked>(slot[2], slot[3], st + 2);
      stage<3, kChecked>(slot[3], slot[0], st + 3);
    }
  }

  __device__ __forceinline__ void ring(char* __restrict__ x0, char* __restrict__ x1, char* __restrict__ x2, char* __restrict__ x3,
                                       char* __restrict__ w0, char* __restrict__ w1, char* __restrict__ w2, char* __restrict__ w3,
                                       char* __restrict__ s0, char* __restrict__ s1, char* __restrict__ s2, char* __restrict__ s3) {
    constexpr int kN = S::kSlots;
    const Slot slot[4] = {{x0, w0, s0}, {x1, w1, s1}, {x2, w2, s2}, {x3, w3, s3}};
#pragma unroll
    for (int n = 0; n < kN; ++n) copy<true>(slot[n], n, 0, S::kLoads);
    wait_vm<(kN - 1) * S::kLoads>();
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kI; ++i) read_x(slot[0], i);
    read_w(slot[0], 0, 0);
    if (kOneBlock) read_ws(slot[0], 0, 0);
#pragma unroll
    for (int m = 0; m < 8; ++m)
      if (!kX8) decode(m);
    // Rounds that copy whole stages of whole tiles, then those that may not (stages past the end are zeros).
    int st = 0;
    for (; st + 2 * kN <= plain_stages; st += kN) round<false>(slot, st);
    for (; st < stages; st += kN) round<true>(slot, st);
    settle(acc[kI - 1][kJ - 1], t[(kN * kPairs - 1) & 1], 0, 16);
  }

  // The tile of `count` rows from `first` on, weight rows of column tile nt.
  __device__ __forceinline__ void run(char* lds, const Segment& seg, int first, int count, int nt) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    h = lane >> 5;
    const int wm = wave & 1, wn = wave >> 1, c = lane & 31;
    blocks = int(fp8::blocks_of(p.k));
    stages = blocks;
    plain_stages = p.swiglu ? ((nt + 1) * 32 * kJ <= p.width ? p.k / fp8::kBlock : 0)
                            : ((nt + 1) * 64 * kJ <= p.n ? p.k / fp8::kBlock : 0);
    const int last = first + count - 1;

    // Rows of 128 bytes: row r's unit u sits at u ^ (r / 2 % 8), eight rows a copy; rows of 256 bytes: at u ^ (r % 16),
    // four rows a copy. The 16 lanes of a pass of a 16-byte read then meet no bank twice.
    constexpr int kXRows = 1024 / S::kXRow;  // of a copy
    const int xr = lane / (64 / kXRows), wr = lane >> 3;
    xunit = 16 * (kX8 ? (lane & 7) ^ ((wave & 1) * 4 + (xr >> 1)) : (lane & 15) ^ ((wave & 3) * 4 + xr));
    wunit = 16 * ((lane & 7) ^ ((wave & 1) * 4 + (wr >> 1)));
    // (Offsets are below 2^31: checked by the host.)
    xbuf = buffer(p.x, uint32_t((int64_t(p.x_rows) - 1) * p.x_row + (kX8 ? p.k : 2 * p.k)));
    xsbuf = buffer(p.xs8, kX8 ? uint32_t(int64_t(p.x_rows) * blocks * 4) : 0u);
    wbuf = buffer(p.w + int64_t(seg.expert) * p.n * p.k, uint32_t(int64_t(p.n) * p.k));
    wsbuf = buffer(fp8_scales(p, seg.expert, 0), uint32_t(fp8::blocks_of(p.n) * blocks * 4));
#pragma unroll
    for (int d = 0; d < S::kXCopies; ++d) {
      const int64_t row = x_row_of(p, min(first + kXRows * (d * 4 + wave) + xr, last));
      xrow[d] = far(uint32_t(row * p.x_row) + xunit);
    }
    // (Weight rows past n lie past the buffer's end, or are up rows in the place of gate columns that nobody stores.)
    const int r0 = 8 * wave + wr;
    wrow = uint32_t(p.swiglu ? nt * 32 * kJ + r0 % 16 + (r0 / 16 ? p.width : 0) : nt * 64 * kJ + r0) * uint32_t(p.k) + wunit;
    wstep = uint32_t(p.swiglu ? 16 : 32) * uint32_t(p.k);
    const int row = threadIdx.x;
    if constexpr (kX8) xsrow = uint32_t(x_row_of(p, min(first + row, last)) * blocks * 4);
    wsrow = uint32_t(weight_row(nt, row % (64 * kJ)) / fp8::kBlock) * blocks * 4;

#pragma unroll
    for (int u = 0; u < S::kXUnits; ++u)
      xat[u] = (32 * wm + c) * S::kXRow + 16 * ((S::kXUnits * h + u) ^ (kX8 ? c / 2 % 8 : c % 16));
#pragma unroll
    for (int u = 0; u < 4; ++u) wat[u] = (32 * kJ * wn + c) * kWRow + 16 * ((4 * h + u) ^ (c / 2 % 8));
    xsat = (32 * wm + c) * 4;
    wsat = 32 * kJ * wn * 4;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      t[0][r] = t[1][r] = 0.f;
#pragma unroll
      for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j) acc[i][j][r] = 0.f;
    }
    due[0] = due[1] = 0.f;

    // (By operand, then slot: offsets of a read then fit the instruction.)
    constexpr int kN = S::kSlots;
    auto xs = [&](int n) { return lds + (n % kN) * S::kXBytes; };
    auto ws = [&](int n) { return lds + kN * S::kXBytes + (n % kN) * S::kWBytes; };
    auto ss = [&](int n) { return lds + kN * (S::kXBytes + S::kWBytes) + (n % kN) * S::kScaleBytes; };
    ring(xs(0), xs(1), xs(2), xs(3), ws(0), ws(1), ws(2), ws(3), ss(0), ss(1), ss(2), ss(3));

    // Copies of zeros for stages past the end are still on their way, and other
    // waves read their last operands.
    wait_vm<0>();
    lds_barrier();
    if (p.swiglu)
      tile::finish<kI, kJ, true, kPair>(p, acc, lds, seg.expert, first, count, nt);
    else
      tile::finish<kI, kJ, false, kPair>(p, acc, lds, seg.expert, first, count, nt);
  }
};

template <bool kX8, int kJ>
__global__ __launch_bounds__(kThreads, 1) void tile_kernel(Params p, int cap, int column_tiles) {
  extern __shared__ char lds[];
  const auto [seg, first, count, nt] = tile::locate(p, cap, column_tiles);
  if (count <= 0) return;
  constexpr int kMost = most_rows(kX8, 64 * kJ) / 64;
  const int height = (count + 63) / 64;
  if (height == 1) Body<kX8, 1, kJ>(p).run(lds, seg, first, count, nt);
  else if (height == 2) Body<kX8, 2, kJ>(p).run(lds, seg, first, count, nt);
  else if constexpr (kMost >= 3) {
    if (kMost == 3 || height == 3) Body<kX8, 3, kJ>(p).run(lds, seg, first, count, nt);
    else if constexpr (kMost >= 4) Body<kX8, 4, kJ>(p).run(lds, seg, first, count, nt);
  }
}

template <bool kX8>
int launch(const Params& p, int cap, int columns, hipStream_t stream) {
  switch (columns) {
    case 64: return tile::launch_kernel<1>(tile_kernel<kX8, 1>, p, cap, stream);
    case 128: return tile::launch_kernel<2>(tile_kernel<kX8, 2>, p, cap, stream);
    case 192: return tile::launch_kernel<3>(tile_kernel<kX8, 3>, p, cap, stream);
    default: return tile::launch_kernel<4>(tile_kernel<kX8, 4>, p, cap, stream);
  }
}

}  // namespace tile8
}  // namespace expert
}  // namespace lf
