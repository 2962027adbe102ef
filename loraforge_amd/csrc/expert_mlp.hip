// A whole mixture-of-experts MLP for a few tokens (a decode step), in two launches:
// y[t] = base[t] + sum_j s_tj down_e (silu(gate_e x[t]) * (up_e x[t])), e the j-th choice of token t.
//
// Bound by HBM: every weight of a chosen expert is read once; beside it, launches, routing and
// joins are latency. Four operators in a chain (route, product, product, combine) take
// four launches for it. In a graph, us beside the chain's (128 experts, top 8, 4096 x 1024): one token MXFP4 19.5 (29; the
// bytes 10.4 at a copy's rate), FP8 24.8 (32; 19.6), bf16 37 (46; 39); 8 tokens 74 (82; 67), 127 (129; 125), 223 (250; 250).
// The first launch reads at 5.6 TB/s once it is under way (FP8, 7 tokens: 193 MB in 35 us), the second at 4.2 (98 MB in
// 23). Of one token's 19.5 us the first launch is 10.3 (routing 4, until weights that it asked for come 7),
// the second 7.5 (2 until weights come, 1.5 for the join).
//
// First launch. Every workgroup routes all tokens by itself (as expert_routing.hip does: the
// logits come from L2, and nobody waits for another workgroup), x in registers meanwhile.
// Then it takes items in turn: 8 columns of one chosen expert, 8 gate and 8 up rows over the whole of k.
// Its eight waves share k (stage s of 128 bytes of a row to wave s % 8), each streaming its weights through a
// ring of its own in LDS by direct copies; the ring runs on from one item to the next. The weight is
// the A operand of 16 x 16 matrix instructions, *all* tokens are the B operand (of x, held
// in registers: at most 128 of them, which bounds tokens and k): columns of tokens
// that did not choose the expert are computed and dropped, which costs nothing beside the bytes.
// The waves' sums meet in LDS, in a fixed order; the intermediate s silu(g) u, with the routing weight
// in it so that the second product needs no weights, is kept as a pair of bf16 (rounded to one, it is as far
// from the formula as y's own rounding: 1.0 times as much again, and 1.5 of both).
//
// Second launch. With rows of the intermediate in expert order, y is one product whose k runs
// over (chosen experts) x (intermediate): a workgroup owns 16 columns of y, its waves share that long
// k, and their sums meet once at the end. Tokens are the columns of B again, twice: for the high and for the low halves of
// their pairs, which of up to eight tokens fit one tile. A token that did not choose the
// stage's expert reads zeros (past the end of a buffer).
//
// More tokens, and widths that these do not take: routing, gate and up product, down product and sum one after
// another, in the kernels of the operators, with pairs between the products and rows of fp32 before the sum; up to 32 tokens with
// the first launch in place of the first two.
#include <type_traits>

#include "expert_choose.h"
#include "expert_params.h"
#include "lds_pipeline.h"
#include "../../include/loraforge_amd.h"

namespace lf {
namespace expert {
namespace {

constexpr int kWaves = 8;            // of the first launch
constexpr int kThreads = 64 * kWaves;
// Eight tokens: with the halves of their pairs 16 columns of the second launch. (A second tile for up to 16 takes the address
// unit twice as long for x as for the weights: 128 experts, top 8, 4096 x 1024, MXFP4, 12 tokens 111 us, in a chain 100.)
constexpr int kMostTokens = 8;
// What the first launch takes, two tiles of x, also ahead of the operators' down product and sum, in place of the routing and the
// gate and up product: 16 tokens over 32 experts, top 4, 2048 x 1408, bf16 96 us and 117, 24 tokens 104 and 122; 128 experts, top 8,
// 4096 x 1024, 12 tokens MXFP4 98.6 and 99.5, FP8 155 and 161, bf16 287 and 312, 24 tokens FP8 209 and 221, bf16 395 and 399; 8 experts,
// top 2, 8192 x 1024, 16 tokens MXFP4 35.8 and 40.4 (bf16 82.8 and 80.2). Of MXFP4 weights one tile (levels made for two
// cost more than the launch), of FP8 weights two only for a hidden width above 2048: below, an item is two stages or
// fewer to a wave and its join weighs more (24 tokens over 60 experts, top 6, 1024 x 512, 34.8 us and 29.6; 2048 x 1408 59.4 and 56.9).
constexpr int kMostFirst = 32;
// Choices of an expert, on average, up to which a chain keeps pairs: they double the rows of the down product, which costs
// little while its weights' bytes bound it (16 experts, top 4, 4096 x 2048, 64 tokens, 16 choices each: MXFP4 76 us and 68 with
// the intermediate in bf16, FP8 105 and 104, bf16 205 and 202; 128 tokens 97 and 85, 123 and 108, 215 and 207; 512 tokens 237
// and 170, 259 and 209, 278 and 228).
constexpr int kMostEach = 32;
constexpr int kFewTokens = 2;        // routed by ranks
constexpr int kMostExperts = 256;
constexpr int kMostTop = 16;
constexpr int kMostChoices = 256;
constexpr int kTable = kMostTokens * kMostTop;  // chosen experts of two launches
constexpr int kSlotWeights = 16 * 128;
constexpr uint32_t kPast = 0x80000000u;  // past the end of every buffer here

struct MlpParams {
  const char* x;  // bf16 [tokens, hidden]
  int64_t x_row;  // bytes
  const void* logits;
  int64_t logits_stride;
  int32_t fp32, tokens, experts, top, renormalize;
  int32_t hidden, inter;
  const char *gate_up, *down;            // [experts, 2 inter, hidden], [experts, hidden, inter]
  const uint8_t *gate_up_s, *down_s;     // MXFP4 scales
  const float *gate_up_s8, *down_s8;     // FP8 scales
  const uint16_t* base;                  // bf16 [tokens, hidden] or null
  int64_t base_stride;
  uint16_t* y;
  int64_t y_stride;
  uint16_t* h;   // [tokens * top, 2, inter], rows in expert order, halves of pairs
  int4* table;   // x of entry 0: chosen experts; entry 1 + u: expert, first row, mask of its tokens
  // Ahead of the operators (else null): what lf_route_experts gives, and h without weights.
  int32_t *offsets, *positions;
  float* weights;
};

typedef int i32x4 __attribute__((ext_vector_type(4)));

template <int kType>
struct Format {
  static constexpr int kStage = kType == kBf16 ? 64 : kType == kFp8 ? 128 : 256;  // k of 128 bytes
  static constexpr int kUnits = kStage / 32;        // 16-byte units of x that a lane holds of a stage
  static constexpr int kCopies = kType == kMxfp4 ? 3 : 2;
  static constexpr int kSlot = kSlotWeights + (kType == kMxfp4 ? 256 : 0);
  static __host__ __device__ __forceinline__ int64_t row_bytes(int64_t k) { return kType == kBf16 ? 2 * k : kType == kFp8 ? k : k / 2; }
};

typedef __attribute__((address_space(3))) void* LdsPtr;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}

// Exchanges units between the quarters of a wave: of kUnits loads, load n of lane quarter q becomes unit 4 (n % (kUnits / 4)) + q of
// quarter n / (kUnits / 4).
template <int kUnits>
__device__ __forceinline__ void transpose_quarters(u32x4 (&v)[kUnits]) {
  constexpr int kPer = kUnits / 4;  // loads of a quarter
  u32x4 to[kUnits];
#pragma unroll
  for (int h = 0; h < kPer; ++h)
#pragma unroll
    for (int word = 0; word < 4; ++word) {
      // Rows n = kPer q + h, q = 0 .. 3: a 4 x 4 transpose, first within pairs of quarters, then between pairs.
      const auto ab = __builtin_amdgcn_permlane16_swap(v[h][word], v[kPer + h][word], false, false);
      const auto cd = __builtin_amdgcn_permlane16_swap(v[2 * kPer + h][word], v[3 * kPer + h][word], false, false);
      const auto ac = __builtin_amdgcn_permlane32_swap(ab[0], cd[0], false, false);
      const auto bd = __builtin_amdgcn_permlane32_swap(ab[1], cd[1], false, false);
      to[4 * h][word] = ac[0];
      to[4 * h + 1][word] = bd[0];
      to[4 * h + 2][word] = ac[1];
      to[4 * h + 3][word] = bd[1];
    }
#pragma unroll
  for (int n = 0; n < kUnits; ++n) v[n] = to[n];
}

// LDS accesses beside copies in flight, each block with its own wait (the compiler would wait for every copy).
__device__ __forceinline__ void lds_two(u32x4 (&v)[2], uint32_t a, uint32_t b) {
  asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)" : "=&v"(v[0]), "=&v"(v[1]) : "v"(a), "v"(b) : "memory");
}
__device__ __forceinline__ uint32_t lds_scales(uint32_t at) {
  uint32_t v;
  asm volatile("ds_read_u16 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(at) : "memory");
  return v;
}
__device__ __forceinline__ void lds_write16(uint32_t at, const f32x4& v) {
  // (Sums of a matrix instruction: the compiler does not wait for them before an asm block.)
  asm volatile("s_nop 15\n\ts_nop 3\n\tds_write_b128 %0, %1" ::"v"(at), "v"(v) : "memory");
}
__device__ __forceinline__ uint32_t lds_word(uint32_t at) {
  uint32_t v;
  asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(at) : "memory");
  return v;
}
// Words at `at`, at + 1024, ... (one for each of eight waves), summed in that order.
__device__ __forceinline__ float lds_sum8(uint32_t at) {
  float v[8];
  asm volatile(
      "ds_read_b32 %0, %8\n\t"
      "ds_read_b32 %1, %8 offset:0x400\n\t"
      "ds_read_b32 %2, %8 offset:0x800\n\t"
      "ds_read_b32 %3, %8 offset:0xc00\n\t"
      "ds_read_b32 %4, %8 offset:0x1000\n\t"
      "ds_read_b32 %5, %8 offset:0x1400\n\t"
      "ds_read_b32 %6, %8 offset:0x1800\n\t"
      "ds_read_b32 %7, %8 offset:0x1c00\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(at)
      : "memory");
  float sum = v[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) sum += v[i];
  return sum;
}

// Copies of one stage of 16 weight rows: eight rows of 128 bytes each, unit u of row r at u ^ (r & 7), and of MXFP4
// the eight scale bytes of each row (lanes 32 to 63 fetch nothing).
template <int kType>
struct Copier {
  uint32_t at[2], unit, scale_at;  // the lane's offsets of the first and the second eight rows; its unit's byte in a stage
  uint32_t row_bytes, blocks4;     // of a weight row: bytes, and words of scales

  // Rows r and 8 + r of the 16 are `row0` + r and `row1` + r, in rows of `k`.
  __device__ __forceinline__ Copier(int k, uint32_t row0, uint32_t row1) {
    const int lane = threadIdx.x & 63, r8 = lane >> 3;
    row_bytes = uint32_t(Format<kType>::row_bytes(k));
    unit = uint32_t(((lane & 7) ^ r8) * 16);
    at[0] = (row0 + r8) * row_bytes + unit;
    at[1] = (row1 + r8) * row_bytes + unit;
    blocks4 = uint32_t(k / mx::kBlock / 4);
    const uint32_t r = lane >> 1;
    scale_at = lane < 32 ? ((r < 8 ? row0 + r : row1 + r - 8) * blocks4 + (lane & 1)) * 4 : kPast;
  }
  // Stage `stage` (`live`: there is one) into `slot`. Past the end of a row the buffers give zeros.
  __device__ __forceinline__ void copy(__amdgpu_buffer_rsrc_t w, __amdgpu_buffer_rsrc_t s, int stage, bool live, char* slot) const {
    const uint32_t past = live && stage * 128 + unit < row_bytes ? 0u : kPast;
    const uint32_t base = live ? stage * 128 : 0;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(w, (LdsPtr)slot, 16, at[0] | past, base, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(w, (LdsPtr)(slot + 1024), 16, at[1] | past, base, 0, 0);
    if constexpr (kType == kMxfp4) {
      const uint32_t gone = live && stage * 2 + (threadIdx.x & 1) < blocks4 ? 0u : kPast;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(s, (LdsPtr)(slot + kSlotWeights), 4, scale_at | gone, live ? stage * 8 : 0, 0, 0);
    }
  }
};

// One stage: 16 weight rows (in the slot) times kT tiles of 16 columns of x (units of a lane's quarter of the stage's k).
// `scale`: FP8, of the lane's weight rows. kMasked: only columns whose token (c % 8) is in `mask` take part in the stage, so that
// what is not finite in an expert's weights (NaN times zero is NaN) reaches no other token.
template <int kType, int kT, bool kMasked>
__device__ __forceinline__ void contract(uint32_t slot, const u32x4 (&x)[kT][Format<kType>::kUnits], float scale, uint32_t mask, f32x4 (&acc)[kT]) {
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  u32x4 w[2];
  lds_two(w, slot + c * 128 + ((2 * q) ^ (c & 7)) * 16, slot + c * 128 + ((2 * q + 1) ^ (c & 7)) * 16);
  constexpr bool kApart = kMasked || kType == kFp8;  // a stage's products from zero
  f32x4 sum[kT];
#pragma unroll
  for (int t = 0; t < kT; ++t) sum[t] = kApart ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[t];
  auto multiply = [&](const u32x4& a, int j) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < kT; ++t) sum[t] = lf::mfma16(vec_bf16x8(a), vec_bf16x8(x[t][j]), sum[t]);
  };
  if constexpr (kType == kBf16) {
#pragma unroll
    for (int j = 0; j < 2; ++j) multiply(w[j], j);
  } else if constexpr (kType == kFp8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) multiply(fp8::decode8(w[j >> 1][j % 2 * 2], w[j >> 1][j % 2 * 2 + 1]), j);
  } else {
    const uint32_t scales = lds_scales(slot + kSlotWeights + c * 8 + 2 * q);
#pragma unroll
    for (int j = 0; j < 8; ++j) multiply(mx::decode8(w[j >> 2][j & 3], mx::scale_f32(j < 4 ? scales & 0xffu : scales >> 8)), j);
  }
  const bool in = !kMasked || (mask >> (c & 7) & 1);
#pragma unroll
  for (int t = 0; t < kT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = kType == kFp8 ? fmaf(scale, sum[t][e], acc[t][e]) : kApart ? acc[t][e] + sum[t][e] : sum[t][e];
      acc[t][e] = in ? v : acc[t][e];
    }
}

// ---------------------------------------------------------------------------
// Routing by one workgroup: chosen experts in order, with the masks of their tokens and their first rows
// in expert order; weights by row.
// ---------------------------------------------------------------------------
struct Routing {
  uint32_t mask[kMostExperts];   // by expert
  int first[kMostExperts];
  uint32_t rank[kFewTokens * 64];  // of a few tokens: a byte each for a lane's experts
  int used;
  int4 chosen[kMostChoices];     // expert, first row, mask
  float weight[kMostChoices];
};

// The tables, from masks that a barrier has passed. Each wave writes them for itself (all the same), so that it needs
// no barrier to read what it wrote.
__device__ __forceinline__ void tabulate(Routing& r) {
  const int lane = threadIdx.x & 63;
  // Places: counts of chosen experts and of choices before each of the lane's four experts, in one word.
  constexpr int kPer = kMostExperts / 64;
  uint32_t mask[kPer];
  int mine = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    mask[i] = r.mask[kPer * lane + i];
    mine += (mask[i] != 0) << 16 | __popc(mask[i]);
  }
  const int sum = scan_lanes(mine);
  r.used = __builtin_amdgcn_readlane(sum, 63) >> 16;
  int before = sum - mine;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    r.first[kPer * lane + i] = before & 0xffff;
    if (mask[i]) r.chosen[before >> 16] = make_int4(kPer * lane + i, before & 0xffff, int(mask[i]), 0);
    before += (mask[i] != 0) << 16 | __popc(mask[i]);
  }
}

// (Weights are read behind the barrier of an item's sums.)
__device__ __forceinline__ void keep_weight(Routing& r, int t, int e, float weight) {
  r.weight[r.first[e] + __popc(r.mask[e] & ((1u << t) - 1))] = weight;
}

// One or two tokens: the rank of every expert of a token by counting those before it, as many waves a token
// as there are, each against a part of the experts. (Rounds of maxima, as for more tokens, are a chain of a few
// hundred clocks each, but as long for 16 tokens as for one: routing takes 6200 clocks here, of 4 tokens it took
// 13500, in rounds 8200.)
template <int kPer>
__device__ __forceinline__ void route_few(const MlpParams& p, Routing& r) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int share = p.tokens == 1 ? kWaves : kWaves / kFewTokens;  // waves of a token
  const int t = wave / share, part = wave & (share - 1);
  const bool live = t < p.tokens;  // (always: each of one or two tokens has its waves)
  float value[kPer];
  load_logits<64>(p.logits, p.fp32, p.logits_stride, p.experts, t, live, value);
  if (threadIdx.x < kMostExperts) r.mask[threadIdx.x] = 0;
  if (threadIdx.x < kFewTokens * 64) r.rank[threadIdx.x] = 0;
  uint32_t key[kPer];
  int rank[kPer];
  bool odd = false;  // NaN or +inf
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    key[i] = order_key(value[i]);
    rank[i] = 0;
    odd |= !(value[i] < __builtin_huge_valf());
  }
  const bool bad = __ballot(odd) != 0;
  const int lanes = 64 / share;
  for (int l0 = part * lanes; l0 < (part + 1) * lanes; l0 += 2) {
#pragma unroll
    for (int l1 = 0; l1 < 2; ++l1)
#pragma unroll
      for (int n = 0; n < kPer; ++n) {  // expert l + 64 n against the lane's
        const int l = l0 + l1;
        const uint32_t other = uint32_t(__builtin_amdgcn_readlane(int(key[n]), l));
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          rank[i] += n < i ? other >= key[i] : n > i ? other > key[i] : other > key[i] || (other == key[i] && l < lane);
      }
  }
  wait_vm<0>();  // (x has come too)
  __syncthreads();
  // (Whole numbers below 256: no order shows, and no byte reaches the next.)
  uint32_t packed = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) packed |= uint32_t(rank[i]) << (8 * i);
  atomicAdd(&r.rank[t * 64 + lane], packed);
  __syncthreads();
  packed = r.rank[t * 64 + lane];
#pragma unroll
  for (int i = 0; i < kPer; ++i) rank[i] = int(packed >> (8 * i) & 0xffu);
  bool mine[kPer];
  float weight[kPer];
  if (live && part == 0) {
    float peak = 0.f, total = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      mine[i] = rank[i] < p.top && key[i] != 0;
      const uint64_t first = __ballot(rank[i] == 0);
      if (first) peak = __uint_as_float(uint32_t(__builtin_amdgcn_readlane(int(__float_as_uint(key_value(key[i]))), __builtin_ctzll(first))));
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      weight[i] = key[i] != 0 ? expf(key_value(key[i]) - peak) : 0.0f;
      total += mine[i] || !p.renormalize ? weight[i] : 0.0f;
    }
    total = sum_across<64>(total);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      weight[i] = bad ? __builtin_nanf("") : weight[i] / total;
      if (mine[i]) atomicOr(&r.mask[lane + 64 * i], 1u << t);  // (a token chooses an expert once: no order shows)
    }
  }
  __syncthreads();
  tabulate(r);
  if (live && part == 0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (mine[i]) keep_weight(r, t, lane + 64 * i, weight[i]);
  }
}

// More tokens: 16 lanes each.
template <int kPer>
__device__ __forceinline__ void route_many(const MlpParams& p, Routing& r) {
  const int t = threadIdx.x >> 4, j = threadIdx.x & 15;
  if (threadIdx.x < kMostExperts) r.mask[threadIdx.x] = 0;
  float value[kPer];
  load_logits<16>(p.logits, p.fp32, p.logits_stride, p.experts, t, t < p.tokens, value);
  Choice c{-1, 0.f};
  // (A wave as a whole: its lanes take maxima together.)
  if (int(threadIdx.x & ~63u) / 16 < p.tokens) c = choose_experts<true, 16>(value, p.top, p.renormalize);
  const bool live = t < p.tokens && j < p.top && c.expert >= 0;
  wait_vm<0>();  // (x has come too, if it was asked for)
  __syncthreads();
  if (live) atomicOr(&r.mask[c.expert], 1u << t);
  __syncthreads();
  tabulate(r);
  if (live) keep_weight(r, t, c.expert, p.positions ? 1.0f : c.weight);
  if (p.positions && blockIdx.x == 0) {
    if (t < p.tokens && j < p.top) {
      p.positions[t * p.top + j] = live ? r.first[c.expert] + __popc(r.mask[c.expert] & ((1u << t) - 1)) : -1;
      p.weights[t * p.top + j] = live ? c.weight : 0.0f;
    }
    if (threadIdx.x < kMostExperts) {
      const int e = threadIdx.x, first = r.first[e], end = first + __popc(r.mask[e]);
      if (e < p.experts) p.offsets[e] = first;
      if (e == p.experts - 1) p.offsets[e + 1] = end;
    }
  }
}

__device__ __forceinline__ void route(const MlpParams& p, Routing& r) {
  if (p.tokens <= kFewTokens) {
    if (p.experts <= 128) route_few<2>(p, r);
    else route_few<4>(p, r);
  } else {
    if (p.experts <= 128) route_many<8>(p, r);
    else route_many<16>(p, r);
  }
}

// ---------------------------------------------------------------------------
// First launch: routing, gate and up products, SwiGLU.
// ---------------------------------------------------------------------------
template <int kType, int kT, int kStages>
struct GateUp {
  using F = Format<kType>;
  static constexpr bool kTwo = kT == 1 && kStages * F::kUnits <= 16;  // two workgroups on a CU: 64 registers of x
  static constexpr int kRing = kTwo ? 3 : 5;                    // stages
  static constexpr int kRed = 2 * kT * kWaves * 1024;
  static constexpr int kLds = kWaves * kRing * F::kSlot + kRed;
};

template <int kType, int kT, int kStages>
__global__ __launch_bounds__(kThreads, (GateUp<kType, kT, kStages>::kTwo ? 4 : 2)) void gate_up_kernel(MlpParams p) {
  using F = Format<kType>;
  using G = GateUp<kType, kT, kStages>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ Routing routing;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, q = lane >> 4;
  const int stages = int((F::row_bytes(p.hidden) + 127) / 128);
  const int mine = stages > wave ? (stages - wave + kWaves - 1) / kWaves : 0;  // stages wave, wave + 8, ...

  // x: unit n of a lane holds k 8 n .. of its quarter of the stage.
  u32x4 x[kStages][kT][F::kUnits];
  const auto xbuf = buffer(p.x, uint32_t((p.tokens - 1) * p.x_row + p.hidden * 2));
  // A few rows go through LDS (where the weights come later) while the tokens are routed: KiB by KiB, unit u of row t at
  // u ^ t. (A load of 16 rows takes the address unit as long for one row as for 16.)
  const int pieces = (p.hidden * 2 + 1023) / 1024, pitch = pieces * 1024;
  const bool through_lds = kT == 1 && p.tokens * pitch <= G::kLds;
  if (through_lds)
    for (int t = 0; t < p.tokens; ++t)
      for (int piece = wave; piece < pieces; piece += kWaves) {
        const int at = piece * 1024 + (lane ^ t) * 16;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xbuf, (LdsPtr)(lds + t * pitch + piece * 1024), 16,
                                                 at < p.hidden * 2 ? uint32_t(t * p.x_row) + at : kPast, 0, 0, 0);
      }
  route(p, routing);
  if (through_lds) {  // (tokens past the last one: its row again, in columns that nobody stores)
    const int t = min(c, p.tokens - 1);
#pragma unroll
    for (int i = 0; i < kStages; ++i)
      if (i < mine)
#pragma unroll
        for (int n = 0; n < F::kUnits; ++n) {
          const int unit = ((wave + kWaves * i) * F::kStage + q * (F::kStage / 4)) / 8 + n;
          x[i][0][n] = *reinterpret_cast<const u32x4*>(lds + t * pitch + (unit ^ t) * 16);
        }
    lds_barrier();
  }

  const int used = __builtin_amdgcn_readfirstlane(routing.used);
  if (blockIdx.x == 0 && p.table) {
    if (threadIdx.x == 0) p.table[0] = make_int4(used, 0, 0, 0);
    if (int(threadIdx.x) < used) p.table[1 + threadIdx.x] = routing.chosen[threadIdx.x];
  }

  // Items: eight columns of a chosen expert each.
  const int groups = p.inter / 8, items = used * groups;
  const int64_t row_bytes = F::row_bytes(p.hidden);
  const uint32_t extent = uint32_t((p.inter + 8) * row_bytes);
  const int blocks = int(fp8::blocks_of(p.hidden));
  const Copier<kType> copier(p.hidden, 0, p.inter);
  char* const ring = lds + wave * G::kRing * F::kSlot;
  const uint32_t ring_at = lds_addr(ring), red_at = lds_addr(lds + kWaves * G::kRing * F::kSlot);
  const uint32_t chosen_at = lds_addr(&routing.chosen[0]), weight_at = lds_addr(&routing.weight[0]);

  // Items blockIdx.x, + gridDim.x, ... as (chosen expert, group of columns).
  struct At {
    int item, u, group;
  };
  const int jump_u = gridDim.x / groups, jump_group = gridDim.x - jump_u * groups;
  auto next = [&](At& a) __attribute__((always_inline)) {
    a.item += gridDim.x;
    a.u += jump_u;
    a.group += jump_group;
    if (a.group >= groups) a.group -= groups, ++a.u;
  };
  At to{int(blockIdx.x), int(blockIdx.x) / groups, 0};
  to.group = to.item - to.u * groups;
  At at = to;
  // The stage that is copied next: of item `to`, the wave's stage number `step`.
  int step = 0, in = 0;
  __amdgpu_buffer_rsrc_t wbuf = buffer(p.gate_up, 0), sbuf = buffer(p.gate_up_s, 0);
  auto aim = [&]() __attribute__((always_inline)) {  // buffers of item `to`
    if (to.item >= items) return;
    const int e = __builtin_amdgcn_readfirstlane(int(lds_word(chosen_at + to.u * 16)));
    const int64_t row = int64_t(e) * 2 * p.inter + to.group * 8;
    wbuf = buffer(p.gate_up + row * row_bytes, extent);
    if constexpr (kType == kMxfp4) sbuf = buffer(p.gate_up_s + row * (p.hidden / mx::kBlock), uint32_t(p.inter + 8) * (p.hidden / mx::kBlock));
  };
  auto copy_next = [&]() __attribute__((always_inline)) {
    copier.copy(wbuf, sbuf, wave + kWaves * step, to.item < items, ring + in * F::kSlot);
    in = in + 1 == G::kRing ? 0 : in + 1;
    if (++step == mine) {
      step = 0;
      next(to);
      aim();
    }
  };
  if (mine > 0) {
    aim();
    for (int n = 0; n < G::kRing - 1; ++n) copy_next();
  }
  if (!through_lds) {
    // Loaded with quarter after quarter of a load's 64 bytes of a row, if the lane's own lie further apart (16 rows of
    // 4 x 16 bytes at 128 bytes from one another come four times over from L2: 10 us of 16 tokens)...
#pragma unroll
    for (int i = 0; i < kStages; ++i)
#pragma unroll
      for (int t = 0; t < kT; ++t)
#pragma unroll
        for (int n = 0; n < F::kUnits; ++n) {
          const int token = 16 * t + c, k = (wave + kWaves * i) * F::kStage + (kType == kBf16 ? q * 16 + 8 * n : 32 * n + 8 * q);
          const uint32_t from = token < p.tokens && k < p.hidden ? uint32_t(token * p.x_row) + k * 2 : kPast;
          x[i][t][n] = __builtin_amdgcn_raw_buffer_load_b128(xbuf, from, 0, 0);
        }
    wait_vm<0>();  // (or the compiler would wait for x, and every copy, in the loop)
    if constexpr (kType != kBf16) {
      // ... and exchanged between the quarters: unit j of quarter q is load kUnits / 4 q + j / 4 of quarter j % 4.
#pragma unroll
      for (int i = 0; i < kStages; ++i)
#pragma unroll
        for (int t = 0; t < kT; ++t) transpose_quarters<F::kUnits>(x[i][t]);
    }
  }

  int out = 0, turn = 0;
  for (; at.item < items; next(at), turn ^= 1) {
    const int u = at.u, column = at.group * 8;
    const float *gate_s = nullptr, *up_s = nullptr;
    float gs = 0.f, us = 0.f;
    if constexpr (kType == kFp8) {
      const int e = __builtin_amdgcn_readfirstlane(int(lds_word(chosen_at + u * 16)));
      const int64_t first = int64_t(e) * fp8::blocks_of(2 * p.inter);
      gate_s = p.gate_up_s8 + (first + column / fp8::kBlock) * blocks;
      up_s = p.gate_up_s8 + (first + (p.inter + column) / fp8::kBlock) * blocks;
      gs = sload(gate_s, min(wave, blocks - 1)), us = sload(up_s, min(wave, blocks - 1));
    }
    f32x4 acc[kT];
#pragma unroll
    for (int t = 0; t < kT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      if (i < mine) {
        wait_vm<(G::kRing - 2) * F::kCopies>();
        copy_next();  // (into the slot whose reads are done)
        float scale = 0.f;
        if constexpr (kType == kFp8) {
          scale = q >= 2 ? us : gs;
          const int ahead = min(wave + kWaves * (i + 1), blocks - 1);
          gs = sload(gate_s, ahead), us = sload(up_s, ahead);
        }
        contract<kType, kT, false>(ring_at + out * F::kSlot, x[i], scale, 0u, acc);
        out = out + 1 == G::kRing ? 0 : out + 1;
      }
    }
    // Sums as [turn][tile][wave][token][row]; two places in turn, so one barrier an item.
    const uint32_t red = red_at + turn * (G::kRed / 2);
#pragma unroll
    for (int t = 0; t < kT; ++t) lds_write16(red + (t * kWaves + wave) * 1024 + c * 64 + q * 16, acc[t]);
    lds_barrier();
    if (threadIdx.x < 128 * kT) {
      const int token = threadIdx.x >> 3, r = threadIdx.x & 7;
      const uint32_t from = red + (token >> 4) * kWaves * 1024 + (token & 15) * 64 + r * 4;
      const uint32_t mask = lds_word(chosen_at + u * 16 + 8);
      if (mask >> token & 1) {
        const int row = int(lds_word(chosen_at + u * 16 + 4)) + __popc(mask & ((1u << token) - 1));
        const float g = lds_sum8(from), up = lds_sum8(from + 32);
        uint16_t* h = p.h + int64_t(row) * 2 * p.inter + column + r;
        split_pair(silu_mul_f32(g, up) * __uint_as_float(lds_word(weight_at + row * 4)), h[0], h[p.inter]);
      }
    }
  }
  wait_vm<0>();  // (copies past the last item are on their way into this workgroup's LDS)
}

// ---------------------------------------------------------------------------
// Second launch: down products over all chosen experts at once.
// ---------------------------------------------------------------------------
constexpr int kDownRing = 4;

template <int kType, int kW>
constexpr int down_lds() {
  return kW * kDownRing * Format<kType>::kSlot + kW * 1024;
}

template <int kType, int kW>
__global__ __launch_bounds__(64 * kW, 2) void down_kernel(MlpParams p) {
  using F = Format<kType>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, q = lane >> 4;
  const int column = blockIdx.x * 16;
  const int64_t row_bytes = F::row_bytes(p.inter);
  const int per = int((row_bytes + 127) / 128);  // stages of an expert
  const int used = sload(reinterpret_cast<const int*>(p.table), 0), total = used * per;
  const int blocks = int(fp8::blocks_of(p.inter));
  const Copier<kType> copier(p.inter, 0, 8);
  const uint32_t extent = uint32_t((p.hidden - column) * row_bytes);  // (rows past the last one: zeros)
  char* const ring = lds + wave * kDownRing * F::kSlot;
  const uint32_t ring_at = lds_addr(ring), red_at = lds_addr(lds + kW * kDownRing * F::kSlot);

  // Stages wave, wave + kW, ... of the experts' one after another, each as (chosen expert, stage).
  struct At {
    int n, u, s;
  };
  const int jump_u = kW / per, jump_s = kW % per;
  auto next = [&](At& a) __attribute__((always_inline)) {
    a.n += kW;
    a.u += jump_u;
    a.s += jump_s;
    if (a.s >= per) a.s -= per, ++a.u;
  };
  // (Past the last one whatever is there: copies and rows of x are zeros then. So no entry waits for their number.)
  auto entry = [&](int u) { return sload(reinterpret_cast<const i32x4*>(p.table), 1 + min(u, kTable - 1)); };
  At to{wave, wave / per, wave % per}, x_at = to, at = to;
  int in = 0, out = 0;
  auto copy_next = [&]() __attribute__((always_inline)) {
    const int64_t row = int64_t(entry(to.u)[0]) * p.hidden + column;
    const auto wbuf = buffer(p.down + row * row_bytes, extent);
    auto sbuf = wbuf;
    if constexpr (kType == kMxfp4) sbuf = buffer(p.down_s + row * (p.inter / mx::kBlock), uint32_t(p.hidden - column) * (p.inter / mx::kBlock));
    copier.copy(wbuf, sbuf, to.s, to.n < total, ring + in * F::kSlot);
    in = in + 1 == kDownRing ? 0 : in + 1;
    next(to);
  };
  const auto hbuf = buffer(p.h, uint32_t(p.tokens) * p.top * p.inter * 4);
  auto load_x = [&](u32x4 (&x)[1][F::kUnits]) __attribute__((always_inline)) {  // returns the mask of the stage's tokens
    const i32x4 chosen = entry(x_at.u);
    const uint32_t mask = x_at.n < total ? uint32_t(chosen[2]) : 0u;
    const int k0 = x_at.s * F::kStage + q * (F::kStage / 4);
    const bool whole = (x_at.s + 1) * F::kStage <= p.inter;
    // Column c: token c % 8, of the pairs the high half before column 8, then the low one.
    const int token = c & 7;
    const uint32_t row = uint32_t((chosen[1] + __popc(mask & ((1u << token) - 1))) * 2 + (c >> 3)) * uint32_t(p.inter) + k0;
    const uint32_t from = mask >> token & 1 ? row * 2 : kPast;
#pragma unroll
    for (int n = 0; n < F::kUnits; ++n)
      x[0][n] = __builtin_amdgcn_raw_buffer_load_b128(hbuf, whole || k0 + 8 * n < p.inter ? from + 16 * n : kPast, 0, 0);
    next(x_at);
    return mask;
  };
  f32x4 acc[1] = {{0.f, 0.f, 0.f, 0.f}};
  auto step = [&](const u32x4 (&x)[1][F::kUnits], uint32_t mask, u32x4 (&ahead)[1][F::kUnits]) __attribute__((always_inline)) {
    // Behind the copies of this stage went those of kDownRing - 2 more, and as many stages of x.
    wait_vm<(kDownRing - 2) * (F::kCopies + F::kUnits)>();
    const uint32_t mask_ahead = load_x(ahead);
    asm volatile("" ::: "memory");
    copy_next();
    float scale = 0.f;
    if constexpr (kType == kFp8) {
      const int64_t block = int64_t(entry(at.u)[0]) * fp8::blocks_of(p.hidden) + column / fp8::kBlock;
      scale = sload(p.down_s8 + block * blocks, at.s);
    }
    contract<kType, 1, true>(ring_at + out * F::kSlot, x, scale, mask, acc);
    out = out + 1 == kDownRing ? 0 : out + 1;
    next(at);
    return mask_ahead;
  };
  u32x4 x0[1][F::kUnits], x1[1][F::kUnits];
  if (wave < total) {
    // (x behind all copies but the last, as in every step: what the compiler waits for before x is the same then.)
    for (int n = 0; n < kDownRing - 2; ++n) copy_next();
    asm volatile("" ::: "memory");
    uint32_t mask = load_x(x0);
    asm volatile("" ::: "memory");
    copy_next();
    wait_vm<(kDownRing - 2) * F::kCopies + F::kUnits>();  // (the first stage; the second has two of x behind it)
    while (at.n < total) {
      mask = step(x0, mask, x1);
      if (at.n >= total) break;
      mask = step(x1, mask, x0);
    }
  }
  lds_write16(red_at + wave * 1024 + c * 64 + q * 16, acc[0]);
  wait_vm<0>();
  lds_barrier();
  if (threadIdx.x < 16 * kMostTokens) {
    const int token = threadIdx.x >> 4, n = column + (threadIdx.x & 15);
    if (token >= p.tokens || n >= p.hidden) return;
    const uint32_t high = red_at + threadIdx.x * 4, low = high + 16 * kMostTokens * 4;
    float sum = lds_sum8(high), rest = lds_sum8(low);
    if constexpr (kW == 16) sum += lds_sum8(high + 8 * 1024), rest += lds_sum8(low + 8 * 1024);
    sum = join_pair(sum, rest);
    if (p.base) sum += bf16_to_f32(p.base[token * p.base_stride + n]);
    p.y[token * p.y_stride + n] = uint16_t(f32_to_bf16(sum));
  }
}

// ---------------------------------------------------------------------------

template <class K>
int launch(K kernel, unsigned grid, unsigned threads, unsigned lds, const MlpParams& p, hipStream_t stream) {
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), lds, stream, p);
  LF_HIP(hipGetLastError());
  return kOk;
}

template <int kType, int kT, int kStages>
int launch_gate_up(const MlpParams& p, hipStream_t stream) {
  using G = GateUp<kType, kT, kStages>;
  return launch(gate_up_kernel<kType, kT, kStages>, G::kTwo ? 512 : 256, kThreads, G::kLds, p, stream);
}

// Registers of x: 32, 64 or (one workgroup a CU) all of 128.
template <int kType, int kT>
int launch_gate_up(const MlpParams& p, hipStream_t stream) {
  const int per_wave = int(((Format<kType>::row_bytes(p.hidden) + 127) / 128 + kWaves - 1) / kWaves);
  constexpr int kAll = 32 / (kT * Format<kType>::kUnits);
  if constexpr (kAll >= 8)
    if (per_wave <= kAll / 4) return launch_gate_up<kType, kT, kAll / 4>(p, stream);
  if (per_wave <= kAll / 2) return launch_gate_up<kType, kT, kAll / 2>(p, stream);
  return launch_gate_up<kType, kT, kAll>(p, stream);
}

template <int kType>
int launch_gate_up(const MlpParams& p, hipStream_t stream) {
  if constexpr (kType != kMxfp4)
    if (p.tokens > 16) return launch_gate_up<kType, 2>(p, stream);
  return launch_gate_up<kType, 1>(p, stream);
}

template <int kType>
int launch_down(const MlpParams& p, hipStream_t stream) {
  const unsigned grid = unsigned((p.hidden + 15) / 16);
  // Few workgroups get twice the waves: 64 experts, top 4, 2048 x 1024, 8 tokens FP8 39.6 us with them and 43.7 without, bf16
  // 69.2 and 71.0; 32 experts, 1024 x 2048, FP8 48.6 and 54.0, bf16 70.3 and 77.9. (Not of MXFP4 weights, whose bytes are few: a
  // token 13.8 and 13.1, eight tokens 30.9 and 31.4.)
  if constexpr (kType != kMxfp4)
    if (grid <= 160) return launch(down_kernel<kType, 16>, grid, 1024, down_lds<kType, 16>(), p, stream);
  return launch(down_kernel<kType, 8>, grid, 512, down_lds<kType, 8>(), p, stream);
}

int64_t padded16(int64_t n) { return (n + 15) / 16 * 16; }

// What the first kernel takes, and (up to kMostTokens) the second.
bool first_fits(int64_t tokens, int32_t experts, int32_t top, int64_t hidden, int64_t inter, int32_t type) {
  if (tokens > kMostFirst || experts > kMostExperts || top > kMostTop || tokens * top > kMostChoices) return false;
  if (tokens > 16 && (type == LF_EXPERT_MXFP4 || (type == LF_EXPERT_FP8 && hidden <= 2048))) return false;
  if (type == LF_EXPERT_MXFP4 && (hidden % 128 || inter % 128)) return false;
  // x of a wave's stages in 128 registers; an expert's weights within 31 bits.
  return hidden <= (tokens <= 16 ? 8192 : 4096) && inter <= (int64_t(1) << 20) && (hidden + 16) * (inter + 16) * 2 < (int64_t(1) << 31);
}

bool fused_fits(int64_t tokens, int32_t experts, int32_t top, int64_t hidden, int64_t inter, int32_t type) {
  return tokens <= kMostTokens && first_fits(tokens, experts, top, hidden, inter, type);
}

// (32-bit offsets of x in the first kernel.)
bool x_within(const lf_expert_mlp_call& a) {
  return a.tokens == 1 || a.x_stride < ((int64_t(1) << 30) - a.hidden) / (a.tokens - 1);
}

MlpParams params_of(const lf_expert_mlp_call& a) {
  MlpParams p{};
  p.x = static_cast<const char*>(a.x);
  p.x_row = a.x_stride * 2;
  p.logits = a.logits;
  p.logits_stride = a.logits_stride;
  p.fp32 = a.fp32 ? 1 : 0;
  p.tokens = int32_t(a.tokens);
  p.experts = a.experts;
  p.top = a.top;
  p.renormalize = a.renormalize ? 1 : 0;
  p.hidden = int32_t(a.hidden);
  p.inter = int32_t(a.inter);
  p.gate_up = static_cast<const char*>(a.gate_up);
  p.down = static_cast<const char*>(a.down);
  if (a.type == LF_EXPERT_FP8) {
    p.gate_up_s8 = static_cast<const float*>(a.gate_up_scales);
    p.down_s8 = static_cast<const float*>(a.down_scales);
  } else {
    p.gate_up_s = static_cast<const uint8_t*>(a.gate_up_scales);
    p.down_s = static_cast<const uint8_t*>(a.down_scales);
  }
  p.base = a.base;
  p.base_stride = a.base_stride;
  p.y = a.y;
  p.y_stride = a.y_stride;
  return p;
}

int launch_first(const MlpParams& p, int32_t type, hipStream_t stream) {
  return type == LF_EXPERT_BF16    ? launch_gate_up<kBf16>(p, stream)
         : type == LF_EXPERT_MXFP4 ? launch_gate_up<kMxfp4>(p, stream)
                                   : launch_gate_up<kFp8>(p, stream);
}

// Parts of the workspace of a chain, each 16-byte aligned.
struct ChainSpace {
  int64_t weights, chosen, offsets, tokens, positions, scratch, h, rows, bytes;
  ChainSpace(int64_t count, int32_t experts, int32_t top, int64_t hidden, int64_t inter) {
    int64_t at = 0;
    auto part = [&](int64_t size) { return at += padded16(size), at - padded16(size); };
    const int64_t choices = count * top;
    weights = part(choices * 4);
    chosen = part(choices * 4);
    offsets = part((experts + 1) * 4);
    tokens = part(choices * 4);
    positions = part(choices * 4);
    scratch = part(lf_route_experts_workspace_size(count, experts));
    h = part(choices * inter * 4);
    rows = part(choices * hidden * 4);
    bytes = at;
  }
};

int launch_chain(const lf_expert_mlp_call& a, char* space, hipStream_t stream) {
  const ChainSpace part(a.tokens, a.experts, a.top, a.hidden, a.inter);
  const int64_t choices = a.tokens * a.top;
  auto* weights = reinterpret_cast<float*>(space + part.weights);
  auto* offsets = reinterpret_cast<int32_t*>(space + part.offsets);
  auto* tokens = reinterpret_cast<int32_t*>(space + part.tokens);
  auto* positions = reinterpret_cast<int32_t*>(space + part.positions);
  auto* h = reinterpret_cast<uint16_t*>(space + part.h);
  // The first kernel, or routing and product: see kMostFirst.
  if (first_fits(a.tokens, a.experts, a.top, a.hidden, a.inter, a.type) && x_within(a)) {
    MlpParams p = params_of(a);
    p.h = h;
    p.offsets = offsets;
    p.positions = positions;
    p.weights = weights;
    if (const int rc = launch_first(p, a.type, stream)) return rc;
  } else {
    if (const int rc = lf_route_experts(a.logits, a.fp32, a.tokens, a.experts, a.logits_stride, a.top, a.renormalize, weights,
                                        reinterpret_cast<int32_t*>(space + part.chosen), offsets, tokens, positions,
                                        space + part.scratch, part.h - part.scratch, stream))
      return rc;
    lf_expert_product g{};
    g.x = a.x;
    g.x_stride = a.x_stride;
    g.x_rows = a.tokens;
    g.w = a.gate_up;
    g.offsets = offsets;
    g.tokens = tokens;
    g.y = h;
    g.k = a.hidden;
    g.y_stride = a.inter;
    g.rows = choices;
    g.n = 2 * a.inter;
    g.experts = a.experts;
    g.swiglu = 1;
    if (a.type == LF_EXPERT_FP8) g.w_fp8_scales = static_cast<const float*>(a.gate_up_scales);
    else g.w_scales = static_cast<const uint8_t*>(a.gate_up_scales);
    if (const int rc = launch_pairs(g, kSplit, stream)) return rc;
  }
  lf_expert_product d{};
  d.x = h;
  d.x_stride = a.inter;
  d.x_rows = d.rows = 2 * choices;
  d.w = a.down;
  d.offsets = offsets;
  d.y = reinterpret_cast<uint16_t*>(space + part.rows);
  d.y_stride = d.n = a.hidden;
  d.k = a.inter;
  d.experts = a.experts;
  if (a.type == LF_EXPERT_FP8) d.w_fp8_scales = static_cast<const float*>(a.down_scales);
  else d.w_scales = static_cast<const uint8_t*>(a.down_scales);
  if (const int rc = launch_pairs(d, kJoin, stream)) return rc;
  return combine_f32(reinterpret_cast<const float*>(space + part.rows), choices, positions, weights, a.tokens, a.top, a.hidden,
                     a.base, a.base_stride, a.y, a.y_stride, stream);
}

}  // namespace
}  // namespace expert
}  // namespace lf

// Bytes of workspace, or -1 for what this entry point does not take.
extern "C" int64_t lf_expert_mlp_workspace_size(int64_t tokens, int32_t experts, int32_t top, int64_t hidden, int64_t inter, int32_t type) {
  using namespace lf::expert;
  if (type < LF_EXPERT_BF16 || type > LF_EXPERT_FP8 || tokens < 1 || experts < 1 || experts > 1024 || top < 1 || top > 64 || top > experts)
    return -1;
  const int64_t unit = type == LF_EXPERT_BF16 ? 8 : type == LF_EXPERT_FP8 ? 16 : 32;
  if (hidden < 1 || inter < 1 || hidden % unit || inter % unit || (type == LF_EXPERT_FP8 && inter % lf::fp8::kBlock)) return -1;
  if (hidden >= (int64_t(1) << 24) || inter >= (int64_t(1) << 24)) return -1;
  if (fused_fits(tokens, experts, top, hidden, inter, type)) return padded16(tokens * top * inter * 4) + 16 * (1 + kTable);
  if (tokens > kMostEach * int64_t(experts) / top) return -1;
  return ChainSpace(tokens, experts, top, hidden, inter).bytes;
}

extern "C" int lf_expert_mlp(const lf_expert_mlp_call* a, void* workspace, int64_t workspace_bytes, void* stream) {
  LF_REQUIRE(a != nullptr, "null pointer argument");
  const int64_t need = lf_expert_mlp_workspace_size(a->tokens, a->experts, a->top, a->hidden, a->inter, a->type);
  LF_REQUIRE(need >= 0, "an expert MLP of these sizes has to run as routing, products and sum");
  LF_REQUIRE(workspace != nullptr && workspace_bytes >= need, "workspace of %lld bytes required", static_cast<long long>(need));
  LF_REQUIRE(lf::aligned16(workspace), "the workspace must be 16-byte aligned");
  LF_REQUIRE(a->x && a->logits && a->gate_up && a->down && a->y, "null pointer argument");
  LF_REQUIRE((a->type == LF_EXPERT_BF16) == (a->gate_up_scales == nullptr) && (a->gate_up_scales == nullptr) == (a->down_scales == nullptr),
             "MXFP4 and FP8 weights need scales, bf16 weights have none");
  LF_REQUIRE(lf::aligned16(a->x) && a->x_stride % 8 == 0 && a->x_stride >= a->hidden, "x rows must be 16-byte aligned");
  LF_REQUIRE(lf::aligned16(a->gate_up) && lf::aligned16(a->down), "weights must be 16-byte aligned");
  LF_REQUIRE(reinterpret_cast<uintptr_t>(a->gate_up_scales) % 4 == 0 && reinterpret_cast<uintptr_t>(a->down_scales) % 4 == 0,
             "scales must be 4-byte aligned");
  LF_REQUIRE(a->logits_stride >= a->experts, "the row stride must cover the experts");
  LF_REQUIRE(a->y_stride >= a->hidden && (!a->base || a->base_stride >= a->hidden), "row strides must cover the columns");
  auto s = static_cast<hipStream_t>(stream);
  if (!lf::expert::fused_fits(a->tokens, a->experts, a->top, a->hidden, a->inter, a->type))
    return lf::expert::launch_chain(*a, static_cast<char*>(workspace), s);
  LF_REQUIRE(lf::expert::x_within(*a), "x rows of up to 8 tokens must lie within 2 GiB");
  lf::expert::MlpParams p = lf::expert::params_of(*a);
  p.h = static_cast<uint16_t*>(workspace);
  p.table = reinterpret_cast<int4*>(static_cast<char*>(workspace) + lf::expert::padded16(a->tokens * a->top * a->inter * 4));
  if (const int rc = lf::expert::launch_first(p, a->type, s)) return rc;
  switch (a->type) {
    case LF_EXPERT_BF16: return lf::expert::launch_down<lf::expert::kBf16>(p, s);
    case LF_EXPERT_MXFP4: return lf::expert::launch_down<lf::expert::kMxfp4>(p, s);
    default: return lf::expert::launch_down<lf::expert::kFp8>(p, s);
  }
}
