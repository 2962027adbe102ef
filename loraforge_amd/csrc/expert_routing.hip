// Mixture-of-experts routing (top-k of a softmax, stable order by expert) and
// the weighted sum of the experts' rows.
//
// Choice: p = softmax(logits) over the experts of a token; the k largest
// logits, of equal ones the lowest expert first; weight p_e, or p_e over the
// sum of the chosen p. -inf: not allowed (fewer than k allowed experts leave
// choices of expert -1 and weight 0). A token whose logits hold NaN or +inf has NaN
// weights for its choices, as the formula gives (NaN ranks with -inf: it is not chosen).
//
// Order: choices sorted by expert, then by token and choice. Integer counts
// only, each place computed from counts of what precedes it, so no result
// depends on the order in which workgroups run.
//
// Bound by latency: loads, k dependent maxima, barriers, and for more than 64 tokens a
// second launch, which needs all counts. 128 experts, top 8: 16 tokens 4.8 us in one
// workgroup; 8191 tokens 5.5 us to choose and 5.8 to order (with a wave for each token
// in turn, and places by counting choices wave by wave, 11.2 and 13.0). The sum is
// HBM-bound: 8191 tokens of 8 rows of 4096 take 119 us (5.1 TB/s, a copy's rate).
#include "common.h"
#include "../../include/loraforge_amd.h"

namespace lf {
namespace {

constexpr int kSmallThreads = 1024;   // a few tokens, all in one workgroup
constexpr int kChooseThreads = 512;
constexpr int kOrderThreads = 1024;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTop = 64;       // a choice lives in a lane
constexpr int kMaxChunks = 256;   // token chunks counted apart

// fp32 -> integer of the same order, NaN and -inf lowest (0), -0 as +0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -__builtin_huge_valf())) return 0u;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k); }

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), kCtrl, 0xf, 0xf, false));
}
// `op` over the kLanes lanes that share a token (16 or 64), the result in each of
// them: rotations within a row of 16 lanes, then the four rows, in a fixed order.
template <int kLanes, class Op>
__device__ __forceinline__ uint32_t across(uint32_t v, Op op) {
  v = op(v, dpp<0x128>(v));
  v = op(v, dpp<0x124>(v));
  v = op(v, dpp<0x122>(v));
  v = op(v, dpp<0x121>(v));
  if constexpr (kLanes == 64) {
    auto row = [&](int lane) { return uint32_t(__builtin_amdgcn_readlane(int(v), lane)); };
    v = op(op(row(0), row(16)), op(row(32), row(48)));
  }
  return v;
}
template <int kLanes>
__device__ __forceinline__ uint32_t max_across(uint32_t v) {
  return across<kLanes>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int kLanes>
__device__ __forceinline__ float sum_across(float v) {
  return __uint_as_float(across<kLanes>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

struct RouteParams {
  const void* logits;
  int64_t stride;
  int32_t fp32, tokens, experts, top, renormalize;
  int32_t chunk;     // tokens per chunk
  int32_t chunks;
  int32_t row;       // counts of a chunk, a multiple of four
  float* weights;    // [tokens, top]
  int32_t* chosen;   // [tokens, top]
  int32_t* offsets;  // [experts + 1]
  int32_t* token_of; // [tokens * top]
  int32_t* positions;// [tokens, top]
  int32_t* counts;   // [chunks, row]
};

// The choices of the token of these kLanes lanes; lane l of them holds experts l,
// l + kLanes, ... and at the end choice l (-1: none), whose weight it stores.
// k rounds of a maximum over keys in the order of the logits. A bf16 key leaves 16 bits
// for the expert (lowest first), so one maximum finds both; fp32 takes a second one.
template <bool kFp32, int kLanes, int kPer>
__device__ __forceinline__ int choose(const RouteParams& p, int t, bool live) {
  const int lane = threadIdx.x & (kLanes - 1);
  uint32_t key[kPer];
  float value[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = lane + i * kLanes;
    const int64_t at = int64_t(t) * p.stride + e;
    value[i] = -__builtin_huge_valf();
    if (live && e < p.experts)
      value[i] = kFp32 ? static_cast<const float*>(p.logits)[at] : bf16_to_f32(static_cast<const uint16_t*>(p.logits)[at]);
  }
  bool odd = false;  // NaN or +inf
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    key[i] = order_key(value[i]);
    if (!kFp32 && key[i]) key[i] = (key[i] & 0xffff0000u) | uint32_t(0xffff - (lane + i * kLanes));
    odd |= !(value[i] < __builtin_huge_valf());
  }
  const uint64_t odd_lanes = __ballot(odd);
  const bool bad = (kLanes == 64 ? odd_lanes : (odd_lanes >> (threadIdx.x & 48)) & 0xffff) != 0;
  uint32_t my_key = 0, top_key = 0;
  int my_expert = -1;
  for (int j = 0; j < p.top; ++j) {
    uint32_t best = key[0];
#pragma unroll
    for (int i = 1; i < kPer; ++i) best = max(best, key[i]);
    best = max_across<kLanes>(best);
    int e = 0xffff - int(best & 0xffff);
    if constexpr (kFp32) {
      uint32_t last = 0;  // of the experts that have it, the lowest: ~e largest
#pragma unroll
      for (int i = 0; i < kPer; ++i) last = max(last, key[i] == best ? ~uint32_t(lane + i * kLanes) : 0u);
      e = int(~max_across<kLanes>(last));
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (kFp32 ? e - lane == i * kLanes : key[i] == best) key[i] = 0;
    if (!kFp32) best = best >> 31 ? best & 0xffff0000u : best | (best ? 0xffffu : 0u);
    if (j == 0) top_key = best;
    if (lane == j && best) my_expert = e, my_key = best;
  }
  const float peak = key_value(top_key);
  float share = my_expert >= 0 ? expf(key_value(my_key) - peak) : 0.0f;
  float total = share;
  if (!p.renormalize) {
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) total += value[i] > -__builtin_huge_valf() ? expf(value[i] - peak) : 0.0f;
  }
  total = sum_across<kLanes>(total);
  if (live && lane < p.top) {
    float w = my_expert >= 0 ? share / total : 0.0f;
    if (bad && my_expert >= 0) w = __builtin_nanf("");
    p.weights[int64_t(t) * p.top + lane] = w;
    p.chosen[int64_t(t) * p.top + lane] = my_expert;
  }
  return my_expert;
}

// Chooses for tokens [first, last), as many at once as the workgroup has lanes for (64 at most),
// and hands place(token, choice, expert, earlier) each choice with the count of earlier
// tokens of [first, last) that have the same expert (-1, 0: none). A token chooses an expert
// once, so a pass' choices of an expert are a mask of its tokens: no order of atomics shows.
// run[e] counts an expert's choices so far.
template <bool kFp32, int kLanes, int kPer, class Place>
__device__ __forceinline__ void choose_range(const RouteParams& p, int first, int last, unsigned long long* mask, int* run, Place place) {
  constexpr int kMost = 64;  // tokens of a mask
  const int slot = threadIdx.x / kLanes, slots = min(kMost, int(blockDim.x) / kLanes);
  const int lane = threadIdx.x & (kLanes - 1);
  for (int at = first; at < last; at += slots) {
    for (int e = threadIdx.x; e < p.experts; e += blockDim.x) mask[e] = 0;
    __syncthreads();
    const int t = at + slot;
    const bool live = slot < slots && t < last;
    int e = -1;
    if (at + int(threadIdx.x & ~63u) / kLanes < last) e = choose<kFp32, kLanes, kPer>(p, t, live);  // (a wave as a whole)
    if (live && e >= 0) atomicOr(&mask[e], 1ull << slot);
    __syncthreads();
    if (live && lane < p.top) place(t, lane, e, e >= 0 ? run[e] + __popcll(mask[e] & ((1ull << slot) - 1)) : 0);
    __syncthreads();
    for (int x = threadIdx.x; x < p.experts; x += blockDim.x) run[x] += __popcll(mask[x]);
    __syncthreads();
  }
}

// Exclusive sums of count[0 .. n), n <= the threads, in place; returns the total.
__device__ int scan_counts(int* count, int n, int* wave_total) {
  const int i = threadIdx.x, lane = i & 63, wave = i >> 6;
  const int mine = i < n ? count[i] : 0;
  int sum = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(sum, d, 64);
    if (lane >= d) sum += up;
  }
  if (lane == 63) wave_total[wave] = sum;
  __syncthreads();
  int before = 0, total = 0;
  for (int w = 0; w < (n + 63) >> 6; ++w) {
    if (w < wave) before += wave_total[w];
    total += wave_total[w];
  }
  if (i < n) count[i] = before + sum - mine;
  __syncthreads();
  return total;
}

// Tokens that one workgroup routes by itself.
constexpr int kSmallTokens = 64;

// A few tokens: the whole routing in one workgroup, in one pass where 16 lanes hold a token's experts.
template <bool kFp32, int kLanes, int kPer>
__global__ __launch_bounds__(kSmallThreads) void route_small_kernel(RouteParams p) {
  __shared__ unsigned long long mask[kMaxExperts];
  __shared__ int run[kMaxExperts], wave_total[kSmallThreads / 64];
  __shared__ int choice[kSmallTokens * kMaxTop];  // expert, and above 16 bits the earlier choices of it; or -1
  for (int e = threadIdx.x; e < p.experts; e += kSmallThreads) run[e] = 0;
  choose_range<kFp32, kLanes, kPer>(p, 0, p.tokens, mask, run, [&](int t, int j, int e, int earlier) {
    choice[t * p.top + j] = e >= 0 ? e | earlier << 16 : -1;
  });
  const int total = scan_counts(run, p.experts, wave_total);
  for (int e = threadIdx.x; e < p.experts; e += kSmallThreads) p.offsets[e] = run[e];
  if (threadIdx.x == 0) p.offsets[p.experts] = total;
  for (int i = threadIdx.x; i < p.tokens * p.top; i += kSmallThreads) {
    const int c = choice[i];
    const int place = c >= 0 ? run[c & 0xffff] + (c >> 16) : -1;
    p.positions[i] = place;
    if (c >= 0) p.token_of[place] = i / p.top;
    if (i >= total) p.token_of[i] = -1;
  }
}

// Choices of a chunk, their places among the chunk's choices of the same expert, and the chunk's counts.
template <bool kFp32, int kLanes, int kPer>
__global__ __launch_bounds__(kChooseThreads) void route_choose_kernel(RouteParams p) {
  __shared__ unsigned long long mask[kMaxExperts];
  __shared__ int run[kMaxExperts];
  for (int e = threadIdx.x; e < p.row; e += kChooseThreads) run[e] = 0;
  const int first = blockIdx.x * p.chunk;
  choose_range<kFp32, kLanes, kPer>(p, first, min(first + p.chunk, p.tokens), mask, run, [&](int t, int j, int e, int earlier) {
    p.positions[int64_t(t) * p.top + j] = e >= 0 ? earlier : -1;
  });
  for (int e = threadIdx.x; e < p.row; e += kChooseThreads) p.counts[int64_t(blockIdx.x) * p.row + e] = run[e];
}

// Places of a chunk's choices: those of smaller experts, of the same expert in earlier chunks, and before it in its own.
__global__ __launch_bounds__(kOrderThreads) void route_order_kernel(RouteParams p) {
  __shared__ int base[kMaxExperts];  // all choices of an expert, then its first place
  __shared__ int mine[kMaxExperts];  // those of the chunks before this one
  __shared__ int wave_total[kOrderThreads / 64];
  for (int e = threadIdx.x; e < p.experts; e += kOrderThreads) base[e] = mine[e] = 0;
  const int first = int(blockIdx.x) * p.chunk * p.top;
  const int last = min(int(blockIdx.x) * p.chunk + p.chunk, p.tokens) * p.top;
  int at = first + int(threadIdx.x);
  int e = -1, place = 0;
  if (at < last) e = p.chosen[at], place = p.positions[at];
  __syncthreads();
  // A thread sums some chunks of four experts.
  const int quads = p.row / 4, parts = kOrderThreads / quads;
  const int quad = int(threadIdx.x) % quads, part = int(threadIdx.x) / quads;
  if (part < parts) {
    int4 all = make_int4(0, 0, 0, 0), before = make_int4(0, 0, 0, 0);
    const int4* counts = reinterpret_cast<const int4*>(p.counts) + quad;
#pragma unroll 8
    for (int c = part; c < p.chunks; c += parts) {
      const int4 v = counts[int64_t(c) * quads];
      all.x += v.x, all.y += v.y, all.z += v.z, all.w += v.w;
      if (c < int(blockIdx.x)) before.x += v.x, before.y += v.y, before.z += v.z, before.w += v.w;
    }
    auto add = [&](int x, int a, int b) {
      if (x < p.experts) atomicAdd(&base[x], a), atomicAdd(&mine[x], b);
    };
    add(quad * 4, all.x, before.x), add(quad * 4 + 1, all.y, before.y);
    add(quad * 4 + 2, all.z, before.z), add(quad * 4 + 3, all.w, before.w);
  }
  __syncthreads();
  const int total = scan_counts(base, p.experts, wave_total);
  if (blockIdx.x == 0) {
    for (int x = threadIdx.x; x < p.experts; x += kOrderThreads) p.offsets[x] = base[x];
    if (threadIdx.x == 0) p.offsets[p.experts] = total;
  }
  for (int64_t i = total + int64_t(blockIdx.x) * kOrderThreads + threadIdx.x; i < int64_t(p.tokens) * p.top;
       i += int64_t(gridDim.x) * kOrderThreads)
    p.token_of[i] = -1;  // (choices that fell away)
  while (at < last) {
    if (e >= 0) {
      place += base[e] + mine[e];
      p.positions[at] = place;
      p.token_of[place] = at / p.top;
    }
    at += kOrderThreads;
    if (at < last) e = p.chosen[at], place = p.positions[at];
  }
}

int chunk_tokens(int64_t tokens) {
  const int64_t c = (tokens + kMaxChunks - 1) / kMaxChunks;
  return int(c < 32 ? 32 : c);
}
int count_row(int32_t experts) { return (experts + 3) / 4 * 4; }

template <bool kFp32, int kLanes, int kPer>
void launch_route(const RouteParams& p, hipStream_t s) {
  if (p.chunks == 0) {
    hipLaunchKernelGGL((route_small_kernel<kFp32, kLanes, kPer>), dim3(1), dim3(kSmallThreads), 0, s, p);
  } else {
    hipLaunchKernelGGL((route_choose_kernel<kFp32, kLanes, kPer>), dim3(p.chunks), dim3(kChooseThreads), 0, s, p);
    hipLaunchKernelGGL(route_order_kernel, dim3(p.chunks), dim3(kOrderThreads), 0, s, p);
  }
}

// A token takes 16 lanes where its choices and at most 16 experts a lane fit.
template <bool kFp32>
void launch_route(const RouteParams& p, hipStream_t s) {
  if (p.top > 16 || p.experts > 256) launch_route<kFp32, 64, 16>(p, s);
  else if (p.experts > 128) launch_route<kFp32, 16, 16>(p, s);
  else if (p.experts > 64) launch_route<kFp32, 16, 8>(p, s);
  else launch_route<kFp32, 16, 4>(p, s);
}

// ---------------------------------------------------------------------------
// y[t] = base[t] + sum_j weights[t, j] rows[positions[t, j]], j in order, in fp32,
// rounded once. HBM-bound: every row read once.
// ---------------------------------------------------------------------------
constexpr int kCombineThreads = 256;

struct CombineParams {
  const uint16_t* rows;
  int64_t rows_stride, num_rows;
  const int32_t* positions;
  const float* weights;
  const uint16_t* base;
  int64_t base_stride;
  uint16_t* y;
  int64_t y_stride;
  int64_t tokens;
  int32_t top;
  int64_t n;
};

// Eight columns per thread (16-byte accesses), or one.
template <int kVec>
__global__ __launch_bounds__(kCombineThreads) void combine_kernel(CombineParams p) {
  const int64_t chunks = p.n / kVec, total = p.tokens * chunks;
  for (int64_t i = int64_t(blockIdx.x) * kCombineThreads + threadIdx.x; i < total; i += int64_t(gridDim.x) * kCombineThreads) {
    const int64_t t = i / chunks, c = (i - t * chunks) * kVec;
    float sum[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) sum[k] = 0.0f;
    auto add = [&](const uint16_t* src, float w) {
      if constexpr (kVec == 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(src);
        const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          sum[2 * k] = fmaf(w, bf16_lo(word[k]), sum[2 * k]);
          sum[2 * k + 1] = fmaf(w, bf16_hi(word[k]), sum[2 * k + 1]);
        }
      } else {
        sum[0] = fmaf(w, bf16_to_f32(*src), sum[0]);
      }
    };
    if (p.base) add(p.base + t * p.base_stride + c, 1.0f);
    for (int j = 0; j < p.top; ++j) {
      const int64_t row = p.positions[t * p.top + j];
      if (row >= 0 && row < p.num_rows) add(p.rows + row * p.rows_stride + c, p.weights[t * p.top + j]);
    }
    uint16_t* dst = p.y + t * p.y_stride + c;
    if constexpr (kVec == 8)
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3]),
                                                  pack_bf16x2(sum[4], sum[5]), pack_bf16x2(sum[6], sum[7]));
    else
      *dst = uint16_t(f32_to_bf16(sum[0]));
  }
}

}  // namespace
}  // namespace lf

extern "C" int64_t lf_route_experts_workspace_size(int64_t tokens, int32_t experts) {
  if (tokens < 0 || tokens >= (int64_t(1) << 31) || experts < 1 || experts > lf::kMaxExperts) return -1;
  if (tokens <= lf::kSmallTokens) return 0;
  const int chunk = lf::chunk_tokens(tokens);
  return (tokens + chunk - 1) / chunk * lf::count_row(experts) * int64_t(sizeof(int32_t));
}

extern "C" int lf_route_experts(const void* logits, int32_t fp32, int64_t tokens, int32_t experts, int64_t stride,
                                int32_t top, int32_t renormalize, float* weights, int32_t* chosen, int32_t* offsets,
                                int32_t* token_of, int32_t* positions, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  LF_REQUIRE(tokens >= 0 && experts >= 1 && experts <= lf::kMaxExperts, "experts must be in 1..%d", lf::kMaxExperts);
  LF_REQUIRE(top >= 1 && top <= lf::kMaxTop && top <= experts, "top_k must be in 1..min(experts, %d)", lf::kMaxTop);
  LF_REQUIRE(stride >= experts, "the row stride must cover the experts");
  // (The count itself first: its product with top wraps round in 64 bits from 2^57 on.)
  LF_REQUIRE(tokens < (int64_t(1) << 31) && tokens * top < (int64_t(1) << 31) - (int64_t(1) << 16),
             "tokens * top_k must fit signed int32 indexing");
  LF_REQUIRE(offsets != nullptr, "null pointer argument");
  LF_REQUIRE(tokens == 0 || (logits && weights && chosen && token_of && positions), "null pointer argument");
  const int64_t need = lf_route_experts_workspace_size(tokens, experts);
  LF_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), "workspace of %lld bytes required",
             static_cast<long long>(need));
  LF_REQUIRE(need == 0 || lf::aligned16(workspace), "the workspace must be 16-byte aligned");
  lf::RouteParams p{logits, stride, fp32, int32_t(tokens), experts, top, renormalize, 0, 0, lf::count_row(experts), weights,
                    chosen, offsets, token_of, positions, static_cast<int32_t*>(workspace)};
  if (tokens > lf::kSmallTokens) {
    p.chunk = lf::chunk_tokens(tokens);
    p.chunks = int32_t((tokens + p.chunk - 1) / p.chunk);
  }
  auto s = static_cast<hipStream_t>(stream);
  if (fp32) lf::launch_route<true>(p, s);
  else lf::launch_route<false>(p, s);
  LF_HIP(hipGetLastError());
  return lf::kOk;
}

extern "C" int lf_combine_experts(const uint16_t* rows, int64_t num_rows, int64_t rows_stride, const int32_t* positions,
                                  const float* weights, int64_t tokens, int32_t top, int64_t n, const uint16_t* base,
                                  int64_t base_stride, uint16_t* y, int64_t y_stride, void* stream) {
  LF_REQUIRE(tokens >= 0 && top >= 1 && n >= 1 && num_rows >= 0, "sizes must be positive");
  if (tokens == 0) return lf::kOk;
  LF_REQUIRE(positions && weights && y && (rows || num_rows == 0), "null pointer argument");
  LF_REQUIRE(rows_stride >= n && y_stride >= n && (!base || base_stride >= n), "row strides must cover n columns");
  const bool vec = n % 8 == 0 && rows_stride % 8 == 0 && y_stride % 8 == 0 && lf::aligned16(rows) && lf::aligned16(y) &&
                   (!base || (base_stride % 8 == 0 && lf::aligned16(base)));
  lf::CombineParams p{rows, rows_stride, num_rows, positions, weights, base, base_stride, y, y_stride, tokens, top, n};
  const int64_t want = (tokens * (vec ? n / 8 : n) + lf::kCombineThreads - 1) / lf::kCombineThreads;
  const dim3 grid(unsigned(want < 65536 ? want : 65536)), threads(lf::kCombineThreads);
  auto s = static_cast<hipStream_t>(stream);
  if (vec)
    hipLaunchKernelGGL(lf::combine_kernel<8>, grid, threads, 0, s, p);
  else
    hipLaunchKernelGGL(lf::combine_kernel<1>, grid, threads, 0, s, p);
  LF_HIP(hipGetLastError());
  return lf::kOk;
}
