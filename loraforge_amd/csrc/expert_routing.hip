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
#include <type_traits>

#include "expert_choose.h"
#include "expert_params.h"
#include "../../include/loraforge_amd.h"

namespace lf {
namespace {

constexpr int kSmallThreads = 1024;   // a few tokens, all in one workgroup
constexpr int kChooseThreads = 512;
constexpr int kOrderThreads = 1024;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTop = 64;       // a choice lives in a lane
constexpr int kMaxChunks = 256;   // token chunks counted apart

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

// The choices of token t, as `choose_experts` makes them, stored; returns the lane's.
template <bool kFp32, int kLanes, int kPer>
__device__ __forceinline__ int choose(const RouteParams& p, int t, bool live) {
  float value[kPer];
  load_logits<kLanes>(p.logits, kFp32, p.stride, p.experts, t, live, value);
  const Choice c = choose_experts<kFp32, kLanes>(value, p.top, p.renormalize);
  const int lane = threadIdx.x & (kLanes - 1);
  if (live && lane < p.top) {
    p.weights[int64_t(t) * p.top + lane] = c.weight;
    p.chosen[int64_t(t) * p.top + lane] = c.expert;
  }
  return c.expert;
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
  const void* rows;  // bf16, or fp32
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

// What is read in place of a row that is none.
__device__ const u32x4 kNothing[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};

template <int kVec>
__device__ __forceinline__ void load_row(const uint16_t* src, float (&v)[kVec]) {
  if constexpr (kVec == 8) {
    const u32x4 word = *reinterpret_cast<const u32x4*>(src);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[2 * k] = bf16_lo(word[k]), v[2 * k + 1] = bf16_hi(word[k]);
  } else {
    v[0] = bf16_to_f32(*src);
  }
}
template <int kVec>
__device__ __forceinline__ void load_row(const float* src, float (&v)[kVec]) {
  if constexpr (kVec == 8) {
    const f32x4 a = reinterpret_cast<const f32x4*>(src)[0], b = reinterpret_cast<const f32x4*>(src)[1];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = a[k], v[4 + k] = b[k];
  } else {
    v[0] = *src;
  }
}

// Eight columns per thread (16-byte accesses), or one. Rows are asked for kTogether at a time (one behind the other,
// their latency was most of a few tokens' time): one and two where a token has no more, since each that it lacks costs
// loads and additions all the same (8191 tokens of 4096 columns: one row 21 us, asked for as four 28).
template <class Row, int kVec, int kTogether>
__global__ __launch_bounds__(kCombineThreads) void combine_kernel(CombineParams p) {
  const int64_t chunks = p.n / kVec, total = p.tokens * chunks;
  for (int64_t i = int64_t(blockIdx.x) * kCombineThreads + threadIdx.x; i < total; i += int64_t(gridDim.x) * kCombineThreads) {
    const int64_t t = i / chunks, c = (i - t * chunks) * kVec;
    float sum[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) sum[k] = 0.0f;
    if (p.base) {
      float v[kVec];
      load_row<kVec>(p.base + t * p.base_stride + c, v);
#pragma unroll
      for (int k = 0; k < kVec; ++k) sum[k] += v[k];
    }
    for (int j0 = 0; j0 < p.top; j0 += kTogether) {
      float v[kTogether][kVec], w[kTogether];
      bool in[kTogether];
      int64_t row[kTogether];
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        const int64_t at = t * p.top + min(j0 + i, p.top - 1);
        row[i] = p.positions[at];
        w[i] = p.weights[at];
        in[i] = j0 + i < p.top && row[i] >= 0 && row[i] < p.num_rows;
      }
#pragma unroll
      for (int i = 0; i < kTogether; ++i)
        load_row<kVec>(in[i] ? static_cast<const Row*>(p.rows) + row[i] * p.rows_stride + c : reinterpret_cast<const Row*>(&kNothing), v[i]);
#pragma unroll
      for (int i = 0; i < kTogether; ++i)
#pragma unroll
        for (int k = 0; k < kVec; ++k) sum[k] = in[i] ? fmaf(w[i], v[i][k], sum[k]) : sum[k];
    }
    uint16_t* dst = p.y + t * p.y_stride + c;
    if constexpr (kVec == 8)
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3]),
                                                  pack_bf16x2(sum[4], sum[5]), pack_bf16x2(sum[6], sum[7]));
    else
      *dst = uint16_t(f32_to_bf16(sum[0]));
  }
}

template <class Row>
int launch_combine(const Row* rows, int64_t num_rows, int64_t rows_stride, const int32_t* positions, const float* weights,
                   int64_t tokens, int32_t top, int64_t n, const uint16_t* base, int64_t base_stride, uint16_t* y,
                   int64_t y_stride, hipStream_t s) {
  const bool vec = n % 8 == 0 && rows_stride % 8 == 0 && y_stride % 8 == 0 && aligned16(rows) && aligned16(y) &&
                   (!base || (base_stride % 8 == 0 && aligned16(base)));
  const CombineParams p{rows, rows_stride, num_rows, positions, weights, base, base_stride, y, y_stride, tokens, top, n};
  const int64_t want = (tokens * (vec ? n / 8 : n) + kCombineThreads - 1) / kCombineThreads;
  const dim3 grid(unsigned(want < 65536 ? want : 65536)), threads(kCombineThreads);
  auto run = [&](void (*one)(CombineParams), void (*two)(CombineParams), void (*more)(CombineParams)) {
    hipLaunchKernelGGL(top == 1 ? one : top == 2 ? two : more, grid, threads, 0, s, p);
  };
  if (vec)
    run(combine_kernel<Row, 8, 1>, combine_kernel<Row, 8, 2>, combine_kernel<Row, 8, 4>);
  else
    run(combine_kernel<Row, 1, 1>, combine_kernel<Row, 1, 2>, combine_kernel<Row, 1, 4>);
  LF_HIP(hipGetLastError());
  return kOk;
}

}  // namespace

namespace expert {

int combine_f32(const float* rows, int64_t num_rows, const int32_t* positions, const float* weights, int64_t tokens, int32_t top,
                int64_t n, const uint16_t* base, int64_t base_stride, uint16_t* y, int64_t y_stride, hipStream_t stream) {
  return launch_combine(rows, num_rows, n, positions, weights, tokens, top, n, base, base_stride, y, y_stride, stream);
}

}  // namespace expert
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
  return lf::launch_combine(rows, num_rows, rows_stride, positions, weights, tokens, top, n, base, base_stride, y, y_stride,
                            static_cast<hipStream_t>(stream));
}
