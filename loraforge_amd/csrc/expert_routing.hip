// Mixture-of-experts routing (top-k of a softmax, stable order by expert) and
// the weighted sum of the experts' rows.
//
// Choice: p = softmax(logits) over the experts of a token; the k largest
// logits, of equal ones the lowest expert first; weight p_e, or p_e over the
// sum of the chosen p. -inf: not allowed (fewer than k allowed experts leave
// choices of expert -1 and weight 0). A token whose logits hold NaN or +inf has
// NaN weights (NaN ranks below every number), as the formula gives.
//
// Order: choices sorted by expert, then by token and choice. Integer counts
// only, each place computed from counts of what precedes it, so no result
// depends on the order in which workgroups run.
#include "common.h"
#include "../../include/loraforge_amd.h"

namespace lf {
namespace {

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

template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), kCtrl, kRows, 0xf, false)));
}
// Largest value over the wave, uniform.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = dpp_max<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8: lane 15 of each row holds its maximum
  v = dpp_max<0x112, 0xf>(v);
  v = dpp_max<0x114, 0xf>(v);
  v = dpp_max<0x118, 0xf>(v);
  v = dpp_max<0x142, 0xa>(v);  // row_bcast 15 into rows 1 and 3
  v = dpp_max<0x143, 0xc>(v);  // row_bcast 31 into rows 2 and 3
  return uint32_t(__builtin_amdgcn_readlane(int(v), 63));
}

struct RouteParams {
  const void* logits;
  int64_t stride;
  int32_t fp32, tokens, experts, top, renormalize;
  int32_t chunk;   // tokens per chunk
  int32_t chunks;
  float* weights;    // [tokens, top]
  int32_t* chosen;   // [tokens, top]
  int32_t* offsets;  // [experts + 1]
  int32_t* token_of; // [tokens * top]
  int32_t* positions;// [tokens, top]
  int32_t* counts;   // [chunks, experts]
};

// The choices of one token, by one wave: lane l holds experts [l kPer, (l + 1) kPer).
template <int kPer>
__device__ __forceinline__ void choose_token(const RouteParams& p, int t, int* hist) {
  const int lane = threadIdx.x & 63;
  uint32_t key[kPer];
  float value[kPer];
  bool odd = false;  // NaN or +inf
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = lane * kPer + i;
    float v = -__builtin_huge_valf();
    if (e < p.experts)
      v = p.fp32 ? static_cast<const float*>(p.logits)[int64_t(t) * p.stride + e]
                 : bf16_to_f32(static_cast<const uint16_t*>(p.logits)[int64_t(t) * p.stride + e]);
    value[i] = v;
    key[i] = order_key(v);
    odd |= !(v < __builtin_huge_valf());
  }
  const bool bad = __ballot(odd) != 0;
  uint32_t best = 0;
  int at = 0;
  int my_expert = -1;
  uint32_t my_key = 0;
  uint32_t top_key = 0;
  for (int j = 0; j < p.top; ++j) {
    best = key[0];
    at = 0;
#pragma unroll
    for (int i = 1; i < kPer; ++i)
      if (key[i] > best) best = key[i], at = i;
    const uint32_t m = wave_max(best);
    if (m == 0) break;  // nothing allowed is left
    if (j == 0) top_key = m;
    const int owner = __builtin_ctzll(__ballot(best == m));
    const int e = owner * kPer + __builtin_amdgcn_readlane(at, owner);
    if (lane == j) my_expert = e, my_key = m;
    if (lane == owner) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i == at) key[i] = 0;
    }
  }
  const float peak = key_value(top_key);
  float share = my_expert >= 0 ? expf(key_value(my_key) - peak) : 0.0f;
  float total = 0.0f;
  if (p.renormalize) {
    total = wave_sum(share);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) total += value[i] > -__builtin_huge_valf() ? expf(value[i] - peak) : 0.0f;
    total = wave_sum(total);
  }
  if (lane < p.top) {
    float w = my_expert >= 0 ? share / total : 0.0f;
    if (bad && my_expert >= 0) w = __builtin_nanf("");
    p.weights[int64_t(t) * p.top + lane] = w;
    p.chosen[int64_t(t) * p.top + lane] = my_expert;
    if (my_expert >= 0) atomicAdd(&hist[my_expert], 1);
  }
}

__device__ __forceinline__ void choose_chunk(const RouteParams& p, int first, int last, int* hist) {
  const int waves = blockDim.x >> 6;
  for (int t = first + int(threadIdx.x >> 6); t < last; t += waves) {
    if (p.experts <= 64) choose_token<1>(p, t, hist);
    else if (p.experts <= 128) choose_token<2>(p, t, hist);
    else if (p.experts <= 256) choose_token<4>(p, t, hist);
    else choose_token<16>(p, t, hist);
  }
}

// Places of a chunk's choices: base[e] is the place of the chunk's first choice of
// expert e. 1024 choices a pass, in order: a wave finds the earlier choices of the
// same expert among its 64 by comparing the experts' bits, and adds the counts of
// the waves before it.
__device__ __forceinline__ void place_chunk(const RouteParams& p, int first, int last, int* base, int* wave_counts) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int begin = first * p.top, end = last * p.top;
  for (int at = begin; at < end; at += blockDim.x) {
    for (int i = threadIdx.x; i < waves * p.experts; i += blockDim.x) wave_counts[i] = 0;
    __syncthreads();
    const int i = at + int(threadIdx.x);
    const int e = i < end ? p.chosen[i] : -1;
    uint64_t same = __ballot(e >= 0);
    for (int bit = 1; bit < p.experts; bit <<= 1) {
      const uint64_t has = __ballot((e & bit) != 0);
      same &= (e & bit) ? has : ~has;
    }
    const int before = __popcll(same & ((uint64_t(1) << lane) - 1));
    if (e >= 0 && before == 0) wave_counts[wave * p.experts + e] = __popcll(same);
    __syncthreads();
    if (i < end) {
      int place = -1;
      if (e >= 0) {
        place = base[e] + before;
        for (int w = 0; w < wave; ++w) place += wave_counts[w * p.experts + e];
        p.token_of[place] = i / p.top;
      }
      p.positions[i] = place;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < p.experts; x += blockDim.x) {
      int sum = 0;
      for (int w = 0; w < waves; ++w) sum += wave_counts[w * p.experts + x];
      base[x] += sum;
    }
    __syncthreads();
  }
}

// Exclusive sums of count[0 .. n) in LDS, in place; returns the total.
__device__ int scan_counts(int* count, int n) {
  __shared__ int wave_total[kOrderThreads / 64];
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
  for (int w = 0; w < int(blockDim.x >> 6); ++w) {
    if (w < wave) before += wave_total[w];
    total += wave_total[w];
  }
  if (i < n) count[i] = before + sum - mine;
  __syncthreads();
  return total;
}

__device__ __forceinline__ void fill_rest(const RouteParams& p, int total, int part, int parts) {
  const int64_t end = int64_t(p.tokens) * p.top;
  for (int64_t i = total + int64_t(part) * blockDim.x + threadIdx.x; i < end; i += int64_t(parts) * blockDim.x) p.token_of[i] = -1;
}

// A few tokens: the whole routing in one workgroup.
__global__ __launch_bounds__(kOrderThreads) void route_small_kernel(RouteParams p) {
  extern __shared__ int lds[];
  int* base = lds;                        // [experts]
  int* wave_counts = lds + p.experts;     // [16, experts]
  for (int e = threadIdx.x; e < p.experts; e += kOrderThreads) base[e] = 0;
  __syncthreads();
  choose_chunk(p, 0, p.tokens, base);
  __syncthreads();
  const int total = scan_counts(base, p.experts);
  for (int e = threadIdx.x; e < p.experts; e += kOrderThreads) p.offsets[e] = base[e];
  if (threadIdx.x == 0) p.offsets[p.experts] = total;
  fill_rest(p, total, 0, 1);
  __syncthreads();  // (place_chunk reads choices that other waves of this workgroup stored)
  place_chunk(p, 0, p.tokens, base, wave_counts);
}

__global__ __launch_bounds__(kChooseThreads) void route_choose_kernel(RouteParams p) {
  extern __shared__ int lds[];
  for (int e = threadIdx.x; e < p.experts; e += kChooseThreads) lds[e] = 0;
  __syncthreads();
  const int first = blockIdx.x * p.chunk;
  choose_chunk(p, first, min(first + p.chunk, p.tokens), lds);
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += kChooseThreads) p.counts[int64_t(blockIdx.x) * p.experts + e] = lds[e];
}

__global__ __launch_bounds__(kOrderThreads) void route_order_kernel(RouteParams p) {
  extern __shared__ int lds[];
  int* base = lds;                      // [experts]: all choices of an expert, then its first place
  int* mine = lds + p.experts;          // [experts]: those of the chunks before this one
  int* wave_counts = lds + 2 * p.experts;
  for (int e = threadIdx.x; e < 2 * p.experts; e += kOrderThreads) lds[e] = 0;
  __syncthreads();
  // A thread sums some chunks of one expert.
  const int parts = max(1, kOrderThreads / p.experts);
  for (int i = threadIdx.x; i < p.experts * parts; i += kOrderThreads) {
    const int e = i % p.experts, part = i / p.experts;
    int all = 0, before = 0;
    for (int c = part; c < p.chunks; c += parts) {
      const int v = p.counts[int64_t(c) * p.experts + e];
      all += v;
      before += c < int(blockIdx.x) ? v : 0;
    }
    atomicAdd(&base[e], all);
    atomicAdd(&mine[e], before);
  }
  __syncthreads();
  const int total = scan_counts(base, p.experts);
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e < p.experts; e += kOrderThreads) p.offsets[e] = base[e];
    if (threadIdx.x == 0) p.offsets[p.experts] = total;
  }
  fill_rest(p, total, blockIdx.x, gridDim.x);
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += kOrderThreads) base[e] += mine[e];
  __syncthreads();
  const int first = blockIdx.x * p.chunk;
  place_chunk(p, first, min(first + p.chunk, p.tokens), base, wave_counts);
}

// Tokens that one workgroup routes by itself.
constexpr int kSmallTokens = 64;

int chunk_tokens(int64_t tokens) {
  const int64_t c = (tokens + kMaxChunks - 1) / kMaxChunks;
  return int(c < 16 ? 16 : c);
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
  return (tokens + chunk - 1) / chunk * experts * int64_t(sizeof(int32_t));
}

extern "C" int lf_route_experts(const void* logits, int32_t fp32, int64_t tokens, int32_t experts, int64_t stride,
                                int32_t top, int32_t renormalize, float* weights, int32_t* chosen, int32_t* offsets,
                                int32_t* token_of, int32_t* positions, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  LF_REQUIRE(tokens >= 0 && experts >= 1 && experts <= lf::kMaxExperts, "experts must be in 1..%d", lf::kMaxExperts);
  LF_REQUIRE(top >= 1 && top <= lf::kMaxTop && top <= experts, "top_k must be in 1..min(experts, %d)", lf::kMaxTop);
  LF_REQUIRE(stride >= experts, "the row stride must cover the experts");
  LF_REQUIRE(tokens * top < (int64_t(1) << 31) - (int64_t(1) << 16), "tokens * top_k must fit signed int32 indexing");
  LF_REQUIRE(offsets != nullptr, "null pointer argument");
  LF_REQUIRE(tokens == 0 || (logits && weights && chosen && token_of && positions), "null pointer argument");
  const int64_t need = lf_route_experts_workspace_size(tokens, experts);
  LF_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), "workspace of %lld bytes required",
             static_cast<long long>(need));
  lf::RouteParams p{logits, stride, fp32, int32_t(tokens), experts, top, renormalize, 0, 0, weights, chosen, offsets,
                    token_of, positions, static_cast<int32_t*>(workspace)};
  auto s = static_cast<hipStream_t>(stream);
  const unsigned place_lds = unsigned(1 + lf::kOrderThreads / 64) * experts * sizeof(int);
  if (tokens <= lf::kSmallTokens) {
    hipLaunchKernelGGL(lf::route_small_kernel, dim3(1), dim3(lf::kOrderThreads), place_lds, s, p);
  } else {
    p.chunk = lf::chunk_tokens(tokens);
    p.chunks = int32_t((tokens + p.chunk - 1) / p.chunk);
    hipLaunchKernelGGL(lf::route_choose_kernel, dim3(p.chunks), dim3(lf::kChooseThreads), experts * sizeof(int), s, p);
    hipLaunchKernelGGL(lf::route_order_kernel, dim3(p.chunks), dim3(lf::kOrderThreads),
                       place_lds + experts * sizeof(int), s, p);
  }
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
