// The k largest of a token's logits and their softmax weights, by the lanes that share
// the token (expert_routing.hip and, for a few tokens, expert_mlp.hip).
#pragma once

#include "common.h"

namespace lf {

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

// A token's choice (-1: none) and its weight (0 beside -1).
struct Choice {
  int expert;
  float weight;
};

// A token's logits (row t of `logits`, rows `stride` apart) in the kLanes lanes that share it: lane l holds
// experts l, l + kLanes, ...; -inf past the last, and everywhere if not `live` (there is a first row all the same:
// addresses are clamped instead of loads skipped, as the compiler waits for a load behind each condition).
template <int kLanes, int kPer>
__device__ __forceinline__ void load_logits(const void* logits, bool fp32, int64_t stride, int experts, int t, bool live, float (&value)[kPer]) {
  const int lane = threadIdx.x & (kLanes - 1);
  const int64_t row = int64_t(live ? t : 0) * stride;
  if (fp32) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) value[i] = static_cast<const float*>(logits)[row + min(lane + i * kLanes, experts - 1)];
  } else {
    uint16_t bits[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) bits[i] = static_cast<const uint16_t*>(logits)[row + min(lane + i * kLanes, experts - 1)];
#pragma unroll
    for (int i = 0; i < kPer; ++i) value[i] = bf16_to_f32(bits[i]);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (!live || lane + i * kLanes >= experts) value[i] = -__builtin_huge_valf();
}

// The choices of the token whose logits these kLanes lanes hold; lane l gets choice l.
// k rounds of a maximum over keys in the order of the logits. The key of a logit that is a bf16 (kFp32 false) leaves
// 16 bits for the expert (lowest first), so one maximum finds both; fp32 takes a second one.
template <bool kFp32, int kLanes, int kPer>
__device__ __forceinline__ Choice choose_experts(const float (&value)[kPer], int top, bool renormalize) {
  const int lane = threadIdx.x & (kLanes - 1);
  uint32_t key[kPer];
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
  for (int j = 0; j < top; ++j) {
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
  if (!renormalize) {
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) total += value[i] > -__builtin_huge_valf() ? expf(value[i] - peak) : 0.0f;
  }
  total = sum_across<kLanes>(total);
  float w = my_expert >= 0 ? share / total : 0.0f;
  if (bad && my_expert >= 0) w = __builtin_nanf("");
  return {my_expert, w};
}

}  // namespace lf
