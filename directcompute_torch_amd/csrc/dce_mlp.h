// What the kernels of the gated feed-forward block (dce_mlp.hip, and those on fp16
// parts, dce_mlp_parts.hip) share.
#pragma once
#include "dce_internal.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace dce {

// Workgroup L of a product's n, such that those next to each other run on one XCD, and every XCD
// has its part of each product of a launch (their depths differ).
__device__ __forceinline__ uint32_t xcd_place(uint32_t L, uint32_t n) {
  const uint32_t q = n >> 3, r = n & 7, x = L & 7;
  return x * q + min(x, r) + (L >> 3);
}

// act(g), and its derivative d.
template <MlpAct ACT>
__device__ __forceinline__ float act_grad(float g, float& d) {
  if constexpr (ACT == kGelu) {  // erfc: 1 + erf would cancel for g << 0
    const float p = 0.5f * erfcf(-g * 0.70710678f);
    d = p + g * (0.39894228f * expf(-0.5f * g * g));
    return g * p;
  } else if constexpr (ACT == kRelu) {
    d = g > 0.f ? 1.f : 0.f;
    return g <= 0.f ? 0.f : g;  // NaN stays
  } else {
    float p, q;
    sigmoid_pair(g, p, q);
    d = ACT == kSilu ? p + g * p * q : p * q;
    return ACT == kSilu ? g * p : p;
  }
}
template <MlpAct ACT>
__device__ __forceinline__ float act(float g) {
  float d;
  return act_grad<ACT>(g, d);
}

// f(std::integral_constant<MlpAct, act>)
template <class F>
void by_act(MlpAct act, F&& f) {
  if (act == kSilu) f(std::integral_constant<MlpAct, kSilu>{});
  if (act == kGelu) f(std::integral_constant<MlpAct, kGelu>{});
  if (act == kRelu) f(std::integral_constant<MlpAct, kRelu>{});
  if (act == kSigmoid) f(std::integral_constant<MlpAct, kSigmoid>{});
}

// Sums of `splits` shares of n (4 or more) values, one after the other, in order.
struct MlpSums {
  struct One {
    const float* part;
    float* out;
    uint32_t n, splits, start;
  };
  One s[4];
  uint32_t count, blocks;  // of 256 threads, 4 values each
  void add(const float* part, float* out, uint32_t n, uint32_t splits) {
    s[count++] = {part, out, n, splits, blocks};
    blocks += uint32_t((uint64_t(n) + 1023) / 1024);
  }
};
// Four values, by thread i (of all blocks').
__device__ __forceinline__ f4u mlp_sum_of(const MlpSums& t, uint32_t i, int* which, uint32_t* at) {
  int k = 0;
  while (k + 1 < int(t.count) && t.s[k + 1].start <= i / 256) ++k;
  const MlpSums::One& s = t.s[k];
  const uint64_t first = (uint64_t(i) - s.start * 256ull) * 4;
  *which = first < s.n ? k : -1;
  if (*which < 0) return f4u{0.f, 0.f, 0.f, 0.f};
  // the last quad ends with the matrix; fewer than 4 values there are none
  *at = min(uint32_t(first), s.n - 4);
  f4u v = ldus<false, f4u>(s.part + *at);
#pragma unroll 4
  for (uint32_t j = 1; j < s.splits; ++j) v += ldus<false, f4u>(s.part + size_t(j) * s.n + *at);
  return v;
}

// On fp16 parts, for large calls.
bool mlp_on_parts(const MlpArgs& a, bool backward);
bool mlp_forward_parts(const MlpArgs& a);
bool mlp_backward_parts(const MlpArgs& a, const float* dy, float* dx, float* dwg, float* dwu, float* dwd);

// Their last launch: the splits' sums, and on fp32 what parts do not hold.
struct MlpAgain {
  uint32_t* any;      // of these all are zeros at first; set with any of `rows`, or for all gradients
  uint32_t* rows;     // forward: the results' rows that are wanted
  uint32_t* counts;   // two words: places taken, first products done
  float* ws;          // rows x hidden floats, or mlp_again_floats
};
bool mlp_forward_again(const MlpArgs& a, const MlpAgain& g, const MlpSums& sums);
size_t mlp_again_floats(const MlpArgs& a);
bool mlp_backward_again(const MlpArgs& a, const float* dy, float* dx, float* dwg, float* dwu, float* dwd, const MlpAgain& g, const MlpSums& sums);

}  // namespace dce
