// Shaped scores of the paged attention (scored_decode.hip, scored_prefill.hip):
// what a query at position p sees, and how its raw products become scores.
//
//   key j is seen where j <= p and (no window or p - j < window), or where
//   j < prefix; keys past the context and in blocks outside the pool never;
//   x = scale * q.k, or with a soft cap c: c * tanh(x / c)
//   score = x - slope_h * |p - j|
//
// Scores are kept in units of log2(e), so that weights are exp2. The cap costs
// two transcendental operations: c * tanh(x / c) = c - 2 c / (1 + e^(2 x / c)),
// whose error for small x is that of the subtraction from c, 2^-24 c absolute,
// which moves a weight by under 10^-5 of itself for a cap of 50. A cap past
// kMostCap is refused: its error would pass the output's rounding (10^-4 there).
#pragma once

#include <cmath>
#include <type_traits>

#include "half_types.hpp"

namespace swiftllm {
namespace scored {

constexpr float kLog2e = 1.4426950408889634f;

constexpr float kMostCap = 1024.0f;

// Weights are 2^weight_exp * exp2(score - m): m may lag the maximum by kLag
// (log2 units) before the sums are rescaled. In fp16 they stay below 2^15, so
// that small ones are as far from its subnormals as can be; bfloat16 reaches as
// far down as 32 bits do, and there they stay at 1 and below: a weight times the
// type's largest value is still a number.
constexpr float kLag = 8.0f;
template <typename T>
constexpr float weight_exp = std::is_same<T, F16>::value ? 7.0f : -kLag;

struct Shape {
    float scale;         // no cap: scale * log2(e); cap: 2 log2(e) scale / cap
    float cap;           // cap * log2(e); 0: none
    int window;          // 0: none
    const int* prefix;   // [S] or null
    const float* slopes; // [H] or null
};

// The scaled and capped score, times log2(e), of a raw product.
__device__ __forceinline__ float capped_score(float raw, float scale, float cap) {
    const float e = __builtin_amdgcn_exp2f(raw * scale);
    return __builtin_fmaf(__builtin_amdgcn_rcpf(e + 1.0f), -2.0f * cap, cap);
}

inline bool make_shape(Shape& s, float scale, float softcap, int window, const int* prefix, const float* slopes) {
    const double log2e = 1.4426950408889634;
    s.cap = static_cast<float>(softcap * log2e);
    s.scale = softcap > 0.0f ? static_cast<float>(2.0 * log2e * scale / softcap) : static_cast<float>(scale * log2e);
    s.window = window;
    s.prefix = prefix;
    s.slopes = slopes;
    return std::isfinite(s.scale) && std::isfinite(s.cap) && std::isfinite(softcap) && softcap >= 0.0f && window >= 0;
}

// Bits 0 .. n - 1 of 16.
__device__ __forceinline__ unsigned low_bits(int n) { return (1u << min(max(n, 0), 16)) - 1u; }

__device__ __forceinline__ bool block_known(int b, int num_blocks) {
    return b >= 0 && (num_blocks <= 0 || b < num_blocks);
}

}  // namespace scored
}  // namespace swiftllm
