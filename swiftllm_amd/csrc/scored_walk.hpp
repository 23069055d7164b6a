// One wave's walk over blocks of 16 keys for 16 query rows (scored_decode.hip,
// shared_decode.hip), on 16x16x16 products: K comes tokens-contiguous and is turned
// by a product with the identity (exact), S^T = K Q^T and O^T = V P^T, P in two
// 16-bit parts.
#pragma once

#include "scored_core.hpp"

namespace swiftllm {
namespace scored {

template <int D>
struct State {
    float m, l;
    f4 acc[D / 16];
};

__device__ __forceinline__ s4 load4(const uint16_t* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const s4*>(p));
}

// max / sum over lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float max_over_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    v = fmaxf(__builtin_bit_cast(float, static_cast<unsigned>(a[0])), __builtin_bit_cast(float, static_cast<unsigned>(a[1])));
    const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    return fmaxf(__builtin_bit_cast(float, static_cast<unsigned>(b[0])), __builtin_bit_cast(float, static_cast<unsigned>(b[1])));
}
__device__ __forceinline__ float sum_over_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    v = __builtin_bit_cast(float, static_cast<unsigned>(a[0])) + __builtin_bit_cast(float, static_cast<unsigned>(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    return __builtin_bit_cast(float, static_cast<unsigned>(b[0])) + __builtin_bit_cast(float, static_cast<unsigned>(b[1]));
}

// One block for the wave's 16 query heads. Lane (r, kg) has rows 16 J + r,
// tokens 4 kg .. + 3 of K and V. seen: the block's visible tokens; from:
// its first token's position minus the query's.
template <typename T, int D>
__device__ __forceinline__ void attend(State<D>& st, unsigned seen, int from, int kg, s4 (&k)[D / 16], s4 (&v)[D / 16],
                                       const s8 (&q)[D / 32], s4 ident, const Shape& shape, float slope) {
    constexpr int NJ = D / 16;
    const unsigned mine = (seen >> (4 * kg)) & 15u;
    if (seen != 0xffffu) {
        // Hidden tokens may hold anything, NaN too: they become zeros.
        s4 keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) keep[i] = (mine >> i) & 1u ? -1 : 0;
#pragma unroll
        for (int J = 0; J < NJ; ++J) {
            k[J] &= keep;
            v[J] &= keep;
        }
    }
    f4 sc = f4{0, 0, 0, 0};
#pragma unroll
    for (int J = 0; J < NJ; J += 2) {
        const f4 x = T::mfma16(k[J], ident, f4{0, 0, 0, 0});
        const f4 y = T::mfma16(k[J + 1], ident, f4{0, 0, 0, 0});
        const u4 kt = u4{T::cut2(x[0], x[1]), T::cut2(x[2], x[3]), T::cut2(y[0], y[1]), T::cut2(y[2], y[3])};
        sc = T::mfma16x32(__builtin_bit_cast(s8, kt), q[J / 2], sc);
    }
    float sv[4];
    const float d0 = static_cast<float>(from + 4 * kg);
    if (shape.cap > 0.0f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sv[i] = capped_score(sc[i], shape.scale, shape.cap);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) sv[i] = sc[i] * shape.scale;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sv[i] = __builtin_fmaf(slope, d0 + i, sv[i]);
    if (seen != 0xffffu) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sv[i] = (mine >> i) & 1u ? sv[i] : -INFINITY;
    }
    const float bm = max_over_groups(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])));
    if (__any(bm > st.m + kLag)) {
        const float m_new = fmaxf(st.m, bm);
        // A head that has seen no key keeps its zeros.
        const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.m - m_new);
#pragma unroll
        for (int J = 0; J < NJ; ++J) st.acc[J] *= alpha;
        st.l *= alpha;
        st.m = m_new;
    }
    const float c = (st.m == -INFINITY ? 0.0f : st.m) - weight_exp<T>;
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(sv[i] - c);
    st.l += (p[0] + p[1]) + (p[2] + p[3]);
    const unsigned h01 = T::down2(p[0], p[1]), h23 = T::down2(p[2], p[3]);
    float r[4];
    T::rest2(p[0], p[1], h01, r[0], r[1]);
    T::rest2(p[2], p[3], h23, r[2], r[3]);
    const s4 ph = __builtin_bit_cast(s4, u2{h01, h23});
    const s4 pl = __builtin_bit_cast(s4, u2{T::down2(r[0], r[1]), T::down2(r[2], r[3])});
#pragma unroll
    for (int J = 0; J < NJ; ++J) {
        st.acc[J] = T::mfma16(v[J], ph, st.acc[J]);
        st.acc[J] = T::mfma16(v[J], pl, st.acc[J]);
    }
}

}  // namespace scored
}  // namespace swiftllm
