// Tiles of K and V in LDS for 32x32x16 products, which the four waves of a workgroup
// load and all read: in scored_prefill.hip a stage of 64 keys, four blocks, by a wave
// each; in shared_decode.hip a step of two blocks, of which two waves load the K and
// two the V.
#pragma once

#include <type_traits>

#include "scored_core.hpp"

namespace swiftllm {
namespace scored {

constexpr int kStage = 64;             // keys

typedef __attribute__((address_space(3))) s4 lds_s4;

// LDS of a stage of four blocks, in halves: four K tiles [d][16], then four V tiles in
// operand order. The second K tile of a pair sits 128 bytes off, so that the
// rows an operand read takes from both fall in different banks.
template <int D>
struct Stage {
    static constexpr int kTile = D * kBlockTokens;
    static constexpr int kOdd = kTile + 64;
    static constexpr int kPair = 2 * kTile + 128;
    static constexpr int kK = 2 * kPair;
    static constexpr int kV = 4 * kTile;
};

// A block's tile of one kv head, `off` elements into its cache; with no bytes
// there is nothing to load.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const uint16_t* cache, size_t off, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(cache + off), 0, bytes, kRsrcWord3);
}

template <int D>
__device__ __forceinline__ void stage_k(const uint16_t* cache, uint16_t* ks, int w, size_t off, int bytes, int lane) {
    const __amdgpu_buffer_rsrc_t rk = tile_rsrc(cache, off, bytes);
    uint16_t* const k = ks + (w >> 1) * Stage<D>::kPair + (w & 1) * Stage<D>::kOdd;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, to_lds(k + 512 * i), 16, 16u * lane, 1024u * i, 0, 0);
    }
}

// Each 32-row piece's 16-byte chunks: the rows' first 8 tokens, then their last 8.
template <int D>
__device__ __forceinline__ void stage_v(const uint16_t* cache, uint16_t* vs, int w, size_t off, int bytes, int lane) {
    const __amdgpu_buffer_rsrc_t rv = tile_rsrc(cache, off, bytes);
    uint16_t* const v = vs + w * Stage<D>::kTile;
    const unsigned vo = 32u * (lane & 31) + 16u * (lane >> 5);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, to_lds(v + 512 * i), 16, vo, 1024u * i, 0, 0);
    }
}

// Row operand of K: 16 rows of a pair of blocks.
__device__ __forceinline__ s8 k_rows(const uint16_t* p) {
    const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(const_cast<uint16_t*>(p)));
    const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(const_cast<uint16_t*>(p + 64)));
    return join8(x, y);
}

// S^T of the 32 keys of a stage's pair of blocks.
template <typename T, int D>
__device__ __forceinline__ void qk_pair(f16x& sc, const uint16_t* kl, const s8 (&q)[D / 16]) {
    sc = f16x{};
#pragma unroll
    for (int J = 0; J < D / 16; ++J) {
        sc = T::mfma32(k_rows(kl + 256 * J), q[J], sc);
    }
}

// Bits 0 .. n - 1 of 8.
__device__ __forceinline__ unsigned low8(int n) { return (1u << min(max(n, 0), 8)) - 1u; }

// Zeroes the values of the wave's V tile in LDS that are not finite, once its
// loads have landed; which of its 16 keys held one.
template <typename T, int D>
__device__ __forceinline__ unsigned clean_v(uint16_t* vs, int w, int lane) {
    constexpr unsigned kExp = std::is_same<T, F16>::value ? 0x7c007c00u : 0x7f807f80u;
    constexpr unsigned kUlp = std::is_same<T, F16>::value ? 0x04000400u : 0x00800080u;
    uint16_t* const p = vs + w * Stage<D>::kTile + 8 * lane;
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const u4 u = *reinterpret_cast<const u4*>(p + 512 * i);
#pragma unroll
        for (int z = 0; z < 4; ++z) bad |= (u[z] & kExp) + kUlp;
    }
    if (!__any((bad & 0x80008000u) != 0)) return 0;
    unsigned mine = 0;
#pragma unroll 1
    for (int i = 0; i < D / 32; ++i) {
#pragma unroll 1
        for (int z = 0; z < 8; ++z) {
            if ((p[512 * i + z] & (kExp & 0xffffu)) == (kExp & 0xffffu)) {
                p[512 * i + z] = 0;
                mine |= 1u << z;
            }
        }
    }
    // Lanes 0 .. 31 hold keys 0 .. 7 of the block, the others 8 .. 15.
    unsigned keys = 0;
    for (int z = 0; z < 8; ++z) {
        const unsigned long long who = __ballot((mine >> z) & 1u);
        keys |= (static_cast<unsigned>(who) != 0 ? 1u << z : 0u) | (static_cast<unsigned>(who >> 32) != 0 ? 256u << z : 0u);
    }
    return keys;
}

// a + the two values of a packed pair.
__device__ __forceinline__ float add_pair(F16, unsigned p, float a) {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, p), v2{1, 1}, a, false);
}
__device__ __forceinline__ float add_pair(BF16, unsigned p, float a) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, p), __builtin_bit_cast(v2, 0x3f803f80u), a, false);
}

}  // namespace scored
}  // namespace swiftllm
