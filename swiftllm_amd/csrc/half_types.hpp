// The two 16-bit floating types of the attention step (SWIFTLLM_HIP_F16,
// SWIFTLLM_HIP_BF16). Kernels move their values as 16-bit patterns and go
// through these structs for arithmetic.
#pragma once

#include "common.hpp"

namespace swiftllm {

typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef float f16x __attribute__((ext_vector_type(16)));

__device__ __forceinline__ s8 join8(s4 lo, s4 hi) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

struct F16 {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v4 __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ float up(uint16_t b) { return static_cast<float>(__builtin_bit_cast(_Float16, b)); }
    // Round to nearest even.
    static __device__ __forceinline__ uint16_t down(float v) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v)); }
    static __device__ __forceinline__ unsigned down2(float a, float b) {
        typedef _Float16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, v2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
    }
    static __device__ __forceinline__ uint16_t one() { return 0x3c00; }
    static __device__ __forceinline__ f4 mfma16(s4 a, s4 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(v4, a), __builtin_bit_cast(v4, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f4 mfma16x32(s8 a, s8 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f16x mfma32(s8 a, s8 b, f16x c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    // Two values toward zero (exact for values of the type).
    static __device__ __forceinline__ unsigned cut2(float a, float b) {
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(a, b));
    }
    // a and b minus the two values of a cut2.
    static __device__ __forceinline__ void rest2(float a, float b, unsigned h, float& ra, float& rb) {
        asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(h), "v"(a));
        asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(h), "v"(b));
    }
};

struct BF16 {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ float up(uint16_t b) { return __builtin_bit_cast(float, static_cast<unsigned>(b) << 16); }
    static __device__ __forceinline__ uint16_t down(float v) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }
    static __device__ __forceinline__ unsigned down2(float a, float b) {
        typedef __bf16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, v2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
    }
    static __device__ __forceinline__ uint16_t one() { return 0x3f80; }
    static __device__ __forceinline__ f4 mfma16(s4 a, s4 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f4 mfma16x32(s8 a, s8 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f16x mfma32(s8 a, s8 b, f16x c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ unsigned cut2(float a, float b) {
        return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302u);
    }
    static __device__ __forceinline__ void rest2(float a, float b, unsigned h, float& ra, float& rb) {
        ra = a - __builtin_bit_cast(float, h << 16);
        rb = b - __builtin_bit_cast(float, h & 0xffff0000u);
    }
};

}  // namespace swiftllm
