// matrix.hpp -- operands of the matrix cores, shared by the gfx950 kernels of this library: 16x16x32 bf16
// products with float sums, and 8-bit and 4-bit codes as bf16 operands (exact: no code has more than 8
// significant bits).
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "lanes.hpp"

namespace {

typedef __bf16 Bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
typedef int I32x2 __attribute__((ext_vector_type(2)));
typedef float F32x4 __attribute__((ext_vector_type(4)));

// Lane 16 g + r holds eight values of row r of a and of column r of b, the same eight places of the sum for
// both; of the result it holds rows 4 g .. 4 g + 3 of column r.
__device__ __forceinline__ F32x4 mfma(Bf16x8 a, Bf16x8 b, F32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// A lane's 16-byte chunk of 8-bit codes as 16 bf16 values, two operands of 8.  Every code
// is exact in bf16: INT8 has at most 7 significant bits and a sign (-128 = -2^7), E4M3 four.
template <bool kFp8>
__device__ __forceinline__ void codes_to_bf16(U32x4 w, Bf16x8 (&o)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t p[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t c = w[2 * h + i];
            if constexpr (kFp8) {
                p[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, false));
                p[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, true));
            } else {
                float f[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) f[k] = (float)(int8_t)(c >> (8 * k));
                // The high halves of two floats whose low halves are zero.
                p[2 * i] = __builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u);
                p[2 * i + 1] = __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u);
            }
        }
        o[h] = __builtin_bit_cast(Bf16x8, U32x4{p[0], p[1], p[2], p[3]});
    }
}

// Eight 4-bit codes as a matrix-core operand.  FP4: the values, in order.  INT4: 8 + code, which the
// callers take off again: a half byte alone in a byte is an E4M3 number 2^-9 times it, and one
// instruction makes bf16 of two; in the order 0 2 4 6 1 3 5 7.
template <bool kFp4>
__device__ __forceinline__ Bf16x8 operand(uint32_t w) {
    U32x4 d;
    if constexpr (kFp4) {
        d[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0));
        d[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1));
        d[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2));
        d[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3));
    } else {
        const uint32_t even = w & 0x0F0F0F0Fu, odd = (w >> 4) & 0x0F0F0F0Fu;
        d[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(even, 512.0f, false));
        d[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(even, 512.0f, true));
        d[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(odd, 512.0f, false));
        d[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(odd, 512.0f, true));
    }
    return __builtin_bit_cast(Bf16x8, d);
}

// The place of code r of eight in operand().
template <bool kFp4>
__device__ __forceinline__ int place(int r) { return kFp4 ? r : ((r & 1) << 2) + (r >> 1); }

// Eight bf16 values in the order of operand()'s.
template <bool kFp4>
__device__ __forceinline__ Bf16x8 in_order(const uint4& w) {
    U32x4 d = {w.x, w.y, w.z, w.w};
    if constexpr (!kFp4) {
        d[0] = (w.x & 0xffffu) | (w.y << 16);
        d[1] = (w.z & 0xffffu) | (w.w << 16);
        d[2] = (w.x >> 16) | (w.y & 0xffff0000u);
        d[3] = (w.z >> 16) | (w.w & 0xffff0000u);
    }
    return __builtin_bit_cast(Bf16x8, d);
}

// Words handed between workgroups of different XCDs: written through, read past the own L2.
__device__ __forceinline__ void put(float* p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get(const float* p) {
    return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// put() of four neighbouring floats (16-byte aligned) in one store.
__device__ __forceinline__ void put4(float* p, const F32x4& v) {
    asm volatile("global_store_dwordx4 %0, %1, off sc1" ::"v"(p), "v"(v) : "memory");
}

// exp2(m - M) with an empty side (m = -inf) weighing nothing.
__device__ __forceinline__ float weight_of(float m, float M) { return m == -INFINITY ? 0.0f : exp2_fast(m - M); }

// Keeps a wave's rare branch from becoming selects that every tile runs.
__device__ __forceinline__ void stay_a_branch() { asm volatile(""); }

}  // namespace
