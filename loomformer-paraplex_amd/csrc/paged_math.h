// Device pieces that the attention kernels over a paged cache share: reductions
// over the lanes of a score column, the running reference of a softmax, the
// products of 16-bit types, the rotation.
#pragma once

#include "loom_common.h"

namespace loom {

typedef float pg_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 pg_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 pg_f16x8 __attribute__((ext_vector_type(8)));

// Lanes 16 and 32 apart: the two values of each pair in every lane of it
__device__ __forceinline__ float2 pair16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float2 pair32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_16_32(float v) {
    float2 p = pair16(v, v);
    v = fmaxf(p.x, p.y);
    p = pair32(v, v);
    return fmaxf(p.x, p.y);
}
__device__ __forceinline__ float sum_16_32(float v) {
    float2 p = pair16(v, v);
    v = p.x + p.y;
    p = pair32(v, v);
    return p.x + p.y;
}

// The exponents' running reference: it follows the maximum (in powers of two) only
// where that is LAG beyond it, so that the sums are hardly ever rescaled.  A factor of
// 2^8 costs nothing where the weights keep an fp32's range of exponents.
constexpr float kPgLag = 8.0f;
__device__ __forceinline__ float raised(float ref, float most, float lag = kPgLag) { return most > ref + lag ? most : ref; }

// Element pair helpers by type
template <typename T> struct Mfma16;
template <> struct Mfma16<bf16_t> {
    static constexpr float kLag = kPgLag, kShift = 0.0f;
    __device__ __forceinline__ static pg_f32x4 dot(uint4 a, uint4 b, pg_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_bf16x8, a),
                                                       __builtin_bit_cast(pg_bf16x8, b), c, 0, 0, 0);
    }
    __device__ __forceinline__ static uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
};
template <> struct Mfma16<f16_t> {
    // half's exponents end at 2^15 and its normal values at 2^-14, so the reference lies
    // 2^13 below the maximum it follows and lags by 2^2 at most: weights from 2^-27 of
    // the largest on keep their 11 bits, and what a smaller one loses is at most 2^-38
    // of the largest (2^-14 in a row of 2^24 tokens)
    static constexpr float kLag = 2.0f, kShift = 13.0f;
    __device__ __forceinline__ static pg_f32x4 dot(uint4 a, uint4 b, pg_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pg_f16x8, a),
                                                      __builtin_bit_cast(pg_f16x8, b), c, 0, 0, 0);
    }
    __device__ __forceinline__ static uint32_t pack(float a, float b) {
        f16_t x, y;
        st(&x, a);
        st(&y, b);
        return (uint32_t)x.x | ((uint32_t)y.x << 16);
    }
};

// x c + y s of the rotation.  For the 16-bit types in 64 bits, where both products are
// exact; rounded to fp32 here and to the type when it is stored, the value is the exact
// one's rounding but where fp32's falls on the middle of two values: of 2^24 random ones
// 1058 of half and 114 of bf16 come out a step beside it (all in fp32 2966 and 477).
template <typename T>
__device__ __forceinline__ float turn(float x, float c, float y, float s) {
    if constexpr (sizeof(T) == 2) return (float)fma((double)x, (double)c, (double)y * (double)s);
    else return fmaf(x, c, y * s);
}

}  // namespace loom
