// bf16_terms.h -- float32 operands on the bf16 matrix cores.
//
// A float32 goes in as the sum of up to three bf16 terms, each what is left rounded to
// nearest: below 2^-8 of it, of either sign.  One term is off by up to 2^-8 of the value, two
// by 2^-16, three by nothing (8 + 8 + 8 bits with the signs are a float32's 24).  A product of two
// such sums takes the pairs of terms whose magnitude matters; what the others leave out has either
// sign too, and does not add up over a sum:
//   three terms each, six pairs (of terms a, b with a + b < 3)   2^-23 of the product
//   two each, all four pairs                                     2^-15
//   two each, three pairs (a + b < 2)                            3 x 2^-16
// A float32 of 3.396e38 or more is past bf16's largest value, and counts as infinite.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

using f32x4 = __attribute__((ext_vector_type(4))) float;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// Two floats rounded to nearest, ties to even, in one word (v_cvt_pk_bf16_f32).
__device__ __forceinline__ uint32_t round2(float lo, float hi) {
    using f32x2 = __attribute__((ext_vector_type(2))) float;
    using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}
// Two floats' next term, and what is left of them.
__device__ __forceinline__ uint32_t take2(float& lo, float& hi) {
    const uint32_t t = round2(lo, hi);
    lo -= __uint_as_float(t << 16);
    hi -= __uint_as_float(t & 0xffff0000u);
    return t;
}

// Eight floats as N terms, in the order of an MFMA operand's eight values.
template <int N>
__device__ __forceinline__ void split8(float (&x)[8], u32x4 (&t)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) t[n][j] = n + 1 < N ? take2(x[2 * j], x[2 * j + 1]) : round2(x[2 * j], x[2 * j + 1]);
}
template <int N>
__device__ __forceinline__ void split4(f32x4 x, u32x2 (&t)[N]) {
    float y[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) t[n][j] = n + 1 < N ? take2(y[2 * j], y[2 * j + 1]) : round2(y[2 * j], y[2 * j + 1]);
}

// c + the products a[ta] x b[tb] with ta + tb < kMost, the smallest first
template <int NA, int NB, int kMost>
__device__ __forceinline__ f32x4 mfma_terms(const u32x4 (&a)[NA], const u32x4 (&b)[NB], f32x4 c) {
#pragma unroll
    for (int s = NA + NB - 2; s >= 0; --s)
#pragma unroll
        for (int ta = 0; ta < NA; ++ta) {
            const int tb = s - ta;
            if (tb >= 0 && tb < NB && s < kMost) c = mfma(a[ta], b[tb], c);
        }
    return c;
}

template <class T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ float to_float<uint16_t>(uint16_t x) {
    return __uint_as_float((uint32_t)x << 16);
}
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ uint16_t from_float<uint16_t>(float x) {  // to nearest, ties to even
    return __builtin_bit_cast(uint16_t, __float2bfloat16(x));
}
