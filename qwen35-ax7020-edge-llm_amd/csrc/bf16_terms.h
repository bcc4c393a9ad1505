// bf16_terms.h -- float32 operands on the bf16 matrix cores.
//
// A float32 goes in as the sum of up to three bf16 terms, cut (not rounded) from
// its 24 bits: three hold it exactly, two to 2^-16.  A product of two such sums
// takes the pairs of terms whose magnitude matters.
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

// Takes its first term, its upper 16 bits, from x.
__device__ __forceinline__ void cut(float& x) { x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// The upper halves of two words in one.
__device__ __forceinline__ uint32_t pack(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302); }

// Eight floats as N terms, in the order of an MFMA operand's eight values.
template <int N>
__device__ __forceinline__ void split8(float (&x)[8], u32x4 (&t)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            t[n][j] = pack(__float_as_uint(x[2 * j]), __float_as_uint(x[2 * j + 1]));
            if (n + 1 < N) cut(x[2 * j]), cut(x[2 * j + 1]);
        }
}
template <int N>
__device__ __forceinline__ void split4(f32x4 x, u32x2 (&t)[N]) {
    float y[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            t[n][j] = pack(__float_as_uint(y[2 * j]), __float_as_uint(y[2 * j + 1]));
            if (n + 1 < N) cut(y[2 * j]), cut(y[2 * j + 1]);
        }
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
