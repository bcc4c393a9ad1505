// kv_cache.h -- what kv_cache.hip, paged_attention.hip and their host code share.  Not
// part of the public ABI.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "qwen_kernels.h"

// n / d for 0 <= n < 2^31 by one product (d 1 to 2^31): with l = ceil(log2 d) and
// m = floor(2^(31 + l) / d) + 1, n m / 2^(31 + l) is off by less than 2^-l <= 1 / d from above.
struct Divisor {
    uint32_t m;
    int shift;
};
inline Divisor divisor(uint32_t d) {
    int l = 0;
    while ((1u << l) < d) ++l;
    return {(uint32_t)((1ull << (31 + l)) / d + 1), 31 + l};
}
__host__ __device__ inline uint32_t divide(uint32_t n, Divisor d) { return (uint32_t)((uint64_t)n * d.m >> d.shift); }

#if defined(__HIP_DEVICE_COMPILE__) || defined(__HIPCC__)
// The rows of sequence s: starts[s] .. starts[s + 1] - 1, or rows / n_seq each.  Values that are not
// ascending or outside the rows give fewer rows, never others' memory.
struct Span {
    int first, count;
};
__device__ __forceinline__ Span span_of(const int32_t* starts, int rows, int n_seq, int s) {
    if (!starts) {
        const int each = rows / n_seq;
        return {s * each, each};
    }
    const int lo = min(max(starts[s], 0), rows), hi = min(max(starts[s + 1], lo), rows);
    return {lo, hi - lo};
}
#endif

hipError_t rope_launch(const rope_dev_args& a, bool back, hipStream_t s);
hipError_t kv_launch_append(const kv_dev_append_args& a, hipStream_t s);
hipError_t attn_launch_tree(const attn_dev_tree_args& a, hipStream_t s);
