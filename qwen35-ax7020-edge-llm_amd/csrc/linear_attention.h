// linear_attention.h -- what linear_attention.hip and its host code share.
// Not part of the public ABI.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "qwen_kernels.h"

// Tokens of a chunk: within one the recurrence is a triangular system.
constexpr int GDN_CHUNK = 64;
constexpr int GDN_MAX_DIM = 256;

// Where gdn_chunk_kernel leaves a chunk's operands for gdn_scan_kernel, as
// byte counts.  Chunk slot id = starts[s] / 64 + s + (chunk of sequence s):
// different for every chunk, below rows / 64 + n_seq.
struct GdnWork {
    int ks;            // steps of 32 along dim_k (1, 2, 4 or 8: dim_k is padded to 32 ks)
    int nt;            // bf16 terms of an input (1: bf16, 3: float32)
    int no;            // bf16 terms of what only outputs need (2 or 3)
    size_t key_bytes;  // per chunk and key head: K and Q as operands
    size_t tri_bytes;  // per chunk and value head: T and P fragments, the decays
    size_t n_chunks, total;
};

inline GdnWork gdn_work(const gdn_dev_args& a) {
    GdnWork w{};
    w.ks = a.dim_k <= 32 ? 1 : a.dim_k <= 64 ? 2 : a.dim_k <= 128 ? 4 : 8;
    w.nt = a.dtype == QWEN_BF16 ? 1 : 3;
    w.no = a.dtype == QWEN_BF16 ? 2 : 3;
    w.key_bytes = (size_t)2 * 4 * w.ks * w.nt * 1024;
    w.tri_bytes = (size_t)(6 * 3 + 6 * w.no) * 1024 + 1024;
    w.n_chunks = (size_t)(a.rows / GDN_CHUNK) + (size_t)a.n_seq;
    w.total = w.n_chunks * (w.key_bytes * a.heads_k + w.tri_bytes * a.heads_v);
    return w;
}

hipError_t gdn_launch_prompt(const gdn_dev_args& a, const GdnWork& w, hipStream_t s);
hipError_t gdn_launch_step(const gdn_dev_args& a, hipStream_t s);
