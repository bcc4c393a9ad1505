// linear_attention.h -- what linear_attention.hip and its host code share.
// Not part of the public ABI.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "qwen_kernels.h"

// Tokens of a chunk: within one the recurrence is a triangular system.
constexpr int GDN_CHUNK = 64;
constexpr int GDN_MAX_DIM = 256;
// Sequences of up to so many tokens may go token by token, past the latency of a chunk: one of 16 heads of 128 with
// 4 | 16 | 32 tokens in bf16 5.4 | 11 | 18 us, in a chunk 14; 64 of them with 4 | 16 tokens 44 | 73 us, in chunks
// 104 | 108.  That is a third launch where longer ones may be in the call too (their lengths are on the
// device); it is made if the chunks would go over the chip more than once and the average sequence is that short.
constexpr int GDN_SHORT = 16;

// Where gdn_chunk_kernel leaves a chunk's operands for gdn_scan_kernel, as
// byte counts.  Place of chunk c of sequence s: starts[s] / 64 + s + c, different for
// every chunk, below rows / 64 + n_seq.  Where only sequences of more than GDN_SHORT tokens
// have chunks: starts[s] / GDN_SHORT + c, so different too, below rows / GDN_SHORT.  The buffer has
// room for either, and a smaller call never needs a larger one.
struct GdnWork {
    int ks;            // steps of 32 along dim_k (1, 2, 4 or 8: dim_k is padded to 32 ks)
    int nt;            // bf16 terms of an input (1: bf16, 3: float32)
    int no;            // bf16 terms of what only outputs need (2 or 3)
    size_t key_bytes;  // per chunk and key head: K and Q as operands
    size_t tri_bytes;  // per chunk and value head: T and P fragments, the decays
    int short_to;      // sequences of up to so many tokens go token by token (-1: none)
    size_t places;     // chunks' places that this call may use
    size_t n_chunks;   // and that the buffer has
    size_t total;
};

inline GdnWork gdn_work(const gdn_dev_args& a) {
    GdnWork w{};
    w.ks = a.dim_k <= 32 ? 1 : a.dim_k <= 64 ? 2 : a.dim_k <= 128 ? 4 : 8;
    w.nt = a.dtype == QWEN_BF16 ? 1 : 3;
    w.no = a.dtype == QWEN_BF16 ? 2 : 3;
    w.key_bytes = (size_t)2 * 4 * w.ks * w.nt * 1024;
    w.tri_bytes = (size_t)(6 * 3 + 6 * w.no) * 1024 + 1024;
    const size_t rows = (size_t)a.rows, n_seq = (size_t)a.n_seq, each = (size_t)a.heads_v * ((a.dim_v + 31) / 32);
    const bool many = n_seq * each > 256 && rows <= GDN_SHORT * n_seq;
    w.short_to = rows <= GDN_SHORT || many ? GDN_SHORT : -1;
    w.places = w.short_to < 0 ? rows / GDN_CHUNK + n_seq : rows / GDN_SHORT;
    w.n_chunks = rows / GDN_CHUNK + std::min(n_seq, std::max(rows / GDN_SHORT + 1, 256 / each));
    w.total = w.n_chunks * (w.key_bytes * a.heads_k + w.tri_bytes * a.heads_v);
    return w;
}

hipError_t gdn_launch_prompt(const gdn_dev_args& a, const GdnWork& w, hipStream_t s);
hipError_t gdn_launch_step(const gdn_dev_args& a, hipStream_t s);
