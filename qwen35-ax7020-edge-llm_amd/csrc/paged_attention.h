// paged_attention.h -- what paged_attention.hip and its host code share.  Not part of
// the public ABI.
#pragma once
#include <algorithm>
#include <cstddef>

#include "kv_cache.h"

constexpr int ATTN_HELD = 1024;  // places whose tiles of keys a workgroup remembers

// How a call is laid out: from its sizes alone.  A tile of rows is `rows` rows of one sequence on one key
// head, row m being token m / group and query head m % group of it.
struct AttnPlan {
    int group;    // query heads of a key head
    int dim;      // of the kernel: 64, 128 or 256
    int blocks;   // of 16 rows of a wavefront
    int waves;    // of a workgroup
    int rows;     // of a tile: 16 blocks waves
    int keys;     // of a tile of keys
    int grid;     // workgroups
    size_t desc_at;   // AttnDesc [grid]
    size_t stat_at;   // float2 [2 grid][rows]: a part's maximum and sum
    size_t part_at;   // float [2 grid][rows][dim]
    size_t total;
};

inline AttnPlan attn_plan(const attn_dev_args& a) {
    AttnPlan p{};
    const bool bf16 = a.dtype == QWEN_BF16;
    p.group = a.heads_q / a.heads_k;
    p.dim = a.dim <= 64 ? 64 : a.dim <= 128 ? 128 : 256;
    // rows of an average sequence and key head
    const size_t mean = ((size_t)a.rows * p.group + std::max(a.n_seq, 1) - 1) / std::max(a.n_seq, 1);
    p.blocks = bf16 && mean > 16 ? 2 : 1;
    p.waves = mean <= (size_t)16 * p.blocks ? 1 : mean <= (size_t)32 * p.blocks ? 2 : mean <= (size_t)64 * p.blocks ? 4 : 8;
    p.rows = 16 * p.blocks * p.waves;
    p.keys = bf16 && p.waves == 8 ? 64 : 32;
    // as many as are at work at a time, by LDS and registers (8 wavefronts a compute unit), up to four a unit
    const size_t lds = (size_t)4 * p.keys * p.dim * (bf16 ? 2 : 4) + ATTN_HELD * 4 + 256;
    p.grid = 256 * (int)std::min<size_t>(std::min(4, 8 / p.waves), 160 * 1024 / lds);
    size_t at = 0;
    auto put = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.desc_at = put((size_t)p.grid * 32);
    p.stat_at = put((size_t)2 * p.grid * p.rows * 8);
    p.part_at = put((size_t)2 * p.grid * p.rows * p.dim * 4);
    p.total = at;
    return p;
}

hipError_t attn_launch_paged(const attn_dev_args& a, const AttnPlan& p, hipStream_t s);
