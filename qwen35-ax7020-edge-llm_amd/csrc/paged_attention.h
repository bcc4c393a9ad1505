// paged_attention.h -- what paged_attention.hip and its host code share.  Not part of
// the public ABI.
#pragma once
#include <algorithm>
#include <cstddef>

#include "kv_cache.h"

constexpr int ATTN_MOST = 1024;  // workgroups of a call, at most
constexpr int ATTN_HELD = 1024;  // places whose tiles of keys a workgroup remembers

// How a call is laid out: from its sizes alone.  A tile of rows is `rows` rows of one sequence on one key
// head, row m being token m / group and query head m % group of it.
struct AttnPlan {
    int group;    // query heads of a key head
    int few;      // attn_step_kernel: up to 16 rows
    int dim;      // of the kernel: 64, 128 or 256
    int blocks;   // of 16 rows of a wavefront
    int waves;    // of a workgroup
    int rows, rows_log;  // of a tile: 16 blocks waves, a power of two
    int each;     // tiles of rows of a sequence, without starts
    int keys;     // of a tile of keys
    int grid;     // workgroups
    int extra;    // tiles of keys that a tile of rows counts for besides its own
    int least;    // tiles of a workgroup's share
    int rows_most;    // of a sequence and key head, as far as the host knows
    int shared;   // tiles of rows and key heads, at most, if they are few and each in many parts; else 0
    size_t desc_at;   // AttnDesc [grid]
    size_t flag_at;   // int [grid]: there is one
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
    // Up to 16 rows: attn_step_kernel (64 sequences of 4,000 keys, 16 rows of 256 bf16 elements, 130 us, by attn_kernel
    // 135; 32 of 2,000, 128 float32 ones, 47 for 61; but 48 of 2,000 and 16 rows on average, many with more, 71 for
    // 55).  By the mean, for the lengths are on the device: a batch of few long sequences and many short ones pays for it
    // (255 tokens on 1,000 keys each and a chunk of 512 on 30,000 in one call 1,147 us, in two 106 and 172; 32 tokens on
    // 8,000 and one of 2,048 on 2,048 236 | 108 and 109; 1,023 empty places and a prompt of 2,048 226 | 74).
    p.few = mean <= 16;
    // More: as many rows to a tile as there are, so that its keys are read once.  Two wavefronts at least, to copy (one
    // | two: 48 sequences of 28 rows of 128 elements 70 | 62 us, 64 of 32 rows of 256 174 | 149).  Of 256 bf16 elements
    // four wavefronts with their 340 registers are one workgroup a compute unit, two are two (two | four | eight at 64
    // sequences of 128 rows 223 | 240 | 241, one of 128 rows 44 | 45 | 51, at 160 rows 271 | - | 235); of 128 elements
    // two are (48 of 125 rows, two | four | eight: 108 | 93 | 116).
    p.blocks = bf16 && !p.few ? 2 : 1;
    p.waves = p.few ? 1 : mean <= (size_t)32 * p.blocks ? 2 : mean <= (size_t)64 * p.blocks ? 4 : 8;
    if (bf16 && p.dim == 256 && p.waves == 4) p.waves = 2;
    p.rows = 16 * p.blocks * p.waves;
    p.rows_log = 31 - __builtin_clz(p.rows);
    p.each = a.starts || !a.n_seq ? 0 : (a.rows / a.n_seq * p.group + p.rows - 1) / p.rows;
    // (64 keys: half as many waits for the copies; four wavefronts gained nothing by it)
    p.keys = p.few || (bf16 && p.waves == 8) ? 64 : 32;
    // attn_kernel: as many as are at work at a time, by LDS and registers (8 wavefronts a compute unit), up to four a
    // unit.  attn_step_kernel: two a unit, though of 256 float32 elements LDS holds one at a time (64 sequences of 4,096
    // keys 200 us, 5.4 TB/s, for 105 and 5.1 with bf16).
    const size_t lds = (size_t)4 * p.keys * p.dim * (bf16 ? 2 : 4) + ATTN_HELD * 4 + 256;
    p.grid = 256 * (p.few ? 2 : (int)std::min<size_t>(std::min(4, 8 / p.waves), 160 * 1024 / lds));
    // A part is written and read again, 8 bytes an output: of many rows as much as several tiles of keys (one sequence of
    // 6,000 tokens with 26 drafted ones: 1 | 2 | 4 | 8 tiles 96 | 57 | 42 | 40 us; a prompt of 2,048 73 | 71 | 71 | 87).
    p.least = p.few ? 1 : 4;
    // What a tile of rows costs by itself, its first keys' latency, masks and results, in tiles of keys.  Left out, the
    // workgroups with a sequence's first rows, many tiles of rows with few keys, are the last by far: a prompt of 16,384
    // tokens with 0 | 2 | 4 | 8 tiles of 64 keys 1,764 | 1,468 | 1,245 | 1,160 us; 8,192 of 16 heads of 128 589 | 435 |
    // 372 | 381; float32 prompts with 0 | 1 | 2 | 4 tiles of 32 107 | 98 | 98 | 105.
    p.extra = p.few ? 1 : bf16 ? std::max(256, 2 * p.dim) / p.keys : 2;
    p.rows_most = a.starts || !a.n_seq ? p.rows : a.rows / a.n_seq * p.group;
    // Where there are about eight parts or more of each, 16 wavefronts join them, by a workgroup for each tile and not
    // each share (without | with: a token of one sequence of 4,096 19.0 | 15.7 us, 26 drafted ones of 6,000 64 | 33).
    const size_t units = (a.starts ? (size_t)a.rows * p.group / p.rows + a.n_seq : (size_t)a.n_seq * p.each) * a.heads_k;
    p.shared = units * 8 <= (size_t)p.grid ? (int)units : 0;
    size_t at = 0;
    auto put = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.desc_at = put((size_t)p.grid * 32);
    p.flag_at = put((size_t)p.grid * 4);
    p.stat_at = put((size_t)2 * p.grid * p.rows * 8);
    p.part_at = put((size_t)2 * p.grid * p.rows * p.dim * 4);
    p.total = at;
    return p;
}

// Places in the cache as 32-bit multiples of the largest power of two that divides its strides, 16 bytes or more: a cache
// may span 2^32 of them (64 GiB at least, 4 TiB with 1 KiB a token).
struct AttnUnits {
    Divisor divisor;       // by the tokens of a page
    uint32_t page, token;  // their strides in units
    int log;
};
inline AttnUnits attn_units(const attn_dev_args& a) {
    const uint64_t es = a.dtype == QWEN_BF16 ? 2 : 4, page = a.cache_page * es, token = a.cache_token * es;
    AttnUnits u{divisor(a.page), 0, 0, 4};
    while (u.log < 31 && (page | token) >> u.log && ((page | token) >> u.log & 1) == 0) ++u.log;
    u.page = (uint32_t)(page >> u.log);
    u.token = (uint32_t)(token >> u.log);
    return u;
}
// The last place's number is below 2^32 - 1.
inline bool attn_units_fit(const attn_dev_args& a) {
    const AttnUnits u = attn_units(a);
    const uint64_t es = a.dtype == QWEN_BF16 ? 2 : 4;
    if ((uint64_t)a.cache_page * es >> u.log > 0xffffffffull || (uint64_t)a.cache_token * es >> u.log > 0xffffffffull) return false;
    return (unsigned __int128)u.page * std::max(a.pages - 1, 0) + (unsigned __int128)u.token * (a.page - 1) < 0xffffffffull;
}

hipError_t attn_launch_paged(const attn_dev_args& a, const AttnPlan& p, hipStream_t s);
