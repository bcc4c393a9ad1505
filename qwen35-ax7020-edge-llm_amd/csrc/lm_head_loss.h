// lm_head_loss.h -- what lm_head_loss.hip and its host code share.  Not part of
// the public ABI.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "qwen_kernels.h"

constexpr int LHL_TILE = 128;   // vocabulary rows of the smallest tile of logits
constexpr int LHL_WIDE = 256;   // of a large tile; pieces of the vocabulary are multiples of it
constexpr int LHL_STEP = 64;    // terms of a sum that a tile takes in one step

// The caller's work buffer: byte offsets of its parts.
struct LossWork {
    int terms;          // bf16 terms of a hidden state, and of a logit's gradient (1: bf16, 3: float32)
    int pitch;          // hidden rounded up to LHL_STEP
    int vtiles;         // such tiles in the vocabulary
    int piece;          // vocabulary rows whose logits' gradients are held at a time
    int splits;         // parts of a piece that grad_h's sum over the vocabulary is split into
    size_t rows_at;     // int: original row of each counted row
    size_t target_at;   // int: its target
    size_t place_at;    // int: original row -> counted row, -1 ignored, -2 no such target
    size_t logit_at;    // float: the target's logit
    size_t lse_at, gl_at;  // float: lse and the loss's gradient of each counted row
    size_t rest_at;     // float: what the rounding of D left out at the target (the gradient of bf16 states)
    size_t h_at;        // bf16 [terms][rows][pitch]
    size_t part_at;     // float2 [rows][vtiles]: maximum and sum of exponentials of a tile's logits
    size_t d_at;        // bf16 [terms][rows][piece]
    size_t sum_at;      // float [splits][rows][pitch]
    size_t total;
};

inline LossWork loss_work(const lm_head_loss_args& a, bool grad, bool grad_h) {
    LossWork w{};
    const size_t n = (size_t)a.rows;
    w.terms = a.dtype == QWEN_BF16 ? 1 : 3;
    w.pitch = (a.hidden + LHL_STEP - 1) / LHL_STEP * LHL_STEP;
    w.vtiles = (a.vocab + LHL_TILE - 1) / LHL_TILE;
    size_t at = 512;  // the count, the largest weight, and a line of zeros
    auto put = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    w.rows_at = put(4 * n);
    w.target_at = put(4 * n);
    w.place_at = put(4 * n);
    w.logit_at = put(4 * n);
    w.lse_at = put(4 * n);
    w.gl_at = put(4 * n);
    if (grad && w.terms == 1) w.rest_at = put(4 * n);
    w.h_at = put(2 * n * w.terms * w.pitch);
    if (!grad) {
        w.part_at = put(8 * n * w.vtiles);
    } else {
        // pieces whose gradients stay under 128 MiB: they and their part of the table fit the 256 MiB
        // last-level cache that they are read from again (4096 bf16 rows: 1.52 ms; 256 or 512 MiB 1.59); powers
        // of two, whose tiles go over the chip a whole number of times (4096 float32 rows: 4096 columns
        // 4.8 ms, the 5120 that fit 5.8)
        const size_t whole = ((size_t)a.vocab + LHL_WIDE - 1) / LHL_WIDE * LHL_WIDE;
        size_t fit = 1024;
        while (fit < whole && 2 * fit * 2 * n * w.terms <= (size_t)128 << 20) fit *= 2;
        w.piece = (int)std::min(whole, fit);
        w.d_at = put(2 * n * w.terms * w.piece);
        if (grad_h) {
            // one tile's sum over the vocabulary split into as many as run at a time, once over the chip
            const bool wide = w.terms == 3 && n > 64;  // (256 x 128, one a compute unit, else 128 x 128 or 64, two)
            const size_t bm = wide ? 256 : 128, at_once = wide ? 256 : 512;
            const size_t tiles = std::max<size_t>(1, (w.pitch + bm - 1) / bm * ((n + 127) / 128));
            const size_t steps = (size_t)w.piece / LHL_STEP;
            w.splits = (int)std::max<size_t>(1, std::min(steps / 4, at_once / tiles));
            w.sum_at = put(4 * n * w.splits * w.pitch);
        }
    }
    w.total = at;
    return w;
}

hipError_t lhl_launch_loss(const lm_head_loss_args& a, const LossWork& w, hipStream_t s);
hipError_t lhl_launch_grad(const lm_head_loss_args& a, const LossWork& w, hipStream_t s);
