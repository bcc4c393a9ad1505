// qwen_text_api.cpp -- C ABI of the operators over a text's tokens
// (include/qwen_kernels.h): gated linear attention, the head's loss.  Arguments are
// checked here; the library's lock is not held while a kernel is launched, and no
// state of the library is used.
#include <hip/hip_runtime.h>

#include <mutex>

#include "host_internal.h"
#include "linear_attention.h"
#include "lm_head_loss.h"

using namespace qhost;

namespace {

int init() {
    std::lock_guard<std::mutex> lk(g.mu);
    return ensure_init_locked();
}

bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

int refuse(const char* who, const char* why) {
    set_error("%s: %s", who, why);
    return BFP8_EINVAL;
}

// What both forms ask of their sizes; nullptr when they are valid.
const char* gdn_sizes(const gdn_dev_args* a) {
    if (!a) return "no arguments";
    if (a->dtype != QWEN_F32 && a->dtype != QWEN_BF16) return "dtype is neither QWEN_F32 nor QWEN_BF16";
    if (a->heads_k < 1 || a->heads_v < a->heads_k || a->heads_v % a->heads_k || a->heads_v > 65536)
        return "heads_v is not a multiple of heads_k (up to 65536)";
    if (a->dim_k < 4 || a->dim_k > GDN_MAX_DIM || a->dim_k % 4 || a->dim_v < 4 || a->dim_v > GDN_MAX_DIM ||
        a->dim_v % 4)
        return "dim_k and dim_v are multiples of 4 up to 256";
    if (a->rows < 0 || a->n_seq < 0 || a->n_slots < 0) return "rows, n_seq or n_slots below 0";
    // a launch has fewer than 2^32 threads: 576 for 16 value columns of a sequence and head, 256 for a chunk and head
    if ((size_t)a->n_seq * a->heads_v * ((a->dim_v + 15) / 16) > 1 << 22 ||
        ((size_t)a->rows / GDN_CHUNK + a->n_seq) * a->heads_v > 1 << 23)
        return "too many sequences, rows and heads for one call";
    return nullptr;
}

const char* gdn_pointers(const gdn_dev_args* a) {
    const size_t es = a->dtype == QWEN_BF16 ? 2 : 4;
    if (!a->state_out || !aligned(a->state_in, 16) || !aligned(a->state_out, 16))
        return "state_in and state_out have to be 16-byte aligned, state_out not NULL";
    if (!aligned(a->slots, 4) || !aligned(a->starts, 4)) return "slots and starts have to be 4-byte aligned";
    if (a->rows == 0) return nullptr;
    if (!a->out || !a->q || !a->k || !a->v || !a->alpha) return "out, q, k, v or alpha is NULL";
    if (!aligned(a->out, es) || !aligned(a->q, es) || !aligned(a->k, es) || !aligned(a->v, es) ||
        !aligned(a->alpha, 4) || !aligned(a->beta, 4))
        return "a pointer is not aligned to its elements";
    const int64_t keys = (int64_t)a->heads_k * a->dim_k, values = (int64_t)a->heads_v * a->dim_v;
    if (a->rows > 1 && (a->q_row < keys || a->k_row < keys || a->v_row < values || a->out_row < values ||
                        a->gate_row < a->heads_v))
        return "a row stride is below the row's length";
    return nullptr;
}

const char* loss_sizes(const lm_head_loss_args* a) {
    if (!a) return "no arguments";
    if (a->dtype != QWEN_F32 && a->dtype != QWEN_BF16) return "dtype is neither QWEN_F32 nor QWEN_BF16";
    if (a->rows < 0 || a->rows > 1 << 20) return "rows are 0 to 2^20";
    if (a->vocab < 1 || a->vocab > 1 << 28) return "vocab is 1 to 2^28";
    if (a->hidden < 1 || a->hidden > 65536) return "hidden is 1 to 65536";
    // a launch has fewer than 2^32 threads: 256 for a tile of 128 vocabulary rows and 32 or (above 64 rows) 128 rows
    if ((size_t)((a->vocab + LHL_TILE - 1) / LHL_TILE) * (size_t)((a->rows + 31) / 32) > 1 << 25)
        return "too many logits for one call";
    return nullptr;
}

const char* loss_pointers(const lm_head_loss_args* a, bool grad) {
    const size_t es = a->dtype == QWEN_BF16 ? 2 : 4;
    if (!a->table || !aligned(a->table, 2) || (a->vocab > 1 && a->table_row < a->hidden))
        return "table is NULL, not aligned to its elements, or its rows overlap";
    if (a->table_row > 1 << 22) return "table's rows are more than 2^22 elements apart";
    if (grad && (!aligned(a->grad_table, 2) ||
                 (a->grad_table && a->vocab > 1 && a->grad_table_row < a->hidden)))
        return "grad_table is not aligned to its elements, or its rows overlap";
    if (a->rows == 0) return nullptr;
    if (!a->h || !a->targets) return "h or targets is NULL";
    if (!aligned(a->h, es) || !aligned(a->targets, 4) || !aligned(a->loss, 4) || !aligned(a->lse, 4) ||
        (grad && (!aligned(a->grad_h, es) || !aligned(a->grad_loss, 4))))
        return "a pointer is not aligned to its elements";
    if (a->rows > 1 && (a->h_row < a->hidden || (grad && a->grad_h && a->grad_h_row < a->hidden)))
        return "a row stride is below the row's length";
    if (grad && (!a->lse || !a->grad_loss)) return "lse or grad_loss is NULL";
    return nullptr;
}

size_t loss_bytes(const char* who, const lm_head_loss_args* a, bool grad) {
    if (const char* why = loss_sizes(a)) {
        set_error("%s: %s", who, why);
        return 0;
    }
    return loss_work(*a, grad, grad && a->grad_h).total;
}

}  // namespace

extern "C" {

size_t gdn_dev_prompt_work_bytes(const gdn_dev_args* args) {
    if (const char* why = gdn_sizes(args)) {
        set_error("gdn_dev_prompt_work_bytes: %s", why);
        return 0;
    }
    return std::max<size_t>(gdn_work(*args).total, 256);
}

int gdn_dev_prompt(const gdn_dev_args* args, void* stream) {
    const char* who = "gdn_dev_prompt";
    if (const char* why = gdn_sizes(args)) return refuse(who, why);
    if (!args->starts && args->n_seq > 1) return refuse(who, "starts is NULL with more than one sequence");
    if (args->n_seq == 0) return BFP8_OK;
    if (const char* why = gdn_pointers(args)) return refuse(who, why);
    const GdnWork w = gdn_work(*args);
    if (!args->work || !aligned(args->work, 16) || args->work_bytes < w.total)
        return refuse(who, "work is smaller than gdn_dev_prompt_work_bytes() or not 16-byte aligned");
    if (init() != BFP8_OK) return BFP8_EHIP;
    HIP_OK(gdn_launch_prompt(*args, w, pick_stream(stream)));
    return BFP8_OK;
}

int gdn_dev_step(const gdn_dev_args* args, void* stream) {
    const char* who = "gdn_dev_step";
    if (const char* why = gdn_sizes(args)) return refuse(who, why);
    if (args->rows != args->n_seq) return refuse(who, "one row for each sequence");
    if (args->n_seq == 0) return BFP8_OK;
    if (const char* why = gdn_pointers(args)) return refuse(who, why);
    if (init() != BFP8_OK) return BFP8_EHIP;
    HIP_OK(gdn_launch_step(*args, pick_stream(stream)));
    return BFP8_OK;
}

size_t bf16_dev_lm_head_loss_work_bytes(const lm_head_loss_args* args) {
    return loss_bytes("bf16_dev_lm_head_loss_work_bytes", args, false);
}

size_t bf16_dev_lm_head_loss_grad_work_bytes(const lm_head_loss_args* args) {
    return loss_bytes("bf16_dev_lm_head_loss_grad_work_bytes", args, true);
}

int bf16_dev_lm_head_loss(const lm_head_loss_args* args, void* stream) {
    const char* who = "bf16_dev_lm_head_loss";
    if (const char* why = loss_sizes(args)) return refuse(who, why);
    if (const char* why = loss_pointers(args, false)) return refuse(who, why);
    if (args->rows == 0) return BFP8_OK;
    const LossWork w = loss_work(*args, false, false);
    if (!args->work || !aligned(args->work, 256) || args->work_bytes < w.total)
        return refuse(who, "work is smaller than bf16_dev_lm_head_loss_work_bytes() or not 256-byte aligned");
    if (init() != BFP8_OK) return BFP8_EHIP;
    HIP_OK(lhl_launch_loss(*args, w, pick_stream(stream)));
    return BFP8_OK;
}

int bf16_dev_lm_head_loss_grad(const lm_head_loss_args* args, void* stream) {
    const char* who = "bf16_dev_lm_head_loss_grad";
    if (const char* why = loss_sizes(args)) return refuse(who, why);
    if (const char* why = loss_pointers(args, true)) return refuse(who, why);
    if (!args->grad_table && (!args->grad_h || args->rows == 0)) return BFP8_OK;
    const LossWork w = loss_work(*args, true, args->grad_h != nullptr);
    if (!args->work || !aligned(args->work, 256) || args->work_bytes < w.total)
        return refuse(who, "work is smaller than bf16_dev_lm_head_loss_grad_work_bytes() or not 256-byte aligned");
    if (init() != BFP8_OK) return BFP8_EHIP;
    HIP_OK(lhl_launch_grad(*args, w, pick_stream(stream)));
    return BFP8_OK;
}

}  // extern "C"
