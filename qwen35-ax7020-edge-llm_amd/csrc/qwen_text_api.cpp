// qwen_text_api.cpp -- C ABI of the operators over a text's tokens
// (include/qwen_kernels.h): gated linear attention.  Arguments are
// checked here; the library's lock is not held while a kernel is launched, and no
// state of the library is used.
#include <hip/hip_runtime.h>

#include <climits>
#include <mutex>

#include "host_internal.h"
#include "linear_attention.h"

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
    if (a->dtype != GDN_F32 && a->dtype != GDN_BF16) return "dtype is neither GDN_F32 nor GDN_BF16";
    if (a->heads_k < 1 || a->heads_v < a->heads_k || a->heads_v % a->heads_k || a->heads_v > 65536)
        return "heads_v is not a multiple of heads_k (up to 65536)";
    if (a->dim_k < 4 || a->dim_k > GDN_MAX_DIM || a->dim_k % 4 || a->dim_v < 4 || a->dim_v > GDN_MAX_DIM ||
        a->dim_v % 4)
        return "dim_k and dim_v are multiples of 4 up to 256";
    if (a->rows < 0 || a->n_seq < 0 || a->n_slots < 0) return "rows, n_seq or n_slots below 0";
    if ((size_t)a->n_seq * a->heads_v * ((a->dim_v + 3) / 4) > INT_MAX ||
        ((size_t)a->rows / GDN_CHUNK + a->n_seq) * a->heads_v > INT_MAX)
        return "too many sequences and heads for one call";
    return nullptr;
}

const char* gdn_pointers(const gdn_dev_args* a) {
    const size_t es = a->dtype == GDN_BF16 ? 2 : 4;
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

}  // extern "C"
