// qwen_text_api.cpp -- C ABI of the operators over a text's tokens
// (include/qwen_kernels.h): gated linear attention, the head's loss, rotary positions,
// the paged cache and the attention over it.  Arguments are
// checked here; the library's lock is not held while a kernel is launched, and no
// state of the library is used.
#include <hip/hip_runtime.h>

#include <cmath>
#include <mutex>

#include "host_internal.h"
#include "linear_attention.h"
#include "lm_head_loss.h"
#include "paged_attention.h"

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

// ---- heads of rows and pages
bool in(int64_t x, int64_t lo, int64_t hi) { return lo <= x && x <= hi; }
constexpr int64_t kMaxStride = (int64_t)1 << 34;

// An axis of a tensor whose innermost elements are `dim` in a run.
struct Axis {
    int64_t size, stride;
};
// The axes' places are `dim` elements each that do not overlap, within 2^60 elements.
template <size_t N>
bool apart(Axis (&axes)[N], int64_t dim) {
    std::sort(axes, axes + N, [](const Axis& x, const Axis& y) { return x.stride < y.stride; });
    __int128 reach = dim;
    for (const Axis& x : axes) {
        if (x.size < 2) continue;
        if (x.stride < reach) return false;
        reach += (__int128)x.stride * (x.size - 1);
    }
    return reach <= (__int128)1 << 60;
}
bool heads_apart(int rows, int64_t row, int heads, int64_t head, int dim) {
    Axis axes[] = {{rows, row}, {heads, head}};
    return apart(axes, dim);
}

const char* rope_bad(const rope_dev_args* a) {
    if (!a) return "no arguments";
    if (a->dtype != QWEN_F32 && a->dtype != QWEN_BF16) return "dtype is neither QWEN_F32 nor QWEN_BF16";
    if (!in(a->dim, 2, 1024) || !in(a->rot, 2, a->dim) || a->rot % 2) return "dim is 2 to 1024, rot even and 2 to dim";
    if (a->rows < 0 || !in(a->heads, 1, 65536) || (int64_t)a->rows * a->heads > 1 << 28)
        return "heads are 1 to 65536, rows times heads up to 2^28";
    if (!std::isfinite(a->amplitude)) return "amplitude is not finite";
    if (a->rows == 0) return nullptr;
    const size_t es = a->dtype == QWEN_BF16 ? 2 : 4;
    if (!a->out || !a->x || !a->positions || !a->freqs) return "out, x, positions or freqs is NULL";
    if (!aligned(a->out, es) || !aligned(a->x, es) || !aligned(a->positions, 4) || !aligned(a->freqs, 8))
        return "a pointer is not aligned to its elements";
    if (!in(a->x_row, 0, kMaxStride) || !in(a->x_head, 0, kMaxStride) || !in(a->out_row, 0, kMaxStride) ||
        !in(a->out_head, 0, kMaxStride))
        return "a stride is below 0 or above 2^34";
    if (!heads_apart(a->rows, a->out_row, a->heads, a->out_head, a->dim)) return "out's rows or heads overlap";
    if (a->out == a->x && ((a->rows > 1 && a->x_row != a->out_row) || (a->heads > 1 && a->x_head != a->out_head)))
        return "out is x, with other strides";
    return nullptr;
}

// What kv_dev_append and attn_dev_paged ask of their cache and sequences.
template <class A>
const char* cache_sizes(const A* a) {
    if (!a) return "no arguments";
    if (a->dtype != QWEN_F32 && a->dtype != QWEN_BF16) return "dtype is neither QWEN_F32 nor QWEN_BF16";
    if (!in(a->dim, 8, 256) || a->dim % 8) return "dim is a multiple of 8 up to 256";
    if (!in(a->n_seq, 0, 1 << 20) || a->rows < 0) return "n_seq is 0 to 2^20, rows not below 0";
    if (!in(a->heads_k, 1, 65536) || (int64_t)a->rows * a->heads_k > 1 << 28)
        return "heads_k is 1 to 65536, rows times heads up to 2^28";
    return nullptr;
}
template <class A>
const char* cache_pointers(const A* a) {
    if (!in(a->page, 1, 65536) || a->pages < 0 || a->table_pages < 0 || (int64_t)a->page * a->table_pages > 1 << 30)
        return "page is 1 to 65536, page times table_pages up to 2^30, pages not below 0";
    if (a->n_seq && !a->starts && a->rows % a->n_seq) return "without starts the rows are a multiple of n_seq";
    if (a->n_seq == 0 || a->rows == 0) return nullptr;
    if (!a->cached || !aligned(a->cached, 4) || !aligned(a->starts, 4) || !aligned(a->tables, 4))
        return "cached is NULL, or cached, starts or tables not 4-byte aligned";
    if (a->n_seq > 1 && !in(a->table_row, a->table_pages, kMaxStride)) return "the tables' rows overlap";
    if (a->pages == 0 || a->table_pages == 0) return nullptr;
    const int64_t part = a->dtype == QWEN_BF16 ? 8 : 4;
    if (!a->tables || !a->key_cache || !a->value_cache) return "tables, key_cache or value_cache is NULL";
    if (!aligned(a->key_cache, 16) || !aligned(a->value_cache, 16) || a->cache_page % part || a->cache_token % part ||
        a->cache_head % part)
        return "the caches and their strides are 16-byte aligned";
    if (!in(a->cache_page, 0, (int64_t)1 << 40) || !in(a->cache_token, 0, kMaxStride) || !in(a->cache_head, 0, kMaxStride))
        return "a stride of the caches is below 0 or too large";
    Axis axes[] = {{a->pages, a->cache_page}, {a->page, a->cache_token}, {a->heads_k, a->cache_head}};
    if (!apart(axes, a->dim)) return "the caches' pages, tokens or heads overlap";
    return nullptr;
}

const char* append_bad(const kv_dev_append_args* a) {
    if (const char* why = cache_sizes(a)) return why;
    if (const char* why = cache_pointers(a)) return why;
    if (!in(a->rot, 0, a->dim) || a->rot % 2) return "rot is even, 0 to dim";
    if (!std::isfinite(a->amplitude)) return "amplitude is not finite";
    if (a->q && (a->heads_q < a->heads_k || a->heads_q % a->heads_k || a->heads_q > 65536 ||
                 (int64_t)a->rows * a->heads_q > 1 << 28))
        return "heads_q is a multiple of heads_k, rows times heads up to 2^28";
    if (a->q && a->rot == 0) return "q without a rotation";
    if (a->n_seq == 0 || a->rows == 0) return nullptr;
    const size_t es = a->dtype == QWEN_BF16 ? 2 : 4;
    if (!a->k || !a->v || (a->q && !a->q_out) || (a->rot && !a->freqs)) return "k, v, q_out or freqs is NULL";
    if (!aligned(a->k, es) || !aligned(a->v, es) || !aligned(a->positions, 4) || !aligned(a->freqs, 8) ||
        (a->q && (!aligned(a->q, es) || !aligned(a->q_out, es))))
        return "a pointer is not aligned to its elements";
    for (const int64_t x : {a->k_row, a->k_head, a->v_row, a->v_head})
        if (!in(x, 0, kMaxStride)) return "a stride is below 0 or above 2^34";
    if (!a->q) return nullptr;
    for (const int64_t x : {a->q_row, a->q_head, a->q_out_row, a->q_out_head})
        if (!in(x, 0, kMaxStride)) return "a stride is below 0 or above 2^34";
    if (!heads_apart(a->rows, a->q_out_row, a->heads_q, a->q_out_head, a->dim)) return "q_out's rows or heads overlap";
    if (a->q_out == a->q &&
        ((a->rows > 1 && a->q_row != a->q_out_row) || (a->heads_q > 1 && a->q_head != a->q_out_head)))
        return "q_out is q, with other strides";
    return nullptr;
}

const char* paged_sizes(const attn_dev_args* a) {
    if (const char* why = cache_sizes(a)) return why;
    if (a->heads_q < a->heads_k || a->heads_q % a->heads_k || (int64_t)a->rows * a->heads_q > 1 << 28 ||
        a->heads_q > 1 << 20)
        return "heads_q is a multiple of heads_k up to 2^20, rows times heads up to 2^28";
    return nullptr;
}
const char* paged_bad(const attn_dev_args* a) {
    if (const char* why = cache_pointers(a)) return why;
    if (!std::isnormal(a->scale) || a->scale < 0 || a->scale > 1e38f) return "scale is a normal number of up to 1e38, above 0";
    if (a->mask && (!in(a->mask_words, 0, 1 << 16) || !aligned(a->mask, 4)))
        return "mask_words are 0 to 2^16, mask 4-byte aligned";
    if (a->n_seq == 0 || a->rows == 0) return nullptr;
    if (!attn_units_fit(*a)) return "the caches span more places than 32 bits number";
    const size_t es = a->dtype == QWEN_BF16 ? 2 : 4;
    if (!a->out || !a->q || !aligned(a->out, es) || !aligned(a->q, es))
        return "out or q is NULL or not aligned to its elements";
    if (a->out == a->q) return "out is q";
    for (const int64_t x : {a->q_row, a->q_head, a->out_row, a->out_head})
        if (!in(x, 0, kMaxStride)) return "a stride is below 0 or above 2^34";
    if (!heads_apart(a->rows, a->out_row, a->heads_q, a->out_head, a->dim)) return "out's rows or heads overlap";
    return nullptr;
}

const char* tree_bad(const attn_dev_tree_args* a) {
    if (!a) return "no arguments";
    if (!in(a->n_seq, 0, 1 << 20) || a->rows < 0 || a->words < 0 || (int64_t)a->rows * a->words > 1 << 28)
        return "n_seq is 0 to 2^20, rows times words up to 2^28";
    if (a->n_seq && !a->starts && a->rows % a->n_seq) return "without starts the rows are a multiple of n_seq";
    if (a->n_seq == 0 || a->rows == 0) return nullptr;
    if (a->words < 1) return "no words for the rows' bits";
    if (!a->mask || !a->parents || !a->cached) return "mask, parents or cached is NULL";
    if (!aligned(a->mask, 4) || !aligned(a->positions, 4) || !aligned(a->parents, 4) || !aligned(a->cached, 4) ||
        !aligned(a->starts, 4))
        return "a pointer is not 4-byte aligned";
    return nullptr;
}

int rope(const char* who, const rope_dev_args* a, bool back, void* stream) {
    if (const char* why = rope_bad(a)) return refuse(who, why);
    if (a->rows == 0) return BFP8_OK;
    if (init() != BFP8_OK) return BFP8_EHIP;
    HIP_OK(rope_launch(*a, back, pick_stream(stream)));
    return BFP8_OK;
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

int rope_dev_apply(const rope_dev_args* args, void* stream) { return rope("rope_dev_apply", args, false, stream); }

int rope_dev_grad(const rope_dev_args* args, void* stream) { return rope("rope_dev_grad", args, true, stream); }

int kv_dev_append(const kv_dev_append_args* args, void* stream) {
    if (const char* why = append_bad(args)) return refuse("kv_dev_append", why);
    if (args->n_seq == 0 || args->rows == 0) return BFP8_OK;
    if (init() != BFP8_OK) return BFP8_EHIP;
    HIP_OK(kv_launch_append(*args, pick_stream(stream)));
    return BFP8_OK;
}

size_t attn_dev_paged_work_bytes(const attn_dev_args* args) {
    if (const char* why = paged_sizes(args)) {
        set_error("attn_dev_paged_work_bytes: %s", why);
        return 0;
    }
    return attn_plan(*args).total;
}

int attn_dev_paged(const attn_dev_args* args, void* stream) {
    const char* who = "attn_dev_paged";
    if (const char* why = paged_sizes(args)) return refuse(who, why);
    if (const char* why = paged_bad(args)) return refuse(who, why);
    if (args->n_seq == 0 || args->rows == 0) return BFP8_OK;
    const AttnPlan p = attn_plan(*args);
    if (!args->work || !aligned(args->work, 256) || args->work_bytes < p.total)
        return refuse(who, "work is smaller than attn_dev_paged_work_bytes() or not 256-byte aligned");
    if (init() != BFP8_OK) return BFP8_EHIP;
    HIP_OK(attn_launch_paged(*args, p, pick_stream(stream)));
    return BFP8_OK;
}

int attn_dev_tree(const attn_dev_tree_args* args, void* stream) {
    if (const char* why = tree_bad(args)) return refuse("attn_dev_tree", why);
    if (args->n_seq == 0 || args->rows == 0) return BFP8_OK;
    if (init() != BFP8_OK) return BFP8_EHIP;
    HIP_OK(attn_launch_tree(*args, pick_stream(stream)));
    return BFP8_OK;
}

}  // extern "C"
