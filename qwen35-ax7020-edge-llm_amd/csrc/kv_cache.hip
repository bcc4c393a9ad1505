// kv_cache.hip -- positions rotated into queries and keys, keys and values on their
// way to a paged cache, and the masks of drafted tokens (rope_dev_apply, rope_dev_grad,
// kv_dev_append, attn_dev_tree).
//
//   (x, y) -> A (x cos t - y sin t, x sin t + y cos t),  t = p f_i
//
// A workgroup has a few rows: their angles go to LDS once for all heads, then every thread
// takes 16-byte pieces of the rows' heads.  What bounds it: few rows, the latency of a launch and
// of the loads that depend on one another (sequence, length, page); many, memory.
#include <algorithm>
#include <type_traits>

#include "bf16_terms.h"
#include "kv_cache.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxRows = 4;       // of a workgroup
constexpr int kMaxPairs = 512;    // of a head

// Sine and cosine of p f: the angle is brought into one turn in double, where a float32 product would have lost the
// turn's fraction (2^20 positions of 1 radian: 2^-4 of a radian), and -- as half turns of up to 1 -- is rounded to
// float32 only then, 2^-24 of an angle of up to pi.
__device__ __forceinline__ float2 angle_of(int p, double f, float amplitude, bool back) {
    const double turns = (double)p * f * 0.15915494309189533577;
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    return {amplitude * c, back ? -amplitude * s : amplitude * s};
}

template <class T, int N>
struct Piece {
    T x[N];
};

// How a head is taken apart: first `turned` units of pairs, then the units that pass unchanged.
// VEC: 16 bytes a unit (from both halves of the rotated part in the half layout), else a pair or an element.
template <class T, bool VEC, bool INTER>
struct Head {
    static constexpr int N = VEC ? 16 / sizeof(T) : 1;      // elements of a unit that passes
    static constexpr int P = !VEC ? 1 : INTER ? N / 2 : N;  // pairs of a unit that is rotated
    using V = Piece<T, N>;
    using V2 = Piece<T, VEC && INTER ? N : 2 * P>;

    static __host__ __device__ int turned(int rot) { return rot / 2 / P; }
    static __host__ __device__ int passed(int dim, int rot) { return (dim - rot) / N; }

    static __device__ __forceinline__ void turn(const T* x, T* y, int u, int rot, const float2* cs) {
        float a[P], b[P];
        if constexpr (INTER) {
            V2 v;
            load(v, x + u * 2 * P);
#pragma unroll
            for (int j = 0; j < P; ++j) a[j] = to_float(v.x[2 * j]), b[j] = to_float(v.x[2 * j + 1]);
        } else {
            V v, w;
            load(v, x + u * P);
            load(w, x + rot / 2 + u * P);
#pragma unroll
            for (int j = 0; j < P; ++j) a[j] = to_float(v.x[j]), b[j] = to_float(w.x[j]);
        }
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const float2 t = cs[u * P + j];
            const float xa = a[j], xb = b[j];
            a[j] = __builtin_fmaf(xa, t.x, -(xb * t.y));
            b[j] = __builtin_fmaf(xa, t.y, xb * t.x);
        }
        if constexpr (INTER) {
            V2 v;
#pragma unroll
            for (int j = 0; j < P; ++j) v.x[2 * j] = from_float<T>(a[j]), v.x[2 * j + 1] = from_float<T>(b[j]);
            store(y + u * 2 * P, v);
        } else {
            V v, w;
#pragma unroll
            for (int j = 0; j < P; ++j) v.x[j] = from_float<T>(a[j]), w.x[j] = from_float<T>(b[j]);
            store(y + u * P, v);
            store(y + rot / 2 + u * P, w);
        }
    }
    static __device__ __forceinline__ void pass(const T* x, T* y, int u, int rot) {
        V v;
        load(v, x + rot + u * N);
        store(y + rot + u * N, v);
    }

    template <class X>
    static __device__ __forceinline__ void load(X& v, const T* p) {
        if constexpr (sizeof(X) == 16)
            v = __builtin_bit_cast(X, *reinterpret_cast<const u32x4*>(p));
        else
#pragma unroll
            for (size_t j = 0; j < sizeof(X) / sizeof(T); ++j) v.x[j] = p[j];
    }
    template <class X>
    static __device__ __forceinline__ void store(T* p, const X& v) {
        if constexpr (sizeof(X) == 16)
            *reinterpret_cast<u32x4*>(p) = __builtin_bit_cast(u32x4, v);
        else
#pragma unroll
            for (size_t j = 0; j < sizeof(X) / sizeof(T); ++j) p[j] = v.x[j];
    }
};

// ---- rotation alone -------------------------------------------------------------------
// 16 bytes a thread and piece, both of a pair's elements by the same thread (so that out may be x): 16,384 rows of 10
// heads of 256 bf16 elements, 168 MB, in 36 us among other work, 4.7 TB/s (27.8 us again on the same rows, which the
// memory-side cache holds in part); 5,003 of 12 heads of 96 float32 ones 8.7; one row 3.8, a launch's latency.
template <class T, bool VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void rope_kernel(rope_dev_args a, int each, int back, int units, Divisor by_units,
                                                        Divisor by_heads) {
    using H = Head<T, VEC, INTER>;
    __shared__ float2 cs[kMaxRows * kMaxPairs];
    const int half = a.rot / 2, turned = H::turned(a.rot);
    for (int64_t r0 = (int64_t)blockIdx.x * each; r0 < a.rows; r0 += (int64_t)gridDim.x * each) {
        const int n = (int)min((int64_t)each, a.rows - r0);
        for (int i = threadIdx.x; i < n * half; i += kThreads)
            cs[i] = angle_of(a.positions[r0 + i / half], a.freqs[i % half], a.amplitude, back);
        __syncthreads();
        for (int i = threadIdx.x; i < n * a.heads * units; i += kThreads) {
            const int head = divide(i, by_units), u = i - head * units, r = divide(head, by_heads), h = head - r * a.heads;
            const T* x = static_cast<const T*>(a.x) + (r0 + r) * a.x_row + h * a.x_head;
            T* y = static_cast<T*>(a.out) + (r0 + r) * a.out_row + h * a.out_head;
            if (u < turned)
                H::turn(x, y, u, a.rot, cs + r * half);
            else
                H::pass(x, y, u - turned, a.rot);
        }
        __syncthreads();
    }
}

// ---- to the cache -----------------------------------------------------------------------
// A row's place: its sequence is not skipped; where in the cache (elements), -1 nowhere.
struct Place {
    int there;
    int position;
    int64_t at;
};

// How a row's 16-byte pieces (or elements) follow one another: the keys' heads, the values', the queries'.
struct Units {
    int k, v, q;              // of a head
    int ks, vs, all;          // of the keys' heads, the values', all
    Divisor by_k, by_v, by_q, by_all;
};

// The sequence that holds row r, or -1, by a wavefront: 64 of the starts at a time (a binary search would wait for
// five loads one after the other for 24 sequences).
__device__ __forceinline__ int owner_by_wave(const int32_t* starts, int rows, int n_seq, int r) {
    if (!starts) return r / (rows / n_seq);
    const int lane = threadIdx.x & 63;
    int lo = 0, n = n_seq;  // starts[lo] <= r < starts[lo + n], as far as it is known
    while (n > 1) {
        const int step = (n + 63) / 64, at = lo + lane * step;
        const uint64_t upto = __ballot(lane * step < n && (lane == 0 || starts[at] <= r));
        lo += (63 - __builtin_clzll(upto)) * step;
        n = min(step, n_seq - lo);
    }
    const Span p = span_of(starts, rows, n_seq, lo);
    return r >= p.first && r < p.first + p.count ? lo : -1;
}

// A wavefront a row finds where it goes, then all threads take the rows' pieces: keys, values and queries in one
// launch.  9,001 tokens of 24 sequences, 8 and 2 heads of 256 bf16 elements, 111 MB: 34.8 us among other work, 3.2 TB/s
// (a row's bytes wait for its place, three loads one after the other; 25.6 us again on the same tokens, from the
// memory-side cache in part); one token 5.1 us.
template <class T, bool VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(kv_dev_append_args a, Divisor page, int each, Units n, int copy_v) {
    using H = Head<T, VEC, INTER>;
    using C = Head<T, true, false>;  // values are copied 16 bytes at a time where they are aligned
    __shared__ float2 cs[kMaxRows * kMaxPairs / 4];
    __shared__ Place places[kMaxRows];
    const int half = a.rot / 2, turned = H::turned(a.rot), wave = threadIdx.x >> 6;
    for (int64_t r0 = (int64_t)blockIdx.x * each; r0 < a.rows; r0 += (int64_t)gridDim.x * each) {
        const int rows = (int)min((int64_t)each, a.rows - r0);
        if (wave < rows) {
            const int r = (int)r0 + wave, s = owner_by_wave(a.starts, a.rows, a.n_seq, r);
            Place p{0, 0, -1};
            if (s >= 0) {
                const int held = a.cached[s];
                if (held >= 0) {
                    const int64_t place = (int64_t)held + r - span_of(a.starts, a.rows, a.n_seq, s).first;
                    p.there = 1;
                    p.position = a.positions ? a.positions[r] : (int)min(place, (int64_t)INT32_MAX);
                    if (place < (a.pages ? (int64_t)a.table_pages * a.page : 0)) {  // (without pages tables may be NULL)
                        const uint32_t j = divide((uint32_t)place, page);
                        const int id = a.tables[s * a.table_row + j];
                        if ((unsigned)id < (unsigned)a.pages)
                            p.at = id * a.cache_page + ((uint32_t)place - j * a.page) * a.cache_token;
                    }
                }
            }
            places[wave] = p;
        }
        __syncthreads();
        if (half) {
            for (int i = threadIdx.x; i < rows * half; i += kThreads)
                cs[i] = angle_of(places[i / half].position, a.freqs[i % half], a.amplitude, false);
            __syncthreads();
        }
        for (int i = threadIdx.x; i < rows * n.all; i += kThreads) {
            const int r = divide(i, n.by_all);
            int u = i - r * n.all;
            const Place p = places[r];
            const int64_t row = r0 + r;
            const float2* t = cs + r * half;
            const T* x;
            T* y;
            if (u < n.ks) {
                if (p.at < 0) continue;
                const int h = divide(u, n.by_k);
                u -= h * n.k;
                x = static_cast<const T*>(a.k) + row * a.k_row + h * a.k_head;
                y = static_cast<T*>(a.key_cache) + p.at + h * a.cache_head;
            } else if (u < n.ks + n.vs) {
                if (p.at < 0) continue;
                u -= n.ks;
                const int h = divide(u, n.by_v);
                u -= h * n.v;
                x = static_cast<const T*>(a.v) + row * a.v_row + h * a.v_head;
                y = static_cast<T*>(a.value_cache) + p.at + h * a.cache_head;
                if (copy_v)
                    C::pass(x, y, u, 0);
                else
                    y[u] = x[u];
                continue;
            } else {
                if (!p.there) continue;
                u -= n.ks + n.vs;
                const int h = divide(u, n.by_q);
                u -= h * n.q;
                x = static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head;
                y = static_cast<T*>(a.q_out) + row * a.q_out_row + h * a.q_out_head;
            }
            if (u < turned)
                H::turn(x, y, u, a.rot, t);
            else
                H::pass(x, y, u - turned, a.rot);
        }
        __syncthreads();
    }
}

// ---- drafted tokens' trees -----------------------------------------------------------------
// A workgroup a sequence.  A draft of up to kTreeWalk tokens: a thread a word of a row's mask, which walks up the row's
// ancestors, whose places only fall, until they are below its word; word 0's counts them all.  Of more tokens a walk
// could be as long as the text: a thread has a word of every row, one row after the other, as its parent's word and its
// own bit (and word 0's thread the positions, as the parent's and one). Latency bounds both: 26 tokens 3.4 us, 48 trees
// of 1,500 4.8. (One sequence, a chain of 64 | 256 | 1,000 | 20,000 tokens: walked 11 | 109 us, row after row 50 | 178
// | 3,437 of 256 and more.)
constexpr int kTreeWalk = 128;
__global__ __launch_bounds__(kThreads) void attn_tree_kernel(attn_dev_tree_args a) {
    __shared__ int32_t up[kThreads];
    const int s = blockIdx.x, t0 = blockIdx.y * kThreads + threadIdx.x, threads = gridDim.y * kThreads;
    const Span p = span_of(a.starts, a.rows, a.n_seq, s);
    const int held = a.cached[s];
    const int32_t* parents = a.parents + p.first;
    int32_t* mask = a.mask + (int64_t)p.first * a.words;
    int32_t* positions = a.positions ? a.positions + p.first : nullptr;
    if (p.count <= kTreeWalk) {
        if ((int)threadIdx.x < p.count) up[threadIdx.x] = parents[threadIdx.x];  // (fewer than the threads)
        __syncthreads();
        const int64_t items = (int64_t)p.count * a.words;
        for (int64_t i = t0; i < items; i += threads) {
            const int r = (int)(i / a.words), w = (int)(i - (int64_t)r * a.words);
            uint32_t bits = 0;
            int depth = 0;
            if (held >= 0)
                for (int j = r; j >> 5 >= w;) {
                    if (j >> 5 == w) bits |= 1u << (j & 31);
                    if (up[j] < 0 || up[j] >= j) break;
                    ++depth;
                    j = up[j];
                }
            mask[i] = (int32_t)bits;
            if (w == 0 && positions) positions[r] = held < 0 ? 0 : (int)min((int64_t)held + depth, (int64_t)INT32_MAX);
        }
        return;
    }
    for (int w0 = blockIdx.y * kThreads; w0 < a.words; w0 += threads) {
        const int w = w0 + threadIdx.x;
        const bool mine = w < a.words, first = w == 0 && positions;
        uint32_t last = 0;  // of the row before
        int last_position = 0;
        for (int r0 = 0; r0 < p.count; r0 += kThreads) {
            const int n = min(kThreads, p.count - r0);
            __syncthreads();
            if ((int)threadIdx.x < n) up[threadIdx.x] = parents[r0 + threadIdx.x];
            __syncthreads();
            if (!mine) continue;
            for (int i = 0; i < n; ++i) {
                const int r = r0 + i, j = up[i];
                const bool has = held >= 0 && j >= 0 && j < r;
                uint32_t bits = 0;
                int position = max(held, 0);
                if (has) {
                    if (j >> 5 >= w) bits = j == r - 1 ? last : (uint32_t)mask[(int64_t)j * a.words + w];
                    if (first) position = min(j == r - 1 ? last_position : positions[j], INT32_MAX - 1) + 1;
                }
                if (held >= 0 && r >> 5 == w) bits |= 1u << (r & 31);
                mask[(int64_t)r * a.words + w] = (int32_t)bits;
                if (first) positions[r] = position;
                last = bits;
                last_position = position;
            }
        }
    }
}

bool whole(const void* p, int64_t row, int64_t head, size_t es) {
    return ((uintptr_t)p | (uint64_t)row * es | (uint64_t)head * es) % 16 == 0;
}
// The rotated part falls into 16-byte pieces of whole pairs, what passes into 16-byte pieces.
bool pieces(int dim, int rot, bool inter, size_t es) {
    const int n = (int)(16 / es);
    return rot % (inter ? n : 2 * n) == 0 && dim % n == 0;
}

// Rows of a workgroup: one where they do not fill the device, else four for one set of angles and one look for the
// places (one | four, us: 512 rows rotated 3.8 | 5.4, 2,048 6.0 | 6.7, 4,096 9.9 | 9.8; 1,024 tokens of 24 sequences
// appended 6.5 | 8.6, 2,048 10.6 | 10.1, 4,096 18.7 | 14.6, 9,001 35.7 | 25.6).
int rows_each(int rows) { return rows < 2048 ? 1 : kMaxRows; }

template <class T, bool VEC, bool INTER>
void launch_rope(const rope_dev_args& a, bool back, hipStream_t s) {
    using H = Head<T, VEC, INTER>;
    const int each = rows_each(a.rows), grid = std::min((a.rows + each - 1) / each, 1 << 20);
    const int units = H::turned(a.rot) + (a.out != a.x ? H::passed(a.dim, a.rot) : 0);
    rope_kernel<T, VEC, INTER>
        <<<dim3((unsigned)grid), kThreads, 0, s>>>(a, each, back, units, divisor(units), divisor(a.heads));
}

template <class T, bool VEC, bool INTER>
void launch_append(const kv_dev_append_args& a, hipStream_t s) {
    using H = Head<T, VEC, INTER>;
    const int each = rows_each(a.rows), grid = std::min((a.rows + each - 1) / each, 1 << 20);
    const int copy_v = whole(a.v, a.v_row, a.v_head, sizeof(T));
    Units n{};
    n.k = H::turned(a.rot) + H::passed(a.dim, a.rot);
    n.v = copy_v ? a.dim * (int)sizeof(T) / 16 : a.dim;
    n.q = H::turned(a.rot) + (a.q_out != a.q ? H::passed(a.dim, a.rot) : 0);
    n.ks = a.heads_k * n.k;
    n.vs = a.heads_k * n.v;
    n.all = n.ks + n.vs + (a.q ? a.heads_q * n.q : 0);
    n.by_k = divisor(n.k);
    n.by_v = divisor(n.v);
    n.by_q = divisor(std::max(n.q, 1));
    n.by_all = divisor(n.all);
    kv_append_kernel<T, VEC, INTER><<<dim3((unsigned)grid), kThreads, 0, s>>>(a, divisor(a.page), each, n, copy_v);
}

// f(T{}, VEC, INTER) for a call's type, alignment and layout
template <class F>
void choose(int dtype, bool vec, bool inter, F&& f) {
    using Yes = std::true_type;
    using No = std::false_type;
    auto of = [&](auto t) { vec ? (inter ? f(t, Yes{}, Yes{}) : f(t, Yes{}, No{})) : (inter ? f(t, No{}, Yes{}) : f(t, No{}, No{})); };
    if (dtype == QWEN_BF16)
        of(uint16_t{});
    else
        of(float{});
}

}  // namespace

hipError_t rope_launch(const rope_dev_args& a, bool back, hipStream_t s) {
    const size_t es = a.dtype == QWEN_BF16 ? 2 : 4;
    const bool vec = pieces(a.dim, a.rot, a.interleaved, es) && whole(a.x, a.x_row, a.x_head, es) &&
                     whole(a.out, a.out_row, a.out_head, es);
    choose(a.dtype, vec, a.interleaved, [&](auto t, auto v, auto i) {
        launch_rope<decltype(t), decltype(v)::value, decltype(i)::value>(a, back, s);
    });
    return hipGetLastError();
}

hipError_t kv_launch_append(const kv_dev_append_args& a, hipStream_t s) {
    const size_t es = a.dtype == QWEN_BF16 ? 2 : 4;
    const bool vec = pieces(a.dim, a.rot, a.interleaved, es) && whole(a.k, a.k_row, a.k_head, es) &&
                     (!a.q || (whole(a.q, a.q_row, a.q_head, es) && whole(a.q_out, a.q_out_row, a.q_out_head, es)));
    choose(a.dtype, vec, a.interleaved, [&](auto t, auto v, auto i) {
        launch_append<decltype(t), decltype(v)::value, decltype(i)::value>(a, s);
    });
    return hipGetLastError();
}

hipError_t attn_launch_tree(const attn_dev_tree_args& a, hipStream_t s) {
    // (more workgroups a sequence where a row's words are more than the threads, and the sequences do not fill the
    // device)
    const int more = a.n_seq <= 256 ? std::min((a.words + kThreads - 1) / kThreads, 64) : 1;
    attn_tree_kernel<<<dim3((unsigned)a.n_seq, (unsigned)more), kThreads, 0, s>>>(a);
    return hipGetLastError();
}
