// lm_head_loss.hip -- the score of a text under the bf16 tied-embedding head and
// its gradient (bf16_dev_lm_head_loss, bf16_dev_lm_head_loss_grad).
//
//   z_nv = w_v . h_n;  lse_n = log sum_v exp z_nv;  loss_n = lse_n - z_n,t_n
//   D_nv = g_n (exp(z_nv - lse_n) - [v = t_n]);  grad_h = D W;  grad_w = D^T h
//
// With bf16 states D is an operand of one bf16 term, and holds g_n over the call's largest |g|, which both gradients
// are multiplied by in float32.  Under a mean loss, whose weights are all the same, a target's entry is then -1 + p,
// which bf16 holds almost exactly where p is small; g (-1 + p) would be rounded the same way in every row, by up to
// 2^-8 that no sum takes out.  What the rounding leaves out at a target, the largest of its row's D, goes to grad_h with the
// target's table row in float32.
//
// lhl_prepare_kernel gathers the rows that count (a text's own prompt often does
// not), as bf16 terms.  The rest are tiled products on the matrix cores:
//   lhl_logits_kernel    W h^T; its epilogue leaves a tile's maximum and sum of
//                        exponentials for each row, or D for a piece of the vocabulary
//   lhl_grad_h_kernel    W^T D^T, split over the vocabulary, float32 sums
//   lhl_grad_table_kernel  h^T D
// and lhl_loss_kernel / lhl_finish_kernel join the parts.  Every sum has one fixed
// order: results repeat bit for bit.
//
// What bounds it.  Few rows: the table's bytes (one row of 65536 x 1024: the logits 25 us,
// the table's at the rate of a copy 26).  Many: the matrix cores (4096 rows: the logits and their
// statistics 490 us, 1.12 PFLOP/s; a library product of that shape alone 533).  The
// gradient computes the logits again, in pieces of the vocabulary: 4096 rows, 3277 of
// them counted, for each of four pieces 137 us of logits and D, 140 of grad_h, 110 of grad_table.
#include "bf16_terms.h"
#include "lm_head_loss.h"

namespace {

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void global_void;
using s16x4 = __attribute__((ext_vector_type(4))) short;

// Exponentials in base 2: exp z = 2^(z log2 e).
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }  // below 2^-126: 0

// ---- tiles ----------------------------------------------------------------------------
// An operand in memory: rows x cols bf16 values, `term` elements from one term to the
// next.  Its tiles are B (rows or columns of the result) x 64 (terms of the sum).
struct Operand {
    const uint16_t* p;
    int64_t pitch, term;
    int rows, cols;
};

// Brings an operand's tiles to LDS.  TR false: the sum runs along an operand's rows
// (rows of the tile are rows in memory); LDS holds row r's eight 16-byte parts at
// positions part ^ (r & 7), so that a column of 16 rows' parts spreads over the banks.
// TR true: the sum runs down its columns; LDS holds 64 rows of B values, row k's
// 32-byte blocks at positions block ^ swizzle(k), for ds_read_tr16_b64, whose 16 lanes
// read 4 rows x 32 bytes and get a column of 4 each.  Each wave instruction copies 1 KiB
// to consecutive LDS bytes: the permutations are in the global addresses.
// VEC false: rows without 16-byte alignment, through registers.
template <int B, bool TR, int N, int WAVES, bool VEC>
struct Loader {
    static constexpr int I = N * B / 8 / WAVES;
    static_assert(N * B % (8 * WAVES) == 0, "every wavefront copies the same share");
    static constexpr int kBytes = N * B * 128;
    const char* base[I];  // the same for all lanes, moved on step by step
    uint32_t off[I];      // a lane's own part of an address
    int kc, k_end;        // first element along the sum of this lane's part of a step; the sum's end
    int col_left[I];      // VEC false, TR: columns from the part's first on
    int64_t step;         // bytes from one step to the next
    u32x4 held[VEC ? 1 : I];  // VEC false: a step on its way to LDS

    static __device__ int swizzle(int k) { return (k & 3) | (k >> 1 & 4); }
    static __device__ int k_row(int q, int lane) { return 512 / B * (q % (B / 8)) + lane / (B / 8); }

    // m0: first row or column of the result; the sum from element k0
    __device__ void init(const Operand& op, int m0, int64_t k0, int wave, int lane) {
        k_end = TR ? op.rows : op.cols;
        step = TR ? (int64_t)LHL_STEP * op.pitch * 2 : LHL_STEP * 2;
        kc = 8 * ((lane & 7) ^ (lane >> 3));
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const int q = wave * I + i, term = q / (B / 8);
            base[i] = reinterpret_cast<const char*>(op.p + term * op.term + (TR ? k0 * op.pitch : m0 * op.pitch + k0));
            if constexpr (TR) {
                const int k = k_row(q, lane), pos = lane % (B / 8);
                int col = m0 + 16 * ((pos >> 1) ^ swizzle(k)) + 8 * (pos & 1);
                if (VEC) col = min(col, op.cols - 8);  // past the last column: values that nothing reads
                col_left[i] = op.cols - col;
                off[i] = (uint32_t)(k * op.pitch + col) * 2;
            } else {
                const int row = min(8 * (q % (B / 8)) + lane / 8, op.rows - 1 - m0);  // as above
                off[i] = (uint32_t)(row * op.pitch + kc) * 2;
            }
        }
    }

    // Starts the copy of the step whose sum begins at k (from 0) and moves on.  VEC false: only as far as
    // the registers, from which put() takes it to LDS.
    __device__ void issue(char* lds, int k, const char* zeros, int wave, int lane) {
        if constexpr (!VEC) {
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const int q = wave * I + i, mine = k + (TR ? k_row(q, lane) : kc);
                const int n = TR ? (mine < k_end ? col_left[i] : 0) : k_end - mine;
                if (n >= 8) {
                    __builtin_memcpy(&held[i], base[i] + off[i], 16);
                } else {
                    held[i] = u32x4{0, 0, 0, 0};
                    const uint16_t* p = reinterpret_cast<const uint16_t*>(base[i] + off[i]);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < n) held[i][j / 2] |= (uint32_t)p[j] << (j % 2 * 16);
                }
            }
        } else if (k + LHL_STEP <= k_end) {
#pragma unroll
            for (int i = 0; i < I; ++i)
                __builtin_amdgcn_global_load_lds((global_void*)(base[i] + off[i]),
                                                 (lds_void*)(lds + (wave * I + i) * 1024), 16, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const int q = wave * I + i;
                const char* src = k + (TR ? k_row(q, lane) : kc) < k_end ? base[i] + off[i] : zeros;
                __builtin_amdgcn_global_load_lds((global_void*)src, (lds_void*)(lds + q * 1024), 16, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < I; ++i) base[i] += step;
    }
    __device__ void put(char* lds, int wave, int lane) const {
        if constexpr (!VEC)
#pragma unroll
            for (int i = 0; i < I; ++i)
                *reinterpret_cast<u32x4*>(lds + (wave * I + i) * 1024 + lane * 16) = held[i];
    }
};

// A wavefront's MFMA operands from a tile: T 16-wide parts from column (row) first on.
template <int B, bool TR, int N, int T>
struct Reader {
    int at[TR ? T : 2];
    __device__ void init(int first, int lane) {
        const int c = lane & 15, g = lane >> 4;
        if constexpr (TR) {
            const int f = (c >> 2) | (g & 1) << 2;
#pragma unroll
            for (int t = 0; t < T; ++t)
                at[t] = (8 * g + (c >> 2)) * 2 * B + ((first / 16 + t) ^ f) * 32 + (c & 3) * 8;
        } else {
#pragma unroll
            for (int s = 0; s < 2; ++s) at[s] = (first + c) * 128 + ((4 * s + g) ^ (c & 7)) * 16;
        }
    }
    // part t, half-step s (32 terms of the sum)
    __device__ void read(const char* lds, int t, int s, u32x4 (&x)[N]) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const char* p = lds + n * B * 128;
            if constexpr (TR) {
                using lds_s16x4 = __attribute__((address_space(3))) s16x4;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + at[t] + 32 * s * 2 * B));
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + at[t] + (32 * s + 4) * 2 * B));
                const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
                x[n] = u32x4{a[0], a[1], b[0], b[1]};
            } else {
                x[n] = *reinterpret_cast<const u32x4*>(p + at[s] + t * 2048);
            }
        }
    }
};

// BM x BN of a product by WM x WN wavefronts: acc[i][j] holds rows 16 i + 4 (lane / 16) .. + 3
// and column 16 j + lane % 16 of the wavefront's part.  NA, NB: the operands' terms, the pairs
// with ta + tb < MOST taken.  STAGES steps' tiles in LDS, copied that far ahead.  A step is two halves: the
// second half's operands are read before the first is multiplied, and the next step's first half's before
// the second, with the step's one barrier between, so that the matrix cores work through both waits.
template <int BM_, int BN_, int WM_, int WN_, bool TRA, bool TRB, int NA, int NB, int MOST, bool VEC, int STAGES>
struct Product {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
    static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
    using LA = Loader<BM, TRA, NA, kWaves, VEC>;
    using LB = Loader<BN, TRB, NB, kWaves, true>;
    static constexpr int kStage = LA::kBytes + LB::kBytes;
    static constexpr int kLds = STAGES * kStage;

    // This wavefront's share of the oldest step is in LDS, but for kSteps newer ones; its own reads are done.
    template <int kSteps>
    static __device__ void wait() {
        constexpr int kLeft = VEC ? kSteps * (LA::I + LB::I) : 0;
        static_assert(kLeft < 64, "vmcnt has six bits");
        __builtin_amdgcn_s_waitcnt(0x0070 | (kLeft & 15) | (kLeft >> 4) << 14);  // vmcnt(kLeft) lgkmcnt(0)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }

    // STAGES 1: sums of one step only.
    static __device__ void run(const Operand& a, const Operand& b, int m0, int n0, int k0, int steps, const char* zeros,
                               char* lds, f32x4 (&acc)[MT][NT]) {
        if (steps <= 0) return;
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        LA la;
        LB lb;
        la.init(a, m0, k0, wave, lane);
        lb.init(b, n0, k0, wave, lane);
        Reader<BM, TRA, NA, MT> ra;
        Reader<BN, TRB, NB, NT> rb;
        ra.init(wave / WN * (BM / WM), lane);
        rb.init(wave % WN * (BN / WN), lane);
        auto issue = [&](int s) {
            char* p = lds + s % STAGES * kStage;
            la.issue(p, k0 + s * LHL_STEP, zeros, wave, lane);
            lb.issue(p + LA::kBytes, k0 + s * LHL_STEP, zeros, wave, lane);
        };
        struct Half {
            u32x4 a[MT][NA], b[NT][NB];
        } x, y;
        auto read = [&](int s, int h, Half& f) {
            const char* p = lds + s % STAGES * kStage;
#pragma unroll
            for (int j = 0; j < NT; ++j) rb.read(p + LA::kBytes, j, h, f.b[j]);
#pragma unroll
            for (int i = 0; i < MT; ++i) ra.read(p, i, h, f.a[i]);
            __builtin_amdgcn_sched_barrier(0);  // the reads stay ahead of the products
        };
        auto multiply = [&](const Half& f) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = mfma_terms<NA, NB, MOST>(f.a[i], f.b[j], acc[i][j]);
        };
        // (VEC false: a's newest step waits in registers until the buffers' next barrier)
        auto put = [&](int s) { la.put(lds + s % STAGES * kStage, wave, lane); };
#pragma unroll
        for (int s = 0; s < STAGES; ++s)
            if (s < steps) {
                issue(s);
                if (!VEC && (s + 1 < STAGES || STAGES == 1)) put(s);
            }
        if (steps >= STAGES)
            wait<STAGES - 1>();
        else
            wait<0>();
        read(0, 0, x);
        for (int s = 0; s < steps; ++s) {
            read(s, 1, y);
            multiply(x);
            __builtin_amdgcn_sched_barrier(0);
            if (s + 1 < steps) {
                if (!VEC && s + STAGES - 1 < steps) put(s + STAGES - 1);
                if (s + STAGES <= steps)  // the steps behind s + 1 are all on their way
                    wait<STAGES >= 2 ? STAGES - 2 : 0>();
                else
                    wait<0>();
                if (s + STAGES < steps) issue(s + STAGES);
                read(s + 1, 0, x);
            }
            multiply(y);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

template <int MT, int NT>
__device__ __forceinline__ void clear(f32x4 (&acc)[MT][NT]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
}

// A wavefront's part of a result as bf16, whose lanes hold four rows of a column each, to memory in which the
// rows are consecutive, 16 bytes a lane: through LDS, column by column, the 16-byte parts of column n at
// positions part ^ n.  value(i, j): the four rows of acc[i][j]; store(n, m, x): eight rows from m of column n.
template <class P, class Value, class Store>
__device__ __forceinline__ void store_part(char* lds, Value&& value, Store&& store) {
    constexpr int M = P::BM / P::WM, N = P::BN / P::WN, kParts = M / 8;
    static_assert(P::kWaves * M * N * 2 <= P::kLds && N * kParts % 64 == 0, "a part fits");
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    char* mine = lds + (threadIdx.x >> 6) * (M * N * 2);
#pragma unroll
    for (int j = 0; j < P::NT; ++j)
#pragma unroll
        for (int i = 0; i < P::MT; ++i)
            *reinterpret_cast<u32x2*>(mine + (16 * j + c) * M * 2 + ((2 * i + (g >> 1)) ^ (c % kParts)) * 16 +
                                      (g & 1) * 8) = value(i, j);
    asm volatile("" ::: "memory");  // (one wavefront's accesses to LDS are in order)
#pragma unroll
    for (int q = 0; q < N * kParts / 64; ++q) {
        const int n = q * (64 / kParts) + lane / kParts, part = lane % kParts;
        store(n, 8 * part, *reinterpret_cast<const u32x4*>(mine + n * M * 2 + (part ^ (n % 16 % kParts)) * 16));
    }
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ u32x2 round4(f32x4 x) {
    return u32x2{round2(x[0], x[1]), round2(x[2], x[3])};
}

// Tile t of tm x tn: workgroups go round the eight XCDs, so each XCD gets a run of tiles; in a run
// 8 tiles of m take turns along n, so that the tiles at work in an XCD share their operands in its L2.
__device__ __forceinline__ bool tile_of(int tm, int tn, int& m, int& n) {
    const int total = tm * tn, each = (total + 7) / 8, t = blockIdx.x % 8 * each + blockIdx.x / 8;
    if (blockIdx.x / 8 >= each || t >= total) return false;
    const int group = t / (8 * tn), first = group * 8, deep = min(8, tm - first), in = t - group * 8 * tn;
    m = first + in % deep;
    n = in / deep;
    return true;
}
inline unsigned tile_grid(size_t tiles) { return (unsigned)((tiles + 7) / 8 * 8); }

struct Parts {
    char* work;
    LossWork w;
    template <class T>
    __device__ T* at(size_t offset) const {
        return reinterpret_cast<T*>(work + offset);
    }
    __device__ int count() const { return *reinterpret_cast<const int*>(work); }
    __device__ float& top() const { return reinterpret_cast<float*>(work)[1]; }  // the largest weight (bf16 states)
    __device__ const char* zeros() const { return work + 256; }
};

// ---- the rows that count ---------------------------------------------------------------
// `runs` runs of 16 rows, a part of their columns to a workgroup, which counts the rows before its own by
// itself: four bytes a row, next to the 2 KiB and more of a row's state.  Up to 512 workgroups along the rows,
// so that what they count stays small (the loss of 2^20 rows over 1000 x 1024: 3.8 ms, with a workgroup for
// every 16 rows 19).
constexpr int kPrepRows = 16;
template <int NT, bool kGrad>
__global__ __launch_bounds__(256) void lhl_prepare_kernel(lm_head_loss_args a, Parts p, int runs) {
    __shared__ int before_sh[4], local[kPrepRows], kept_sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto counts = [&](int r) {
        const int t = a.targets[r];
        return t >= 0 && t < a.vocab;
    };
    constexpr bool kWeigh = NT == 1 && kGrad;  // a workgroup of its own, the first, finds the largest finite weight
    if (kWeigh && blockIdx.x == 0) {
        __shared__ float top_sh[4];
        if (blockIdx.y > 0) return;
        float top = 0.0f;
#pragma unroll 8
        for (int r = threadIdx.x; r < a.rows; r += 256) {
            const float g = fabsf(a.grad_loss[r]);
            top = counts(r) && g < __builtin_inff() ? fmaxf(top, g) : top;
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
        if (lane == 0) top_sh[wave] = top;
        __syncthreads();
        top = fmaxf(fmaxf(top_sh[0], top_sh[1]), fmaxf(top_sh[2], top_sh[3]));
        if (threadIdx.x == 0) p.top() = top > 0.0f ? top : 1.0f;
        return;
    }
    const int block = (int)blockIdx.x - kWeigh, first_row = block * runs * kPrepRows;
    int before = 0;
#pragma unroll 8
    for (int r = threadIdx.x; r < first_row; r += 256) before += counts(r);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) before += __shfl_xor(before, d);
    if (lane == 0) before_sh[wave] = before;
    const bool first = blockIdx.y == 0;
    if (first && block == 0 && threadIdx.x < 64) reinterpret_cast<uint32_t*>(p.work + 256)[threadIdx.x] = 0;
    __syncthreads();
    before = before_sh[0] + before_sh[1] + before_sh[2] + before_sh[3];
    uint16_t* out = p.at<uint16_t>(p.w.h_at);
    // this workgroup's parts of eight columns
    const int parts = p.w.pitch / 8, e0 = parts * blockIdx.y / gridDim.y, n = parts * (blockIdx.y + 1) / gridDim.y - e0;
    for (int run = 0; run < runs; ++run) {
        const int r0 = first_row + run * kPrepRows;
        if (wave == 0) {
            const int r = r0 + lane;
            const bool in = lane < kPrepRows && r < a.rows, kept = in && counts(r);
            const uint64_t all = __ballot(kept);
            const int mine = __popcll(all & ((1ull << lane) - 1)), c = before + mine;
            if (kept) local[mine] = r;
            if (first && kept) {
                p.at<int>(p.w.rows_at)[c] = r;
                p.at<int>(p.w.target_at)[c] = a.targets[r];
                if (kGrad) {
                    p.at<float>(p.w.lse_at)[c] = a.lse[r];
                    p.at<float>(p.w.gl_at)[c] = a.grad_loss[r];
                }
            } else if (first && in && !kGrad) {
                const float x = a.targets[r] < 0 ? 0.0f : __builtin_nanf("");
                if (a.loss) a.loss[r] = x;
                if (a.lse) a.lse[r] = x;
            }
            if (first && in) p.at<int>(p.w.place_at)[r] = kept ? c : a.targets[r] < 0 ? -1 : -2;
            if (lane == 0) {
                kept_sh = __popcll(all);
                if (first && r0 + kPrepRows >= a.rows) *reinterpret_cast<int*>(p.work) = before + __popcll(all);
            }
        }
        __syncthreads();
        const int kept = kept_sh;
        for (int u = threadIdx.x; u < kept * n; u += 256) {
            const int i = u / n, e = 8 * (e0 + u % n), c = before + i;
            const int64_t src = (int64_t)local[i] * a.h_row + e;
            u32x4 t[NT];
            if constexpr (NT == 1) {
                const uint16_t* h = static_cast<const uint16_t*>(a.h) + src;
                if (e + 8 <= a.hidden) {
                    __builtin_memcpy(&t[0], h, 16);
                } else {
                    t[0] = u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (e + j < a.hidden) t[0][j / 2] |= (uint32_t)h[j] << (j % 2 * 16);
                }
            } else {
                const float* h = static_cast<const float*>(a.h) + src;
                float x[8];
                if (e + 8 <= a.hidden) {
                    __builtin_memcpy(x, h, 32);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = e + j < a.hidden ? h[j] : 0.0f;
                }
                split8(x, t);
            }
#pragma unroll
            for (int m = 0; m < NT; ++m)
                *reinterpret_cast<u32x4*>(out + ((size_t)m * a.rows + c) * p.w.pitch + e) = t[m];
        }
        before += kept;
        __syncthreads();  // local and kept_sh have been read
    }
}

// ---- logits ---------------------------------------------------------------------------
__device__ __forceinline__ Operand states_of(const lm_head_loss_args& a, const Parts& p, int count) {
    return Operand{p.at<uint16_t>(p.w.h_at), p.w.pitch, (int64_t)a.rows * p.w.pitch, count, p.w.pitch};
}

// Tiles of vocabulary x counted rows.  kGrad false: for each row the tile's maximum and sum of
// exponentials above it (base 2), and the target's logit; true: D for vocabulary rows v0 .. of a piece, with
// bf16 states (NT 1) over the largest weight.
template <class P, int NT, bool kGrad>
__global__ __launch_bounds__(P::kThreads) void lhl_logits_kernel(lm_head_loss_args a, Parts p, int v0, int tm, int tn) {
    __shared__ __attribute__((aligned(1024))) char lds[P::kLds];
    int m, n;
    if (!tile_of(tm, tn, m, n)) return;
    const int count = p.count();
    if (n * P::BN >= count) return;
    const int vfirst = v0 + m * P::BM;
    f32x4 acc[P::MT][P::NT];
    clear(acc);
    const Operand w{a.table, a.table_row, 0, a.vocab, a.hidden};
    P::run(w, states_of(a, p, count), vfirst, n * P::BN, 0, p.w.pitch / LHL_STEP, p.zeros(), lds, acc);

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int vw = vfirst + wave / P::WN * (P::BM / P::WM) + 4 * g;
    const int nw = n * P::BN + wave % P::WN * (P::BN / P::WN) + c;
    const bool inside = vfirst + P::BM <= a.vocab;
    __syncthreads();  // the tiles in LDS have been read
    if constexpr (kGrad) {
#pragma unroll
        for (int j = 0; j < P::NT; ++j) {
            const int row = min(nw + 16 * j, count - 1);
            const float lse = p.at<float>(p.w.lse_at)[row];
            float gl = p.at<float>(p.w.gl_at)[row];
            if (NT == 1) gl /= p.top();
            const int hit = p.at<int>(p.w.target_at)[row] - vw;
            if constexpr (NT == 1) {
                // the target's entry once more, to its last bit: its logit halves the lane's values by a bit of its place
                f32x4 of[P::MT];
#pragma unroll
                for (int i = 0; i < P::MT; ++i) of[i] = acc[i][j];
#pragma unroll
                for (int b = P::MT / 2; b > 0; b /= 2)
#pragma unroll
                    for (int i = 0; i < b; ++i) of[i] = hit & 16 * b ? of[i + b] : of[i];
                const float even = hit & 2 ? of[0][2] : of[0][0], odd = hit & 2 ? of[0][3] : of[0][1];
                const float at_target = gl * (exp2_raw(((hit & 1 ? odd : even) - lse) * kLog2e) - 1.0f);
                if (hit >= 0 && hit < 16 * P::MT && hit % 16 < 4 && nw + 16 * j < count)
                    p.at<float>(p.w.rest_at)[row] = at_target - to_float(from_float<uint16_t>(at_target));
            }
#pragma unroll
            for (int i = 0; i < P::MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = exp2_raw((acc[i][j][e] - lse) * kLog2e);
                    acc[i][j][e] = gl * (hit == 16 * i + e ? y - 1.0f : y);
                    if (!inside && vw + 16 * i + e >= a.vocab) acc[i][j][e] = 0.0f;
                }
        }
        const int n0 = n * P::BN + wave % P::WN * (P::BN / P::WN);
        const int m0 = m * P::BM + wave / P::WN * (P::BM / P::WM);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            uint16_t* out = p.at<uint16_t>(p.w.d_at) + ((size_t)t * a.rows + n0) * p.w.piece + m0;
            store_part<P>(
                lds,
                [&](int i, int j) {
                    // One term: rounded to nearest, half a step of each term of the sums that read it.  The p's
                    // are as independent as the logits are; a target's entry, where its row has the largest weight,
                    // is off by at most 2^-9, and by no more than p where p is below that.
                    if constexpr (NT == 1) return round4(acc[i][j]);
                    float y[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                    const u32x2 x = {take2(y[0], y[1]), take2(y[2], y[3])};
                    acc[i][j] = f32x4{y[0], y[1], y[2], y[3]};  // (the next term's)
                    return x;
                },
                [&](int row, int v, u32x4 x) {
                    if (n0 + row < count) *reinterpret_cast<u32x4*>(out + (size_t)row * p.w.piece + v) = x;
                });
        }
    } else {
        float2* red = reinterpret_cast<float2*>(lds);
#pragma unroll
        for (int j = 0; j < P::NT; ++j) {
            const int row = nw + 16 * j;
            float top = -__builtin_inff(), sum = 0.0f;
            if (!inside)
#pragma unroll
                for (int i = 0; i < P::MT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (vw + 16 * i + e >= a.vocab) acc[i][j][e] = -__builtin_inff();
            // the target's logit, where this lane has it
            const int hit = (row < count ? p.at<int>(p.w.target_at)[row] : -1) - vw;
            if (hit >= 0 && hit < 16 * P::MT && hit % 16 < 4)
#pragma unroll
                for (int i = 0; i < P::MT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (hit == 16 * i + e) p.at<float>(p.w.logit_at)[row] = acc[i][j][e];
#pragma unroll
            for (int i = 0; i < P::MT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, acc[i][j][e]);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            // z log2 e less the maximum in one rounding; the maximum is kept in base 2, so that its own
            // rounding cancels.  Where that is too far from 0 for an exponent, the difference first.  (A part
            // past the vocabulary has no maximum: its terms are 0.)
            const float peak = top == -__builtin_inff() ? 0.0f : top;
            top *= kLog2e;
            if (__any(fabsf(peak) > 1e6f)) {
#pragma unroll
                for (int i = 0; i < P::MT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum += exp2_raw((acc[i][j][e] - peak) * kLog2e);
            } else {
                const float ref = peak * kLog2e;
#pragma unroll
                for (int i = 0; i < P::MT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum += exp2_raw(__builtin_fmaf(acc[i][j][e], kLog2e, -ref));
            }
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (g == 0) red[wave / P::WN * P::BN + wave % P::WN * (P::BN / P::WN) + 16 * j + c] = {top, sum};
        }
        __syncthreads();
        for (int x = threadIdx.x; x < P::BN; x += P::kThreads) {
            const int row = n * P::BN + x;
            if (row >= count) break;
            float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
            for (int y = 0; y < P::WM; ++y) top = fmaxf(top, red[y * P::BN + x].x);
#pragma unroll
            for (int y = 0; y < P::WM; ++y) {
                const float2 r = red[y * P::BN + x];
                sum += r.x == -__builtin_inff() ? r.y : r.y * exp2_raw(r.x - top);
            }
            p.at<float2>(p.w.part_at)[(size_t)row * tm + m] = {top, sum};
        }
    }
}

// One wavefront a row: lse from the tiles' parts.
__global__ __launch_bounds__(256) void lhl_loss_kernel(lm_head_loss_args a, Parts p, int tiles) {
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= p.count()) return;
    const float2* part = p.at<float2>(p.w.part_at) + (size_t)row * tiles;
    float top = -__builtin_inff(), sum = 0.0f;
    for (int t = lane; t < tiles; t += 64) top = fmaxf(top, part[t].x);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    for (int t = lane; t < tiles; t += 64) sum += part[t].y * exp2_raw(part[t].x - top);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    if (lane == 0) {
        const float lse = (top + log2f(sum)) * kLn2;
        const int r = p.at<int>(p.w.rows_at)[row];
        if (a.lse) a.lse[r] = lse;
        if (a.loss) a.loss[r] = lse - p.at<float>(p.w.logit_at)[row];
    }
}

// ---- gradients ------------------------------------------------------------------------
// sum[split][row][h]: tiles of h x counted rows, the sum over a split of the piece's vocabulary
// rows v0 .. v0 + width, on top of the pieces' before.
template <class P>
__global__ __launch_bounds__(P::kThreads) void lhl_grad_h_kernel(lm_head_loss_args a, Parts p, int v0, int width, int tm,
                                                                  int tn) {
    __shared__ __attribute__((aligned(1024))) char lds[P::kLds];
    int m, n;
    if (!tile_of(tm, tn * p.w.splits, m, n)) return;
    const int split = n / tn;
    n %= tn;
    const int count = p.count();
    if (n * P::BN >= count) return;
    const int steps = (width + LHL_STEP - 1) / LHL_STEP, each = (steps + p.w.splits - 1) / p.w.splits;
    const int s0 = min(split * each, steps), s1 = min(s0 + each, steps);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int hw = m * P::BM + wave / P::WN * (P::BM / P::WM) + 4 * g;
    const int nw = n * P::BN + wave % P::WN * (P::BN / P::WN) + c;
    float* sum = p.at<float>(p.w.sum_at) + (size_t)split * a.rows * p.w.pitch;
    f32x4 acc[P::MT][P::NT];
    clear(acc);
    if (v0 > 0)
#pragma unroll
        for (int i = 0; i < P::MT; ++i)
#pragma unroll
            for (int j = 0; j < P::NT; ++j)
                if (nw + 16 * j < count && hw + 16 * i < p.w.pitch)
                    acc[i][j] = *reinterpret_cast<const f32x4*>(sum + (size_t)(nw + 16 * j) * p.w.pitch + hw + 16 * i);
    const Operand w{a.table + (int64_t)v0 * a.table_row, a.table_row, 0, a.vocab - v0, a.hidden};
    const Operand d{p.at<uint16_t>(p.w.d_at), p.w.piece, (int64_t)a.rows * p.w.piece, count, p.w.piece};
    P::run(w, d, m * P::BM, n * P::BN, s0 * LHL_STEP, s1 - s0, p.zeros(), lds, acc);
#pragma unroll
    for (int i = 0; i < P::MT; ++i)
#pragma unroll
        for (int j = 0; j < P::NT; ++j)
            if (nw + 16 * j < count && hw + 16 * i < p.w.pitch)
                *reinterpret_cast<f32x4*>(sum + (size_t)(nw + 16 * j) * p.w.pitch + hw + 16 * i) = acc[i][j];
}

// 256 columns of a row of grad_h from the splits' sums, four columns a lane and a quarter of the splits a
// wavefront; rows that do not count get 0 or NaN.
template <class T>
__global__ __launch_bounds__(256) void lhl_finish_kernel(lm_head_loss_args a, Parts p) {
    __shared__ f32x4 sh[4][64];
    const int row = blockIdx.x, at = p.at<int>(p.w.place_at)[row], target = a.targets[row];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = 256 * blockIdx.y + 4 * lane;
    f32x4 x = {0, 0, 0, 0};
    float rest = 0.0f;
    uint16_t w[4] = {0, 0, 0, 0};
    if (sizeof(T) == 2 && at >= 0 && wave == 0) {  // (bf16 states: the target's part)
        rest = p.at<float>(p.w.rest_at)[at];
        const uint16_t* from = a.table + (int64_t)target * a.table_row + h;
        if (h + 4 <= a.hidden)
            __builtin_memcpy(w, from, 8);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (h + e < a.hidden) w[e] = from[e];
    }
    if (at >= 0 && h < p.w.pitch) {
        const float* sum = p.at<float>(p.w.sum_at) + (size_t)at * p.w.pitch + h;
        const int s0 = p.w.splits * wave / 4, s1 = p.w.splits * (wave + 1) / 4;
#pragma unroll 8
        for (int s = s0; s < s1; ++s) x += *reinterpret_cast<const f32x4*>(sum + (size_t)s * a.rows * p.w.pitch);
    }
    sh[wave][lane] = x;
    __syncthreads();
    if (wave > 0) return;
    x = (sh[0][lane] + sh[1][lane]) + (sh[2][lane] + sh[3][lane]);
    if (sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(rest, to_float(w[e]), x[e]);
        x *= p.top();
    }
    T* out = static_cast<T*>(a.grad_h) + (int64_t)row * a.grad_h_row + h;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (h + e < a.hidden) out[e] = from_float<T>(at == -2 ? __builtin_nanf("") : x[e]);
}

// grad_table for vocabulary rows v0 .. v0 + width: tiles of h x vocabulary.  kTop: D is over the largest weight.
template <class P, bool kTop>
__global__ __launch_bounds__(P::kThreads) void lhl_grad_table_kernel(lm_head_loss_args a, Parts p, int v0, int tm,
                                                                      int tn) {
    __shared__ __attribute__((aligned(1024))) char lds[P::kLds];
    int m, n;
    if (!tile_of(tm, tn, m, n)) return;
    const int count = p.count();
    f32x4 acc[P::MT][P::NT];
    clear(acc);
    const Operand d{p.at<uint16_t>(p.w.d_at), p.w.piece, (int64_t)a.rows * p.w.piece, count, p.w.piece};
    P::run(states_of(a, p, count), d, m * P::BM, n * P::BN, 0, (count + LHL_STEP - 1) / LHL_STEP, p.zeros(), lds, acc);
    const int wave = threadIdx.x >> 6;
    const int h0 = m * P::BM + wave / P::WN * (P::BM / P::WM);
    const int vfirst = v0 + n * P::BN + wave % P::WN * (P::BN / P::WN);
    const float top = kTop ? p.top() : 1.0f;
    __syncthreads();  // the tiles in LDS have been read
    store_part<P>(
        lds, [&](int i, int j) { return round4(kTop ? acc[i][j] * top : acc[i][j]); },
        [&](int v, int h, u32x4 x) {
            if (vfirst + v >= a.vocab) return;
            h += h0;
            uint16_t* out = a.grad_table + (int64_t)(vfirst + v) * a.grad_table_row + h;
            if (h + 8 <= a.hidden) {
                __builtin_memcpy(out, &x, 16);  // (rows may start at any element)
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (h + e < a.hidden) out[e] = (uint16_t)(x[e / 2] >> (e % 2 * 16));
            }
        });
}

// ---- launches --------------------------------------------------------------------------
template <int NT>
hipError_t prepare(const lm_head_loss_args& a, const Parts& p, bool grad, hipStream_t s) {
    const unsigned columns = std::min(4, p.w.pitch / LHL_STEP);
    const int blocks = std::max(1, (a.rows + kPrepRows - 1) / kPrepRows), runs = (blocks + 511) / 512;
    const dim3 grid((unsigned)((blocks + runs - 1) / runs + (NT == 1 && grad)), columns);
    if (grad)
        lhl_prepare_kernel<NT, true><<<grid, 256, 0, s>>>(a, p, runs);
    else
        lhl_prepare_kernel<NT, false><<<grid, 256, 0, s>>>(a, p, runs);
    return hipGetLastError();
}

// Vocabulary rows and counted rows of a tile of logits.  Up to 32 rows take tiles of 128 x 32, which leave two
// workgroups of three stages a compute unit (one row: 25 us); up to 64 of 256 x 64 (48 float32 rows: 30 us, in
// tiles of 128 x 64 a third more); many bf16 ones of 256 x 256 (4096: 490 us, in tiles of 128 x 128 7 % more), whose
// operands are the fewest bytes of LDS a product; the others of 128 x 128, but float32's three terms of 256 x 128 where
// there is more than one such for a compute unit, whose LDS either fills: with eight wavefronts in place of
// four (4096 x 65536 x 1024: 1.28 ms for 1.67; 200 x 3000 45 us for 37).
struct TileOf {
    int vocab, rows;
};
bool more_than_units(size_t tiles) { return tiles > 256; }
template <int NT, bool VEC>
TileOf tile_for(int rows, int width) {
    if (rows <= 32) return {128, 32};
    if (rows <= 64) return {VEC ? 256 : 128, 64};
    if (NT == 1 && VEC && rows >= 1024) return {256, 256};
    if (NT == 3 && more_than_units((size_t)((width + 127) / 128) * ((rows + 127) / 128))) return {256, 128};
    return {128, 128};
}

template <int BM, int BN, int NT, bool VEC, bool kGrad>
hipError_t logits(const lm_head_loss_args& a, const Parts& p, int v0, int width, hipStream_t s) {
    constexpr int WN = BN == 256 ? 4 : BN == 128 ? 2 : 1, WM = (BM == 256 ? 8 : 4) / WN;
    constexpr int kStages = BN >= 128 || !VEC || (BM == 256 && NT == 3) ? 2 : 3;
    using P = Product<BM, BN, WM, WN, false, false, 1, NT, 3, VEC, kStages>;
    const int tm = (width + BM - 1) / BM, tn = (a.rows + BN - 1) / BN;
    lhl_logits_kernel<P, NT, kGrad>
        <<<dim3(tile_grid((size_t)tm * tn)), P::kThreads, 0, s>>>(a, p, v0, tm, tn);
    return hipGetLastError();
}

template <int NT, bool VEC, bool kGrad>
hipError_t logits_of(const lm_head_loss_args& a, const Parts& p, int v0, int width, hipStream_t s) {
    const TileOf t = tile_for<NT, VEC>(a.rows, width);
    if (t.rows == 32) return logits<128, 32, NT, VEC, kGrad>(a, p, v0, width, s);
    if (t.rows == 64) return logits<VEC ? 256 : 128, 64, NT, VEC, kGrad>(a, p, v0, width, s);
    if constexpr (NT == 1 && VEC)
        if (t.rows == 256) return logits<256, 256, NT, VEC, kGrad>(a, p, v0, width, s);
    if constexpr (NT == 3)
        if (t.vocab == 256) return logits<256, 128, NT, VEC, kGrad>(a, p, v0, width, s);
    return logits<128, 128, NT, VEC, kGrad>(a, p, v0, width, s);
}

template <int NT, bool VEC>
hipError_t loss(const lm_head_loss_args& a, const Parts& p, hipStream_t s) {
    hipError_t e = prepare<NT>(a, p, false, s);
    if (e == hipSuccess) e = logits_of<NT, VEC, false>(a, p, 0, a.vocab, s);
    if (e != hipSuccess) return e;
    const int tile = tile_for<NT, VEC>(a.rows, a.vocab).vocab, tiles = (a.vocab + tile - 1) / tile;
    lhl_loss_kernel<<<dim3((unsigned)((a.rows + 3) / 4)), 256, 0, s>>>(a, p, tiles);
    return hipGetLastError();
}

template <int BM, int BN, int NT, bool VEC>
hipError_t grad_h(const lm_head_loss_args& a, const Parts& p, int v0, int width, hipStream_t s) {
    using P = Product<BM, BN, BN == 128 ? BM / 64 : 4, BN / 64, true, false, 1, NT, 3, VEC, 2>;
    const int tm = (p.w.pitch + BM - 1) / BM, tn = (a.rows + BN - 1) / BN;
    lhl_grad_h_kernel<P>
        <<<dim3(tile_grid((size_t)tm * tn * p.w.splits)), P::kThreads, 0, s>>>(a, p, v0, width, tm, tn);
    return hipGetLastError();
}

template <int NT, bool VEC>
hipError_t grad_h_of(const lm_head_loss_args& a, const Parts& p, int v0, int width, hipStream_t s) {
    if (a.rows <= 64) return grad_h<128, 64, NT, VEC>(a, p, v0, width, s);
    if constexpr (NT == 3)  // as for the logits (4096 rows' piece of 4096 columns 99 us)
        if (more_than_units((size_t)((p.w.pitch + 127) / 128) * ((a.rows + 127) / 128) * p.w.splits))
            return grad_h<256, 128, NT, VEC>(a, p, v0, width, s);
    return grad_h<128, 128, NT, VEC>(a, p, v0, width, s);
}

template <int NT, bool VEC>
hipError_t grad(const lm_head_loss_args& a, const Parts& p, hipStream_t s) {
    hipError_t e = prepare<NT>(a, p, true, s);
    for (int v0 = 0; v0 < a.vocab && e == hipSuccess; v0 += p.w.piece) {
        const int width = std::min(p.w.piece, a.vocab - v0);
        if (a.rows > 0) e = logits_of<NT, VEC, true>(a, p, v0, width, s);
        if (e == hipSuccess && a.grad_h && a.rows > 0)
            e = grad_h_of<NT, VEC>(a, p, v0, width, s);
        if (e == hipSuccess && a.grad_table) {
            constexpr int N2 = NT == 1 ? 1 : 2;  // a bf16 result: 3 x 2^-16 of its terms
            if constexpr (NT == 1)
                if (a.rows >= 1024) {  // (4096 rows' piece 110 us, in tiles of 128 x 128 15 % more)
                    using P = Product<256, 256, 2, 4, true, true, 1, 1, 1, true, 2>;
                    const int tm = (p.w.pitch + 255) / 256, tn = (width + 255) / 256;
                    lhl_grad_table_kernel<P, true>
                        <<<dim3(tile_grid((size_t)tm * tn)), P::kThreads, 0, s>>>(a, p, v0, tm, tn);
                    e = hipGetLastError();
                    continue;
                }
            const int tm = (p.w.pitch + 127) / 128, tn = (width + 127) / 128;
            const dim3 grid(tile_grid((size_t)tm * tn));
            if (a.rows <= LHL_STEP) {  // one step: its LDS for two workgroups more
                using P = Product<128, 128, 2, 2, true, true, N2, N2, N2, true, 1>;
                lhl_grad_table_kernel<P, NT == 1><<<grid, P::kThreads, 0, s>>>(a, p, v0, tm, tn);
            } else {  // (two terms' LDS leaves one workgroup a compute unit: of eight wavefronts)
                using P = Product<128, 128, N2 == 2 ? 4 : 2, 2, true, true, N2, N2, N2, true, 2>;
                lhl_grad_table_kernel<P, NT == 1><<<grid, P::kThreads, 0, s>>>(a, p, v0, tm, tn);
            }
            e = hipGetLastError();
        }
    }
    if (e != hipSuccess || !a.grad_h || a.rows == 0) return e;
    const dim3 grid((unsigned)a.rows, (unsigned)((p.w.pitch + 255) / 256));
    if (NT == 1)
        lhl_finish_kernel<uint16_t><<<grid, 256, 0, s>>>(a, p);
    else
        lhl_finish_kernel<float><<<grid, 256, 0, s>>>(a, p);
    return hipGetLastError();
}

bool rows_of_16(const lm_head_loss_args& a) {
    return ((uintptr_t)a.table | (uintptr_t)(a.table_row * 2) | (uintptr_t)(a.hidden * 2)) % 16 == 0;
}

}  // namespace

hipError_t lhl_launch_loss(const lm_head_loss_args& a, const LossWork& w, hipStream_t s) {
    const Parts p{static_cast<char*>(a.work), w};
    if (a.dtype == QWEN_BF16) return rows_of_16(a) ? loss<1, true>(a, p, s) : loss<1, false>(a, p, s);
    return rows_of_16(a) ? loss<3, true>(a, p, s) : loss<3, false>(a, p, s);
}

hipError_t lhl_launch_grad(const lm_head_loss_args& a, const LossWork& w, hipStream_t s) {
    const Parts p{static_cast<char*>(a.work), w};
    if (a.dtype == QWEN_BF16) return rows_of_16(a) ? grad<1, true>(a, p, s) : grad<1, false>(a, p, s);
    return rows_of_16(a) ? grad<3, true>(a, p, s) : grad<3, false>(a, p, s);
}
