// linear_attention.hip -- gated linear attention (gdn_dev_prompt, gdn_dev_step).
//
// One head, one sequence, tokens t = 1, 2, ..:
//   S' = a_t S;  u_t = b_t (v_t - S'^T k_t)  (no b: u_t = v_t)
//   S  = S' + k_t u_t^T;  o_t = scale S^T q_t
// as 04/qwen_kernels_opt.c:664-813 has it for one token.
//
// Prompt form.  In a chunk of 64 tokens that starts from S0, with
// g_i = log2 a_1 + .. + log2 a_i,
//   (I + L) U = diag(b) (V - diag(2^g) K S0),   L_ij = b_i 2^(g_i - g_j) k_i.k_j  (j < i)
//   O = scale (diag(2^g) Q S0 + P U),           P_ij = 2^(g_i - g_j) q_i.k_j      (j <= i)
//   S0 <- 2^(g_C) S0 + K^T diag(2^(g_C - g)) U
// gdn_chunk_kernel makes T = (I + L)^-1 diag(b), P and the decays of every chunk
// side by side; gdn_scan_kernel takes the state from chunk to chunk, 16 of a
// head's value columns in a workgroup (the columns do not mix).
//
// Arithmetic: every product runs on the bf16 matrix cores, a float32 operand as
// the sum of three bf16 terms (bf16_terms.h), a product of two such sums as the
// six pairs of terms above 2^-24.  What only a bf16 output sees (S0 in Q S0, P, U in P U) has two
// terms: 2^-16, against the output's own 2^-9.
#include "bf16_terms.h"
#include "linear_attention.h"

namespace {

constexpr int C = GDN_CHUNK;

// Elements i .. i + 7 of a row as terms; those from dim on are zero.
template <int NT>
__device__ __forceinline__ void load_terms(const void* row, int i, int dim, bool vec, u32x4 (&t)[NT]) {
    if constexpr (NT == 1) {
        const uint16_t* p = static_cast<const uint16_t*>(row);
        if (vec && i + 8 <= dim) {
            t[0] = *reinterpret_cast<const u32x4*>(p + i);
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t lo = i + 2 * j < dim ? p[i + 2 * j] : 0, hi = i + 2 * j + 1 < dim ? p[i + 2 * j + 1] : 0;
            t[0][j] = lo | hi << 16;
        }
    } else {
        const float* p = static_cast<const float*>(row);
        float x[8];
        if (vec && i + 8 <= dim) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p + i), b = *reinterpret_cast<const f32x4*>(p + i + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = a[j], x[4 + j] = b[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = i + j < dim ? p[i + j] : 0.0f;
        }
        split8(x, t);
    }
}

// 2^d, d <= 0 as a rule; the whole part exactly.
__device__ __forceinline__ float exp2_of(double d) {
    const double w = floor(d);
    return ldexpf(exp2f((float)(d - w)), (int)fmax(fmin(w, 1000.0), -1000.0));
}

// A sequence's rows, kept inside [0, rows] whatever starts holds.
__device__ __forceinline__ void span(const gdn_dev_args& a, int s, int& first, int& n) {
    if (!a.starts) {
        first = 0;
        n = a.rows;
        return;
    }
    first = min(max(a.starts[s], 0), a.rows);
    n = min(max(a.starts[s + 1], first), a.rows) - first;
}

// The slot of sequence s, or -1 where it is skipped.  Every lane of the workgroup.
__device__ __forceinline__ int slot_of(const gdn_dev_args& a, int s) {
    if (!a.slots) return s < a.n_slots ? s : -1;
    const int slot = a.slots[s];
    if (slot < 0 || slot >= a.n_slots) return -1;
    int twice = 0;
    for (int i = threadIdx.x & 63; i < s; i += 64) twice |= a.slots[i] == slot;
    return __any(twice) ? -1 : slot;
}

// The byte offsets of the work buffer's parts for one chunk.
struct Places {
    char *k, *kt, *q;            // fragments of key head: [4 or 2 ks row tiles][ks or 2 steps][nt] KiB
    char *t, *p;                 // triangular fragments: tile(rt, ts) of 6, x 3 or no terms
    float *up, *down, *last;     // 2^g, 2^(g_C - g), 2^(g_C)
};
template <int KS, int NT, int NO>
__device__ __forceinline__ Places places(const gdn_dev_args& a, size_t n_chunks, size_t chunk, int hk, int hv) {
    constexpr size_t kKey = (size_t)3 * 4 * KS * NT * 1024, kTri = (size_t)(18 + 6 * NO) * 1024 + 1024;
    char* base = static_cast<char*>(a.work);
    Places w;
    w.k = base + (chunk * a.heads_k + hk) * kKey;
    w.kt = w.k + (size_t)4 * KS * NT * 1024;
    w.q = w.kt + (size_t)4 * KS * NT * 1024;
    char* tri = base + n_chunks * a.heads_k * kKey + (chunk * a.heads_v + hv) * kTri;
    w.t = tri;
    w.p = tri + 18 * 1024;
    w.up = reinterpret_cast<float*>(tri + (18 + 6 * NO) * 1024);
    w.down = w.up + C;
    w.last = w.down + C;
    return w;
}
// Tiles of a lower triangle of 4 x 2 tiles of 16 x 32: row tiles 0 and 1 have only
// step 0.
__device__ __forceinline__ constexpr int tri_tile(int rt, int ts) { return rt < 2 ? rt : 2 + (rt - 2) * 2 + ts; }

// ---- chunks -------------------------------------------------------------------------
// One chunk of one value head; wavefront w has its 16-row tile w.  What it writes is
// in the order in which gdn_scan_kernel's lanes load it.
template <int KS, int NT, bool kDelta>
__global__ __launch_bounds__(256) void gdn_chunk_kernel(gdn_dev_args a, size_t n_chunks, int vec_q, int vec_k) {
    constexpr int NO = NT == 1 ? 2 : 3;
    __shared__ u32x4 ksh[4 * KS * NT * 64];  // K fragments
    __shared__ __attribute__((aligned(16))) float lsh[C][C + 4];
    __shared__ __attribute__((aligned(16))) float psh[C][C + 4];
    __shared__ double gsh[C];
    __shared__ float bsh[C];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
    const size_t chunk = blockIdx.x / a.heads_v;
    const int hv = blockIdx.x % a.heads_v, reach = a.heads_v / a.heads_k, hk = hv / reach;

    // the sequence: the last s with starts[s] / 64 + s <= chunk
    int seq = 0;
    if (a.starts) {
        int lo = 0, hi = a.n_seq;  // key(lo) <= chunk < key(hi)
        while (hi - lo > 1) {
            const int step = (hi - lo + 63) / 64, at = lo + (lane + 1) * step;
            const bool le = at < hi && (size_t)(min(max(a.starts[at], 0), a.rows) / C + at) <= chunk;
            const int below = __popcll(__ballot(le));
            const int nlo = lo + below * step;
            hi = min(hi, lo + (below + 1) * step);
            lo = min(nlo, hi - 1);
        }
        seq = lo;
    }
    int first, len;
    span(a, seq, first, len);
    const long c = (long)chunk - (first / C + seq);
    if (c < 0 || c * C >= len) return;
    const int row0 = first + (int)c * C, n = min(C, len - (int)c * C);
    const Places at = places<KS, NT, NO>(a, n_chunks, chunk, hk, hv);
    const bool keys = hv % reach == 0;  // this workgroup leaves the key head's fragments too

    // K and Q rows of tile w as operand fragments
    u32x4 kf[KS][NT], qf[KS][NT];
    const int r = 16 * w + col;
    const int es = NT == 1 ? 2 : 4;
    const char* krow = static_cast<const char*>(a.k) + ((int64_t)(row0 + r) * a.k_row + (int64_t)hk * a.dim_k) * es;
    const char* qrow = static_cast<const char*>(a.q) + ((int64_t)(row0 + r) * a.q_row + (int64_t)hk * a.dim_k) * es;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int dim = r < n ? a.dim_k : 0;
        load_terms(krow, 32 * s + 8 * grp, dim, vec_k, kf[s]);
        load_terms(qrow, 32 * s + 8 * grp, dim, vec_q, qf[s]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int f = ((w * KS + s) * NT + t) * 64 + lane;
            ksh[f] = kf[s][t];
            if (keys) {
                reinterpret_cast<u32x4*>(at.k)[f] = kf[s][t];
                reinterpret_cast<u32x4*>(at.q)[f] = qf[s][t];
            }
        }
    }
    if (w == 0) {
        // g in double: differences of large sums stay exact to a float32.  A decay of 0
        // counts as 2^-16384, which no product brings back.
        const int64_t row = (int64_t)(row0 + lane) * a.gate_row + hv;
        double g = 0.0;
        if (lane < n) {
            const float al = a.alpha[row];
            g = al == 0.0f ? -16384.0 : log2((double)al);
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double o = __shfl_up(g, d);
            if (lane >= d) g += o;
        }
        const double gc = __shfl(g, 63);
        gsh[lane] = g;
        bsh[lane] = kDelta && lane < n ? a.beta[row] : 0.0f;
        at.up[lane] = exp2_of(g);
        at.down[lane] = exp2_of(gc - g);
        if (lane == 0) at.last[0] = exp2_of(gc);
    }
    __syncthreads();

    // K K^T and Q K^T, the tiles on and below the diagonal
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) {
        if (ct > w) {
#pragma unroll
            for (int e = 0; e < 4; ++e) psh[16 * w + 4 * grp + e][16 * ct + col] = 0.0f;
            continue;
        }
        f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            u32x4 b[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) b[t] = ksh[((ct * KS + s) * NT + t) * 64 + lane];
            if (kDelta) kk = mfma_terms<NT, NT, 3>(kf[s], b, kk);
            qk = mfma_terms<NT, NT, 3>(qf[s], b, qk);
        }
        const int j = 16 * ct + col;
        const double gj = gsh[j];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = 16 * w + 4 * grp + e;
            const float d = i >= j ? exp2_of(gsh[i] - gj) : 0.0f;
            psh[i][j] = i >= j ? qk[e] * d : 0.0f;
            if (kDelta) lsh[i][j] = i > j ? bsh[i] * d * kk[e] : 0.0f;
        }
    }
    __syncthreads();

    if (kDelta && w == 0) {
        // lane j solves (I + L) x = b_j e_j from the first row down: column j of T
        float x[C];
        const float bj = bsh[lane];
#pragma unroll
        for (int i = 0; i < C; ++i) {
            float s0 = i == lane ? bj : 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
#pragma unroll
            for (int j = 0; j < (i & ~3); j += 4) {
                const f32x4 l = *reinterpret_cast<const f32x4*>(&lsh[i][j]);
                s0 = __builtin_fmaf(-l[0], x[j], s0);
                s1 = __builtin_fmaf(-l[1], x[j + 1], s1);
                s2 = __builtin_fmaf(-l[2], x[j + 2], s2);
                s3 = __builtin_fmaf(-l[3], x[j + 3], s3);
            }
#pragma unroll
            for (int j = i & ~3; j < i; ++j) s0 = __builtin_fmaf(-lsh[i][j], x[j], s0);
            x[i] = (s0 + s1) + (s2 + s3);
        }
#pragma unroll
        for (int i = 0; i < C; ++i) lsh[i][lane] = x[i];
    }
    if (keys) {
        // K^T: row i of the state, eight tokens to a lane
        const uint16_t* kw = reinterpret_cast<const uint16_t*>(ksh);
        for (int f = w; f < 2 * KS * 2 * NT; f += 4) {
            const int t = f % NT, ts = f / NT % 2, it = f / NT / 2;
            const int i = 16 * it + col, s = i / 32, sub = i % 32 / 8, e = i % 8;
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                uint32_t h[2];
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    const int tok = 32 * ts + 8 * grp + j + d;
                    h[d] = kw[((((tok / 16) * KS + s) * NT + t) * 64 + sub * 16 + tok % 16) * 8 + e];
                }
                v[j / 2] = h[0] | h[1] << 16;
            }
            reinterpret_cast<u32x4*>(at.kt)[f * 64 + lane] = v;
        }
    }
    if (kDelta) __syncthreads();

    // T and P as operand fragments of row tile w
#pragma unroll
    for (int ts = 0; ts < 2; ++ts) {
        if (ts == 1 && w < 2) break;
        const int tile = tri_tile(w, ts);
        float x[8];
        if (kDelta) {
            u32x4 t[3];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = lsh[r][32 * ts + 8 * grp + j];
            split8(x, t);
#pragma unroll
            for (int m = 0; m < 3; ++m) reinterpret_cast<u32x4*>(at.t)[(tile * 3 + m) * 64 + lane] = t[m];
        }
        u32x4 p[NO];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = psh[r][32 * ts + 8 * grp + j];
        split8(x, p);
#pragma unroll
        for (int m = 0; m < NO; ++m) reinterpret_cast<u32x4*>(at.p)[(tile * NO + m) * 64 + lane] = p[m];
    }
}

// ---- the state from chunk to chunk --------------------------------------------------
// 16 value columns of one head of one sequence.  Wavefront w has rows 16 w .. of each
// chunk, and TPW 16-row tiles of the state in its accumulators; the state, the right
// side, and U pass between the wavefronts as bf16 terms in LDS, [term][column][row], a
// row of padding of 16 bytes.
template <int KS, int NT, bool kDelta, class T>
__global__ __launch_bounds__(256, 1) void gdn_scan_kernel(gdn_dev_args a, size_t n_chunks, int slices) {
    constexpr int NO = NT == 1 ? 2 : 3;
    constexpr int TPW = KS >= 2 ? KS / 2 : 1;
    constexpr int SP = 32 * KS + 8, UP = C + 8;  // pitches, in bf16
    __shared__ __attribute__((aligned(16))) uint16_t ssh[3][16][SP];
    __shared__ __attribute__((aligned(16))) uint16_t rsh[kDelta ? 3 : 1][16][UP];
    __shared__ __attribute__((aligned(16))) uint16_t ush[NO][16][UP];
    __shared__ __attribute__((aligned(16))) uint16_t dsh[3][16][UP];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
    // a head's slices a multiple of the heads apart: with 8 | heads on one XCD, whose
    // L2 then holds the fragments that they share
    const int heads = a.n_seq * a.heads_v;
    const int sh = blockIdx.x % heads, slice = blockIdx.x / heads;
    const int seq = sh / a.heads_v, hv = sh % a.heads_v, hk = hv / (a.heads_v / a.heads_k);
    const int slot = slot_of(a, seq);
    if (slot < 0) return;
    int first, len;
    span(a, seq, first, len);
    const int j = 16 * slice + col;  // value column
    const bool jin = j < a.dim_v;

    // the state: lane holds rows 16 tile + 4 grp .. + 3 of column j
    const size_t head_state = ((size_t)slot * a.heads_v + hv) * a.dim_k * a.dim_v;
    f32x4 S[TPW];
    size_t s_at[TPW];
    bool s_in[TPW];
#pragma unroll
    for (int t = 0; t < TPW; ++t) {
        const int i = 16 * (w * TPW + t) + 4 * grp;
        s_in[t] = jin && i < a.dim_k;
        s_at[t] = head_state + (((size_t)(j / 4) * (a.dim_k / 4) + i / 4) * 4 + j % 4) * 4;
        S[t] = f32x4{0, 0, 0, 0};
        if (s_in[t] && a.state_in) S[t] = *reinterpret_cast<const f32x4*>(a.state_in + s_at[t]);
    }
    auto put_state = [&] {
#pragma unroll
        for (int t = 0; t < TPW; ++t) {
            if (w * TPW + t >= 2 * KS) break;
            u32x2 x[3];
            split4(S[t], x);
#pragma unroll
            for (int m = 0; m < 3; ++m)
                *reinterpret_cast<u32x2*>(&ssh[m][col][16 * (w * TPW + t) + 4 * grp]) = x[m];
        }
    };

    const int nc = (len + C - 1) / C;
    const size_t chunk0 = (size_t)(first / C) + seq;
    u32x4 kf[KS][NT], qf[KS][NT], tf[2][3], ktf[TPW][2][NT], pf[2][NO];
    float v[4];
    f32x4 up, down;
    float last;
    const T* vbase = static_cast<const T*>(a.v) + (int64_t)hv * a.dim_v + j;
    auto load_kq = [&](const Places& at) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int f = ((w * KS + s) * NT + t) * 64 + lane;
                if (kDelta) kf[s][t] = reinterpret_cast<const u32x4*>(at.k)[f];
                qf[s][t] = reinterpret_cast<const u32x4*>(at.q)[f];
            }
    };
    auto load_vt = [&](const Places& at, int c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int t = c * C + 16 * w + 4 * grp + e;
            v[e] = t < len && jin ? to_float<T>(vbase[(int64_t)(first + t) * a.v_row]) : 0.0f;
        }
        up = *reinterpret_cast<const f32x4*>(at.up + 16 * w + 4 * grp);
        if (kDelta)
#pragma unroll
            for (int ts = 0; ts < 2; ++ts)
                if (ts == 0 || w >= 2)
#pragma unroll
                    for (int m = 0; m < 3; ++m)
                        tf[ts][m] = reinterpret_cast<const u32x4*>(at.t)[(tri_tile(w, ts) * 3 + m) * 64 + lane];
    };
    auto load_down = [&](const Places& at) {
        down = *reinterpret_cast<const f32x4*>(at.down + 16 * w + 4 * grp);
    };
    auto load_kt = [&](const Places& at) {
        last = at.last[0];
#pragma unroll
        for (int t = 0; t < TPW; ++t)
            if (w * TPW + t < 2 * KS)
#pragma unroll
                for (int ts = 0; ts < 2; ++ts)
#pragma unroll
                    for (int m = 0; m < NT; ++m)
                        ktf[t][ts][m] =
                            reinterpret_cast<const u32x4*>(at.kt)[(((w * TPW + t) * 2 + ts) * NT + m) * 64 + lane];
    };
    auto load_p = [&](const Places& at) {
#pragma unroll
        for (int ts = 0; ts < 2; ++ts)
            if (ts == 0 || w >= 2)
#pragma unroll
                for (int m = 0; m < NO; ++m)
                    pf[ts][m] = reinterpret_cast<const u32x4*>(at.p)[(tri_tile(w, ts) * NO + m) * 64 + lane];
    };
    if (nc > 0) {
        const Places at = places<KS, NT, NO>(a, n_chunks, chunk0, hk, hv);
        load_kq(at);
        load_vt(at, 0);
        load_down(at);
        load_kt(at);
        load_p(at);
    }
    put_state();
    for (int c = 0; c < nc; ++c) {
        // the next chunk's fragments are loaded into each register as soon as it is free
        const bool more = c + 1 < nc;
        const Places next = places<KS, NT, NO>(a, n_chunks, chunk0 + c + 1, hk, hv);
        __syncthreads();
        // K S0 and Q S0
        f32x4 ks = {0, 0, 0, 0}, o = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            u32x4 b[3], bo[NO];
#pragma unroll
            for (int m = 0; m < 3; ++m) b[m] = *reinterpret_cast<const u32x4*>(&ssh[m][col][32 * s + 8 * grp]);
#pragma unroll
            for (int m = 0; m < NO; ++m) bo[m] = b[m];
            if (kDelta) ks = mfma_terms<NT, 3, 3>(kf[s], b, ks);
            o = mfma_terms<NT, NO, NO>(qf[s], bo, o);
        }
        if (more) load_kq(next);
        o *= up;
        f32x4 u = {v[0], v[1], v[2], v[3]};
        if (kDelta) {
            u -= up * ks;
            u32x2 x[3];
            split4(u, x);
#pragma unroll
            for (int m = 0; m < 3; ++m) *reinterpret_cast<u32x2*>(&rsh[m][col][16 * w + 4 * grp]) = x[m];
            __syncthreads();
            u = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int ts = 0; ts < 2; ++ts)
                if (ts == 0 || w >= 2) {
                    u32x4 b[3];
#pragma unroll
                    for (int m = 0; m < 3; ++m)
                        b[m] = *reinterpret_cast<const u32x4*>(&rsh[m][col][32 * ts + 8 * grp]);
                    u = mfma_terms<3, 3, 3>(tf[ts], b, u);
                }
        }
        if (more) load_vt(next, c + 1);
        {
            u32x2 x[NO], d[3];
            split4(u, x);
            split4(u * down, d);
#pragma unroll
            for (int m = 0; m < NO; ++m) *reinterpret_cast<u32x2*>(&ush[m][col][16 * w + 4 * grp]) = x[m];
#pragma unroll
            for (int m = 0; m < 3; ++m) *reinterpret_cast<u32x2*>(&dsh[m][col][16 * w + 4 * grp]) = d[m];
        }
        if (more) load_down(next);
        __syncthreads();
        // S0 <- last S0 + K^T (down U)
#pragma unroll
        for (int t = 0; t < TPW; ++t) S[t] *= last;
#pragma unroll
        for (int ts = 0; ts < 2; ++ts) {
            u32x4 b[3];
#pragma unroll
            for (int m = 0; m < 3; ++m) b[m] = *reinterpret_cast<const u32x4*>(&dsh[m][col][32 * ts + 8 * grp]);
#pragma unroll
            for (int t = 0; t < TPW; ++t)
                if (w * TPW + t < 2 * KS) S[t] = mfma_terms<NT, 3, 3>(ktf[t][ts], b, S[t]);
        }
        if (more) load_kt(next);
        put_state();
        // O = scale (up Q S0 + P U)
#pragma unroll
        for (int ts = 0; ts < 2; ++ts)
            if (ts == 0 || w >= 2) {
                u32x4 b[NO];
#pragma unroll
                for (int m = 0; m < NO; ++m) b[m] = *reinterpret_cast<const u32x4*>(&ush[m][col][32 * ts + 8 * grp]);
                o = mfma_terms<NO, NO, NO>(pf[ts], b, o);
            }
        if (more) load_p(next);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int t = c * C + 16 * w + 4 * grp + e;
            if (t < len && jin)
                static_cast<T*>(a.out)[(int64_t)(first + t) * a.out_row + (int64_t)hv * a.dim_v + j] =
                    from_float<T>(a.scale * o[e]);
        }
    }
#pragma unroll
    for (int t = 0; t < TPW; ++t)
        if (s_in[t]) *reinterpret_cast<f32x4*>(a.state_out + s_at[t]) = S[t];
}

// ---- one token ------------------------------------------------------------------------
// With the old state S: u = b (v - a S^T k), out = scale (a S^T q + (k.q) u), S <- a S + k u^T:
// one pass over the state, whose bytes bound it.  A wavefront has COLS / 4 groups of
// four value columns; lane 4 g + l has rows 4 (g + 16 n) .. + 3 of column l of each, one
// 16-byte load and store each, 1 KiB a wavefront.
template <int NI, int G, class T>
__global__ __launch_bounds__(256) void gdn_step_kernel(gdn_dev_args a, int groups) {
    const int lane = threadIdx.x & 63, l = lane & 3, g = lane >> 2;
    const int unit = blockIdx.x * 4 + (threadIdx.x >> 6);  // (sequence, head, run of G column groups)
    const int runs = (groups + G - 1) / G, per_seq = a.heads_v * runs;
    const int seq = unit / per_seq;
    if (seq >= a.n_seq) return;
    const int hv = unit % per_seq / runs, jg0 = unit % runs * G;
    const int slot = slot_of(a, seq);
    if (slot < 0) return;
    const int hk = hv / (a.heads_v / a.heads_k);
    const size_t head_state = ((size_t)slot * a.heads_v + hv) * a.dim_k * a.dim_v;
    const int ng = a.dim_k / 4;
    f32x4 S[G][NI];
#pragma unroll
    for (int m = 0; m < G; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            const int ig = g + 16 * n;
            S[m][n] = f32x4{0, 0, 0, 0};
            if (jg0 + m < groups && ig < ng && a.state_in)
                S[m][n] = *reinterpret_cast<const f32x4*>(a.state_in + head_state +
                                                          (((size_t)(jg0 + m) * ng + ig) * 4 + l) * 4);
        }
    const T* q = static_cast<const T*>(a.q) + (int64_t)seq * a.q_row + (int64_t)hk * a.dim_k;
    const T* k = static_cast<const T*>(a.k) + (int64_t)seq * a.k_row + (int64_t)hk * a.dim_k;
    const T* v = static_cast<const T*>(a.v) + (int64_t)seq * a.v_row + (int64_t)hv * a.dim_v;
    const float al = a.alpha[(int64_t)seq * a.gate_row + hv];
    const float be = a.beta ? a.beta[(int64_t)seq * a.gate_row + hv] : 0.0f;
    f32x4 kf[NI], qf[NI];
    float qk = 0.0f;
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = 4 * (g + 16 * n) + e;
            kf[n][e] = i < a.dim_k ? to_float<T>(k[i]) : 0.0f;
            qf[n][e] = i < a.dim_k ? to_float<T>(q[i]) : 0.0f;
            qk = __builtin_fmaf(kf[n][e], qf[n][e], qk);
        }
    float vj[G];
#pragma unroll
    for (int m = 0; m < G; ++m) vj[m] = jg0 + m < groups ? to_float<T>(v[4 * (jg0 + m) + l]) : 0.0f;
    auto over_rows = [](float x) {  // the sum over the 16 lanes of a column, in each
        x += __shfl_xor(x, 4);
        x += __shfl_xor(x, 8);
        x += __shfl_xor(x, 16);
        return x + __shfl_xor(x, 32);
    };
    qk = over_rows(qk);
    float kv[G], qs[G];
#pragma unroll
    for (int m = 0; m < G; ++m) {
        kv[m] = qs[m] = 0.0f;
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                kv[m] = __builtin_fmaf(S[m][n][e], kf[n][e], kv[m]);
                qs[m] = __builtin_fmaf(S[m][n][e], qf[n][e], qs[m]);
            }
    }
#pragma unroll
    for (int m = 0; m < G; ++m) {
        qs[m] = over_rows(qs[m]);
        float u = vj[m];
        if (a.beta) u = be * (u - al * over_rows(kv[m]));
        if (jg0 + m < groups) {
            if (g == 0)
                static_cast<T*>(a.out)[(int64_t)seq * a.out_row + (int64_t)hv * a.dim_v + 4 * (jg0 + m) + l] =
                    from_float<T>(a.scale * __builtin_fmaf(qk, u, al * qs[m]));
#pragma unroll
            for (int n = 0; n < NI; ++n) {
                const int ig = g + 16 * n;
                if (ig < ng) {
                    f32x4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(kf[n][e], u, al * S[m][n][e]);
                    *reinterpret_cast<f32x4*>(a.state_out + head_state + (((size_t)(jg0 + m) * ng + ig) * 4 + l) * 4) =
                        x;
                }
            }
        }
    }
}

bool rows_of_16(const void* p, int64_t row, int dim, int es) {
    return ((uintptr_t)p | (uintptr_t)(row * es) | (uintptr_t)(dim * es)) % 16 == 0;
}

template <int KS, int NT, bool kDelta>
hipError_t launch_prompt(const gdn_dev_args& a, const GdnWork& w, hipStream_t s) {
    using T = std::conditional_t<NT == 1, uint16_t, float>;
    const int es = NT == 1 ? 2 : 4, slices = (a.dim_v + 15) / 16;
    if (a.rows > 0)
        gdn_chunk_kernel<KS, NT, kDelta><<<dim3((unsigned)(w.n_chunks * a.heads_v)), 256, 0, s>>>(
            a, w.n_chunks, rows_of_16(a.q, a.q_row, a.dim_k, es), rows_of_16(a.k, a.k_row, a.dim_k, es));
    gdn_scan_kernel<KS, NT, kDelta, T>
        <<<dim3((unsigned)((size_t)a.n_seq * a.heads_v * slices)), 256, 0, s>>>(a, w.n_chunks, slices);
    return hipGetLastError();
}

template <int KS>
hipError_t launch_prompt_of(const gdn_dev_args& a, const GdnWork& w, hipStream_t s) {
    if (a.dtype == QWEN_BF16)
        return a.beta ? launch_prompt<KS, 1, true>(a, w, s) : launch_prompt<KS, 1, false>(a, w, s);
    return a.beta ? launch_prompt<KS, 3, true>(a, w, s) : launch_prompt<KS, 3, false>(a, w, s);
}

template <int NI, int G>
hipError_t launch_step(const gdn_dev_args& a, hipStream_t s) {
    const int groups = a.dim_v / 4;
    const size_t units = (size_t)a.n_seq * a.heads_v * ((groups + G - 1) / G);
    const dim3 grid((unsigned)((units + 3) / 4));
    if (a.dtype == QWEN_BF16)
        gdn_step_kernel<NI, G, uint16_t><<<grid, 256, 0, s>>>(a, groups);
    else
        gdn_step_kernel<NI, G, float><<<grid, 256, 0, s>>>(a, groups);
    return hipGetLastError();
}

}  // namespace

hipError_t gdn_launch_prompt(const gdn_dev_args& a, const GdnWork& w, hipStream_t s) {
    switch (w.ks) {
        case 1: return launch_prompt_of<1>(a, w, s);
        case 2: return launch_prompt_of<2>(a, w, s);
        case 4: return launch_prompt_of<4>(a, w, s);
        default: return launch_prompt_of<8>(a, w, s);
    }
}

hipError_t gdn_launch_step(const gdn_dev_args& a, hipStream_t s) {
    if (a.dim_k <= 64) return launch_step<1, 4>(a, s);
    if (a.dim_k <= 128) return launch_step<2, 4>(a, s);
    return launch_step<4, 4>(a, s);
}
