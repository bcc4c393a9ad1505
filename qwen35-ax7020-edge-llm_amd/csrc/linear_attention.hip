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
// side by side; gdn_scan_kernel takes the state from chunk to chunk, 16 or 32 of
// a head's value columns in a workgroup (the columns do not mix).
//
// Arithmetic: every product of the scan, and K K^T and Q K^T, run on the bf16
// matrix cores, a float32 operand as the sum of three bf16 terms (bf16_terms.h),
// a product of two such sums as six pairs of terms: 2^-23.  What only a bf16 output
// sees (S0 in Q S0, P and U in P U) has two terms, all pairs taken: 2^-16 and 2^-15,
// against the output's own 2^-8.
#include "bf16_terms.h"
#include "linear_attention.h"

namespace {

using s16x4 = __attribute__((ext_vector_type(4))) short;

constexpr int C = GDN_CHUNK;

// Elements i .. i + 7 of a row as terms, zeros for those from dim on.  full: the whole padded row is
// there, 16-byte aligned.
template <int NT>
__device__ __forceinline__ void load_terms(const void* row, int i, int dim, bool full, u32x4 (&t)[NT]) {
    if constexpr (NT == 1) {
        const uint16_t* p = static_cast<const uint16_t*>(row);
        if (full) {
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
        if (full) {
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

// As bf16 terms: from bf16's largest value and half a step on the first one is infinite.
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < 0x1.ffp127f; }

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

// The place of sequence s's first chunk in the work buffer (GdnWork).
__device__ __forceinline__ int first_place(int first, int s, int short_to) {
    return short_to < 0 ? first / C + s : first / GDN_SHORT;
}

// The sequence with the r-th most chunks (of equal ones the first first) and its rows, where a wavefront holds
// all lengths and the workgroups are more than the compute units; else sequence r.  Every lane of the wavefront:
// bit by bit from the top, the lanes that the r-th may be.
__device__ __forceinline__ int by_length(const gdn_dev_args& a, int r, int& first, int& n) {
    if (!a.starts || a.n_seq > 64 || gridDim.x <= 256) {
        span(a, r, first, n);
        return r;
    }
    const int lane = threadIdx.x & 63;
    int my_first = 0, my_n = 0;
    if (lane < a.n_seq) span(a, lane, my_first, my_n);
    const uint32_t chunks = (my_n + C - 1) / C;
    uint64_t in = a.n_seq == 64 ? ~0ull : (1ull << a.n_seq) - 1;
    for (int b = 31 - __builtin_clz(a.rows / C + 1); b >= 0; --b) {
        const uint64_t ones = __ballot(chunks >> b & 1) & in;
        const int c = __popcll(ones);
        if (r < c) {
            in = ones;
        } else {
            r -= c;
            in &= ~ones;
        }
    }
    const int seq = __ffsll((unsigned long long)__ballot((in >> lane & 1) && __popcll(in & ((1ull << lane) - 1)) == r)) - 1;
    first = __builtin_amdgcn_readlane(my_first, seq);
    n = __builtin_amdgcn_readlane(my_n, seq);
    return seq;
}

// The slot of sequence s, or -1 where it is skipped.  Every lane of the workgroup.
__device__ __forceinline__ int slot_of(const gdn_dev_args& a, int s) {
    if (!a.slots) return s < a.n_slots ? s : -1;
    const int slot = a.slots[s];
    if (slot < 0 || slot >= a.n_slots) return -1;
    int twice = 0;
#pragma unroll 8
    for (int i = threadIdx.x & 63; i < s; i += 64) twice |= a.slots[i] == slot;
    return __any(twice) ? -1 : slot;
}

// Zeros in out's rows first .. end - 1, columns j0 .. j0 + n - 1 of head hv: thread i of threads.
template <class T>
__device__ __forceinline__ void zero_rows(const gdn_dev_args& a, int first, int end, int hv, int j0, int n, int i, int threads) {
    for (size_t u = i; first < end && u < (size_t)(end - first) * n; u += threads) {
        const int j = j0 + (int)(u % n);
        if (j < a.dim_v)
            static_cast<T*>(a.out)[(int64_t)(first + (int)(u / n)) * a.out_row + (int64_t)hv * a.dim_v + j] = T(0);
    }
}
// zero_rest: the rows in front of the first sequence and behind the last, by whoever has that one.
template <class T>
__device__ __forceinline__ void zero_ends(const gdn_dev_args& a, int seq, int first, int len, int hv, int j0, int n, int i,
                                          int threads) {
    if (seq == 0) zero_rows<T>(a, 0, first, hv, j0, n, i, threads);
    if (seq == a.n_seq - 1) zero_rows<T>(a, first + len, a.rows, hv, j0, n, i, threads);
}

// The byte offsets of the work buffer's parts for one chunk.
struct Places {
    char *k, *q;                 // key head: the image of a KTile, Q fragments [4 row tiles][ks][nt] KiB
    char *t, *p;                 // triangular fragments: tile(rt, ts) of 6, x 3 or no terms
    float *up, *down, *last;     // 2^g, 2^(g_C - g), 2^(g_C)
};
template <int KS, int NT, int NO>
struct Layout {
    static constexpr size_t kKey = (size_t)2 * 4 * KS * NT * 1024, kTri = (size_t)(18 + 6 * NO) * 1024 + 1024;
    static __device__ Places at(const gdn_dev_args& a, size_t n_chunks, size_t chunk, int hk, int hv) {
        char* base = static_cast<char*>(a.work);
        Places w;
        w.k = base + (chunk * a.heads_k + hk) * kKey;
        w.q = w.k + kKey / 2;
        char* tri = base + n_chunks * a.heads_k * kKey + (chunk * a.heads_v + hv) * kTri;
        w.t = tri;
        w.p = tri + 18 * 1024;
        w.up = reinterpret_cast<float*>(tri + (18 + 6 * NO) * 1024);
        w.down = w.up + C;
        w.last = w.down + C;
        return w;
    }
    static __device__ void next(const gdn_dev_args& a, Places& w) {
        const size_t key = a.heads_k * kKey, tri = a.heads_v * kTri;
        w.k += key;
        w.q += key;
        w.t += tri;
        w.p += tri;
        w.up += tri / 4;
        w.down += tri / 4;
        w.last += tri / 4;
    }
};

// A chunk's K in LDS: a row of 64 KS bytes a token, [term][token], its 16-byte parts at positions
// part ^ mix(token), so that neither eight consecutive elements of 16 tokens (K as a left operand) nor
// four of four tokens (ds_read_tr16_b64: K^T) meet in a bank.
template <int KS, int NT>
struct KTile {
    static constexpr int kRow = 64 * KS, kTerm = C * kRow, kBytes = NT * kTerm;
    static __device__ __forceinline__ int mix(int t) {
        if (KS >= 4) return (t & 3) << 2 | (t >> 2 & 3);
        if (KS == 2) return (t & 1) << 2 | (t >> 1 & 3);
        return t >> 2 & 3;
    }
    static __device__ __forceinline__ int part(int t, int c) { return t * kRow + (c ^ mix(t)) * 16; }
    // K of tokens 16 w .., step s
    static __device__ __forceinline__ void rows(const char* k, int w, int s, int lane, u32x4 (&f)[NT]) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
            f[t] = *reinterpret_cast<const u32x4*>(k + t * kTerm + part(16 * w + (lane & 15), 4 * s + (lane >> 4)));
    }
    // K^T: the state's rows of `tile`, tokens 32 ts ..
    static __device__ __forceinline__ void columns(const char* k, int tile, int ts, int lane, u32x4 (&f)[NT]) {
        using lds_s16x4 = __attribute__((address_space(3))) s16x4;
        const int g = lane >> 4, c = lane & 15;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            u32x2 v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
                v[h] = __builtin_bit_cast(
                    u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                               (lds_s16x4*)(k + t * kTerm + part(32 * ts + 16 * h + 4 * g + c / 4, 4 * (tile / 2) + c % 4) +
                                            8 * (tile % 2))));
            f[t] = u32x4{v[0][0], v[0][1], v[1][0], v[1][1]};
        }
    }
};
// Tiles of a lower triangle of 4 x 2 tiles of 16 x 32: row tiles 0 and 1 have only
// step 0.
__device__ __forceinline__ constexpr int tri_tile(int rt, int ts) { return rt < 2 ? rt : 2 + (rt - 2) * 2 + ts; }

// A product's result has four consecutive rows of a column in a lane; as the next
// product's right operand it stays in that lane, if the next product sums in this order:
// place e of lane group g is row 4 g + e of the first tile of a pair (e < 4) or 4 g + e - 4
// of the second.  Tokens are in tiles of 16 in order; a pair of the state's tiles holds
// rows 32 s + 8 g + e of dim_k, so that K and Q are eight consecutive elements a lane.
__device__ __forceinline__ int state_row(int tile, int g) { return 32 * (tile / 2) + 8 * g + 4 * (tile % 2); }

__device__ __forceinline__ void sync_lds() {
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): loads from memory stay in flight
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// ---- chunks -------------------------------------------------------------------------
// One chunk of one value head; wavefront w has tokens 16 w .. 16 w + 15.  What it writes is
// in the order in which gdn_scan_kernel loads it.  direct: that kernel takes K and Q from
// the inputs.  Memory bounds it: K and Q in, 31 KiB of T and P out; at 16,384 tokens of 16
// heads of 128 in bf16 62 us, 4.2 TB/s.  Inverting (I + L) one column a lane over all 64 rows
// left three wavefronts idle and took 145; in blocks of 16 all four work.
template <int KS, int NT, bool kDelta>
__global__ __launch_bounds__(256) void gdn_chunk_kernel(gdn_dev_args a, size_t n_chunks, int short_to, int full_q,
                                                        int full_k, int direct) {
    constexpr int NO = NT == 1 ? 2 : 3, KP = 32 * KS + 8;
    __shared__ __attribute__((aligned(16))) uint16_t ksh[NT][C][KP];  // K, a row a token
    __shared__ __attribute__((aligned(16))) float lsh[kDelta ? C : 1][C + 4];
    __shared__ double gsh[C];
    __shared__ float bsh[C];
    __shared__ uint32_t bad_sh[4];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15,
              grp = lane >> 4;
    const size_t chunk = blockIdx.x / a.heads_v;
    const int hv = blockIdx.x % a.heads_v, reach = a.heads_v / a.heads_k, hk = hv / reach;

    // the sequence: the last s whose first place is up to `chunk`
    int seq = 0;
    if (a.starts) {
        int lo = 0, hi = a.n_seq;  // key(lo) <= chunk < key(hi)
        while (hi - lo > 1) {
            const int step = (hi - lo + 63) / 64, at = lo + (lane + 1) * step;
            const bool le = at < hi && (size_t)first_place(min(max(a.starts[at], 0), a.rows), at, short_to) <= chunk;
            const int below = __popcll(__ballot(le));
            const int nlo = lo + below * step;
            hi = min(hi, lo + (below + 1) * step);
            lo = min(nlo, hi - 1);
        }
        seq = lo;
    }
    int first, len;
    span(a, seq, first, len);
    if (len <= short_to) return;
    const long c = (long)chunk - first_place(first, seq, short_to);
    if (c < 0 || c * C >= len) return;
    const int row0 = first + (int)c * C, n = min(C, len - (int)c * C);
    const Places at = Layout<KS, NT, NO>::at(a, n_chunks, chunk, hk, hv);
    const bool keys = hv % reach == 0;  // this workgroup leaves the key head's fragments too

    // K and Q rows of tile w as operand fragments
    u32x4 kf[KS][NT], qf[KS][NT];
    const int r = 16 * w + col;
    const int es = NT == 1 ? 2 : 4;
    // (rows behind the end: the last one, then zeros)
    const int64_t row = row0 + min(r, n - 1);
    const char* krow = static_cast<const char*>(a.k) + (row * a.k_row + (int64_t)hk * a.dim_k) * es;
    const char* qrow = static_cast<const char*>(a.q) + (row * a.q_row + (int64_t)hk * a.dim_k) * es;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        load_terms(krow, 32 * s + 8 * grp, a.dim_k, full_k, kf[s]);
        load_terms(qrow, 32 * s + 8 * grp, a.dim_k, full_q, qf[s]);
    }
    // A token whose k, decay or beta is not finite: a matrix product takes 0 x NaN to the tokens before it too, so it
    // goes in as zeros here, and the first such token's 2^g and 2^(g_C - g) are NaN, which gdn_scan_kernel meets.
    using u16x2 = __attribute__((ext_vector_type(2))) unsigned short;
    u16x2 most = {0, 0};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, kf[s][0][j] & 0x7fff7fffu));
    const uint64_t groups = __ballot(most[0] >= 0x7f80 || most[1] >= 0x7f80);
    uint32_t bad_rows = (uint32_t)groups | (uint32_t)(groups >> 32);
    bad_rows = (bad_rows | bad_rows >> 16) & 0xffff;
    const bool bad_k = bad_rows >> col & 1;
    if (lane == 0) bad_sh[w] = bad_rows;
    uint64_t bad_gates = 0;
    if (w == 0) {
        // g in double: differences of large sums stay exact to a float32.  A decay of 0
        // counts as 2^-16384, which no product brings back.
        const int64_t grow = (int64_t)(row0 + min(lane, n - 1)) * a.gate_row + hv;
        const float al = a.alpha[grow], be = kDelta ? a.beta[grow] : 0.0f;
        double g = lane >= n ? 0.0 : al == 0.0f ? -16384.0 : log2((double)al);
        const bool bad_al = !(fabs(g) < __builtin_inf());
        if (bad_al) g = 0.0;
        bad_gates = __ballot(bad_al || !finite(be));
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double o = __shfl_up(g, d);
            if (lane >= d) g += o;
        }
        const double gc = __shfl(g, 63);
        gsh[lane] = g;
        bsh[lane] = lane < n && finite(be) ? be : 0.0f;
        at.up[lane] = exp2_of(g);
        at.down[lane] = exp2_of(gc - g);
        if (lane == 0) at.last[0] = exp2_of(gc);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (r >= n) qf[s][t] = u32x4{0, 0, 0, 0};
            if (r >= n || bad_k) kf[s][t] = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4*>(&ksh[t][r][32 * s + 8 * grp]) = kf[s][t];
            const int f = ((w * KS + s) * NT + t) * 64 + lane;
            if (keys && !direct) {
                using K = KTile<KS, NT>;
                *reinterpret_cast<u32x4*>(at.k + t * K::kTerm + K::part(r, 4 * s + grp)) = kf[s][t];
                reinterpret_cast<u32x4*>(at.q)[f] = qf[s][t];
            }
        }
    sync_lds();

    // K K^T and K Q^T, the tiles that hold a j <= i: lane has token i = r, four tokens j
    f32x4 pt[4];
    const double gi = gsh[r];
    const float bi = bsh[r];
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) {
        pt[jt] = f32x4{0, 0, 0, 0};
        if (jt > w) continue;
        f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            u32x4 b[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
                b[t] = *reinterpret_cast<const u32x4*>(&ksh[t][16 * jt + col][32 * s + 8 * grp]);
            if (kDelta) kk = mfma_terms<NT, NT, 3>(b, kf[s], kk);
            qk = mfma_terms<NT, NT, 3>(b, qf[s], qk);
        }
        f32x4 l;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = 16 * jt + 4 * grp + e;
            const float d = r >= j ? exp2_of(gi - gsh[j]) : 0.0f;
            pt[jt][e] = r >= j ? qk[e] * d : 0.0f;
            l[e] = r > j ? bi * d * kk[e] : 0.0f;
        }
        if constexpr (kDelta) *reinterpret_cast<f32x4*>(&lsh[r][16 * jt + 4 * grp]) = l;
    }
#pragma unroll
    for (int ts = 0; ts < 2; ++ts) {
        if (ts == 1 && w < 2) break;
        float x[8];
        u32x4 p[NO];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = pt[2 * ts][e], x[4 + e] = pt[2 * ts + 1][e];
        split8(x, p);
#pragma unroll
        for (int m = 0; m < NO; ++m) reinterpret_cast<u32x4*>(at.p)[(tri_tile(w, ts) * NO + m) * 64 + lane] = p[m];
    }
    if (w == 0) {  // (which has the least to do up to here)
        uint64_t bad = bad_gates | bad_sh[0] | (uint64_t)bad_sh[1] << 16 | (uint64_t)bad_sh[2] << 32 | (uint64_t)bad_sh[3] << 48;
        if (n < C) bad &= (1ull << n) - 1;
        if (bad && lane == __builtin_ctzll(bad)) at.up[lane] = at.down[lane] = __builtin_nanf("");
    }
    if constexpr (kDelta) {
        // X = (I + L)^-1 in blocks of 16.  The blocks on the diagonal by substitution, a column a
        // lane (each of the four lane groups does the same); X_ij = -X_ii sum_k L_ik X_kj below, in
        // float32, column j's blocks by wavefront j.
        sync_lds();
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s0 = i == col ? 1.0f : 0.0f, s1 = 0.0f;
#pragma unroll
            for (int j = 0; j < i; j += 4) {
                const f32x4 l = *reinterpret_cast<const f32x4*>(&lsh[16 * w + i][16 * w + j]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (j + e < i) (e % 2 ? s1 : s0) = __builtin_fmaf(-l[e], x[j + e], e % 2 ? s1 : s0);
            }
            x[i] = s0 + s1;
        }
        f32x4 X[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) X[k] = f32x4{0, 0, 0, 0};
        f32x4 d;
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = grp == 0 ? x[e] : grp == 1 ? x[4 + e] : grp == 2 ? x[8 + e] : x[12 + e];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k == w) X[k] = d;
#pragma unroll
        for (int e = 0; e < 4; ++e) lsh[16 * w + 4 * grp + e][16 * w + col] = d[e];
        sync_lds();
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            if (i <= w) continue;
            f32x4 sum = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < i; ++k) {
                if (k < w) continue;
                const f32x4 l = *reinterpret_cast<const f32x4*>(&lsh[16 * i + col][16 * k + 4 * grp]);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(-l[e], X[k][e], sum, 0, 0, 0);
            }
            const f32x4 inv = *reinterpret_cast<const f32x4*>(&lsh[16 * i + col][16 * i + 4 * grp]);
#pragma unroll
            for (int e = 0; e < 4; ++e) X[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(inv[e], sum[e], X[i], 0, 0, 0);
        }
        sync_lds();
        const float bj = bsh[16 * w + col];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) lsh[16 * i + 4 * grp + e][16 * w + col] = X[i][e] * bj;
        sync_lds();
        // T = X diag(b)
#pragma unroll
        for (int ts = 0; ts < 2; ++ts) {
            if (ts == 1 && w < 2) break;
            u32x4 t[3];
            float y[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(&lsh[r][32 * ts + 16 * h + 4 * grp]);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[4 * h + e] = v[e];
            }
            split8(y, t);
#pragma unroll
            for (int m = 0; m < 3; ++m)
                reinterpret_cast<u32x4*>(at.t)[(tri_tile(w, ts) * 3 + m) * 64 + lane] = t[m];
        }
    }
}

// ---- the state from chunk to chunk --------------------------------------------------
// NC x 16 value columns of one head of one sequence in nine wavefronts.  The first four carry the
// state: wavefront w has tokens 16 w .. of each chunk, and TPW tiles of 16 of the state's rows in its
// accumulators.  The next four follow with the outputs, so that a chunk's chain of dependent steps is
// K S0, T R, K^T U and three barriers.  The last brings the next chunk's K to LDS and, with inputs that
// it can copy from as they are (kDirect), V, T and the decays: a load instruction in the chain costs
// it some 30 cycles.  The state, the right side and U pass between wavefronts as bf16 terms in LDS, lane by
// lane (see state_row).  Other fragments of the next chunk are loaded into each register as soon as it
// is free.
// The chain bounds it: at one sequence of 16,384 tokens, 16 heads of 128, bf16, 415 us, 1.6 us (3,600 cycles)
// a chunk, of which the first four wavefronts work 1,100, 720 and 980 cycles between barriers and wait
// for the others and for skew the rest; at 24 float32 prompts of 9,001 tokens in all 181 us.
// With four wavefronts that do everything and load for themselves the first took 1,190 us.
template <int KS, int NT, int NC, bool kDelta, bool kDirect, class T>
__global__ __launch_bounds__(576, 1) void gdn_scan_kernel(gdn_dev_args a, size_t n_chunks, int slices,
                                                            int short_to) {
    constexpr int NO = NT == 1 ? 2 : 3;
    constexpr int TPW = KS >= 2 ? KS / 2 : 1;
    // chunks in LDS: three where they fit (their copies are on the way for a whole chunk), one where two
    // don't; T always two
    constexpr int kBufs = kDirect && KS <= 4 ? 3 : KS * NT <= 12 ? 2 : 1;
    using L = Layout<KS, NT, NO>;
    using K = KTile<KS, NT>;
    static_assert(!kDirect || kBufs >= 2, "kDirect copies a chunk ahead");
    __shared__ __attribute__((aligned(1024))) char ksh[kBufs][K::kBytes];
    constexpr int kVRow = 32 * NC;  // bytes of a token's V
    __shared__ __attribute__((aligned(1024))) char vsh[kDirect ? kBufs : 1][kDirect ? C * kVRow : 16];
    __shared__ __attribute__((aligned(1024))) char tsh[kDirect ? 2 : 1][kDirect && kDelta ? 18 * 1024 : 16];
    __shared__ __attribute__((aligned(1024))) float gsh[kDirect ? kBufs : 1][kDirect ? 256 : 4];
    // [columns][pair of tiles][term][lane][tile of the pair]: an operand is one 16-byte read
    __shared__ u32x4 ssh[NC][KS][3][64];
    __shared__ u32x4 rsh[kDelta ? NC : 1][kDelta ? 2 : 1][3][64];
    __shared__ u32x4 ush[NC][2][NO][64];
    __shared__ u32x4 dsh[NC][2][3][64];
    // the output wavefronts' tiles on their way out, from a chunk's last barrier to the next one's first: R is idle then
    using OutTile = T[16][16];
    __shared__ __attribute__((aligned(16))) OutTile own_osh[kDelta ? 1 : 4];
    static_assert(!kDelta || sizeof(rsh) >= 4 * sizeof(OutTile), "R's place holds them");
    OutTile* const osh = kDelta ? reinterpret_cast<OutTile*>(&rsh[0][0][0][0]) : own_osh;
    // A column's first token whose right side (without the delta rule: v) is not finite, counted in the sequence: its
    // part of R or U is 0, for the sake of the tokens before it; outputs from it on are NaN, and so is the state.
    __shared__ int bad_sh[NC][16], first_bad;  // of each column, of any
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3,
              col = lane & 15, grp = lane >> 4;
    // the longest sequences first, so that none is begun when the others are nearly done (24 of 9001
    // tokens in float32: 251 us, in their order 312);
    // a head's slices a multiple of the heads apart: with 8 | heads on one XCD, whose
    // L2 then holds the fragments that they share
    const int each = a.heads_v * slices, part = blockIdx.x % each;
    int first, len;
    const int seq = by_length(a, blockIdx.x / each, first, len), hv = part % a.heads_v, slice = part / a.heads_v;
    const int hk = hv / (a.heads_v / a.heads_k);
    if (len <= short_to) return;
    const int slot = slot_of(a, seq);
    if (a.zero_rest) {
        zero_ends<T>(a, seq, first, len, hv, 16 * NC * slice, 16 * NC, threadIdx.x, 576);
        if (slot < 0) zero_rows<T>(a, first, first + len, hv, 16 * NC * slice, 16 * NC, threadIdx.x, 576);
    }
    if (slot < 0) return;
    const int j0 = 16 * NC * slice + col;  // first value column
    const int nc = (len + C - 1) / C;
    Places at = L::at(a, n_chunks, first_place(first, seq, short_to), hk, hv);
    auto half = [&](u32x4(&x)[64], int tile) -> u32x2& { return reinterpret_cast<u32x2*>(&x[lane])[tile & 1]; };

    using lds_void = __attribute__((address_space(3))) void;
    using global_void = const __attribute__((address_space(1))) void;
    if (wave == 8) {
        // K, V and the decays of chunk c are kRest copies of 1 KiB, T kT
        constexpr int kK = K::kBytes / 1024, kV = kDirect ? 2 * NC : 0, kRest = kK + (kDirect ? kV + 1 : 0);
        constexpr int kT = kDirect && kDelta ? 18 : 0;
        constexpr int kParts = K::kRow / 16, kKRows = 64 / kParts, kVRows = 32 / NC;  // rows that a copy holds
        constexpr int kMixes = KS == 4 ? 4 : K::kBytes / 1024;  // copies whose rows are mixed differently
        const uint16_t* kp = static_cast<const uint16_t*>(a.k) + first * a.k_row + (int64_t)hk * (32 * KS);
        const uint16_t* vp = static_cast<const uint16_t*>(a.v) + first * a.v_row + (int64_t)hv * a.dim_v;
        const int vcol = min(16 * NC * slice + 8 * (lane % (2 * NC)), a.dim_v - 8);
        auto kcol = [&](int i) { return ((lane % kParts) ^ K::mix(i * kKRows + lane / kParts)) * 8; };
        // a lane's offset from a copy's first row, in bytes: the rest of an address is the same for all lanes
        uint32_t koff[kMixes];
#pragma unroll
        for (int i = 0; i < kMixes; ++i) koff[i] = (uint32_t)(lane / kParts * a.k_row + kcol(i)) * 2;
        const uint32_t voff = (uint32_t)(lane / (2 * NC) * a.v_row + vcol) * 2;
        // (where the chunk is not whole, the last token for those past the end: U is zero there)
        auto copy_as = [&](int c, const Places& p, auto from, auto to, auto whole) {
#pragma unroll
            for (int i = decltype(from)::value; i < decltype(to)::value; ++i) {
                const char* src;
                char* dst = ksh[c % kBufs] + i * 1024;
                if constexpr (kDirect) {
                    const int v = i - kK;
                    if (i < kK) {
                        src = reinterpret_cast<const char*>(kp + (int64_t)(c * C + i * kKRows) * a.k_row) + koff[i % kMixes];
                        if (!decltype(whole)::value)
                            src = reinterpret_cast<const char*>(
                                kp + min(c * C + i * kKRows + lane / kParts, len - 1) * a.k_row + kcol(i));
                    } else if (i < kK + kV) {
                        src = reinterpret_cast<const char*>(vp + (int64_t)(c * C + v * kVRows) * a.v_row) + voff;
                        if (!decltype(whole)::value)
                            src = reinterpret_cast<const char*>(
                                vp + min(c * C + v * kVRows + lane / (2 * NC), len - 1) * a.v_row + vcol);
                        dst = vsh[c % kBufs] + v * 1024;
                    } else {
                        src = reinterpret_cast<const char*>(p.up) + (uint32_t)lane * 16;
                        dst = reinterpret_cast<char*>(gsh[c % kBufs]);
                    }
                } else {
                    src = p.k + i * 1024 + (uint32_t)lane * 16;
                }
                __builtin_amdgcn_global_load_lds((global_void*)src, (lds_void*)dst, 16, 0, 0);
            }
        };
        auto copy = [&](int c, const Places& p, auto from, auto to) {
            if (c * C + C <= len || !kDirect)
                copy_as(c, p, from, to, std::true_type());
            else
                copy_as(c, p, from, to, std::false_type());
        };
        auto copy_t = [&](int c, const Places& p) {
#pragma unroll
            for (int i = 0; i < kT; ++i)
                __builtin_amdgcn_global_load_lds((global_void*)(p.t + i * 1024 + lane * 16),
                                                 (lds_void*)(tsh[c % 2] + i * 1024), 16, 0, 0);
        };
        using Zero = std::integral_constant<int, 0>;
        using Half = std::integral_constant<int, kBufs == 3 && kDelta ? kRest / 6 : 0>;
        using All = std::integral_constant<int, kRest>;
        static_assert(kBufs < 3 || kRest < 64, "vmcnt has six bits");
        Places at2 = at;  // one chunk behind `at`
        if (nc > 0) {
            copy_t(0, at);
            copy(0, at, Zero(), All());
            L::next(a, at);
            if (kBufs == 3 && nc > 1) copy(1, at, Zero(), All());
            if (kBufs == 3) L::next(a, at);
            L::next(a, at2);
        }
        for (int c = 0; c < nc; ++c) {
            // chunk c has to be there, T of it too; of the next one, copied while c - 1 was worked on, not all
            if (kBufs == 3 && c + 1 < nc)
                __builtin_amdgcn_s_waitcnt(0x0F70 | (kRest & 15) | (kRest >> 4) << 14);  // vmcnt(kRest)
            else
                __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
            sync_lds();
            // spread over the chunk, as Q and P are: a load takes the compute unit some 40 cycles, and a
            // wavefront that waits to issue one is late at the barrier
            const bool more = kBufs >= 2 && c + kBufs - 1 < nc;
            if (c + 1 < nc) copy_t(c + 1, at2);
            if (kBufs == 2 && more) copy(c + 1, at, Zero(), All());
            if (kDelta) {
                sync_lds();
                if (kBufs == 3 && more) copy(c + 2, at, Zero(), Half());
            }
            sync_lds();
            if (kBufs == 3 && more) copy(c + 2, at, Half(), All());
            if (kBufs == 1) {
                sync_lds();
                if (c + 1 < nc) copy(c + 1, at, Zero(), All());
            }
            L::next(a, at);
            L::next(a, at2);
        }
        return;
    }

    if (wave >= 4) {
        // O = scale (2^g Q S0 + P U), Q and P loaded two chunks ahead (float32: one, for the registers):
        // nobody is to wait for these wavefronts at a barrier
        constexpr int kSets = NT == 1 ? 2 : 1;
        struct Ahead {
            u32x4 q[KS][NT], p[2][NO];
            f32x4 up;
        } set[kSets];
        const uint16_t* qp = nullptr;
        int loaded = 0;
        auto load_q = [&](Ahead& x) {
            const int c = min(loaded, nc - 1);  // behind the last chunk its own again
            if constexpr (kDirect) {
                if (loaded == 0 || loaded >= nc - 1)
                    qp = static_cast<const uint16_t*>(a.q) + (first + min(c * C + 16 * w + col, len - 1)) * a.q_row +
                         (int64_t)hk * (32 * KS) + 8 * grp;
                else
                    qp += C * a.q_row;
#pragma unroll
                for (int s = 0; s < KS; ++s) x.q[s][0] = *reinterpret_cast<const u32x4*>(qp + 32 * s);
            } else {
                const u32x4* p = reinterpret_cast<const u32x4*>(at.q) + w * KS * NT * 64 + lane;
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int t = 0; t < NT; ++t) x.q[s][t] = p[(s * NT + t) * 64];
            }
        };
        auto load_p = [&](Ahead& x) {
            const u32x4* p = reinterpret_cast<const u32x4*>(at.p) + tri_tile(w, 0) * NO * 64 + lane;
#pragma unroll
            for (int m = 0; m < NO; ++m) x.p[0][m] = p[m * 64];
            if (w >= 2)
#pragma unroll
                for (int m = 0; m < NO; ++m) x.p[1][m] = p[(NO + m) * 64];
            if (!kDirect) x.up = *reinterpret_cast<const f32x4*>(at.up + 16 * w + 4 * grp);
            if (++loaded < nc) L::next(a, at);
        };
#pragma unroll
        for (int h = 0; h < kSets; ++h) {
#pragma unroll
            for (int m = 0; m < NO; ++m) set[h].p[1][m] = u32x4{0, 0, 0, 0};
            if (nc > 0) {
                load_q(set[h]);
                load_p(set[h]);
            }
        }
        // a lane's part of a tile of 16 tokens x 16 columns as it is stored: EL elements of a token's row
        constexpr int EL = 16 / (int)sizeof(T) / (NT == 1 ? 2 : 1), kLanes = 16 / EL;
        static_assert(64 / kLanes == 16, "a tile is one store of a wavefront");
        const int token = 16 * w + lane / kLanes, part = lane % kLanes * EL;
        T* out = static_cast<T*>(a.out) + (first + token) * a.out_row + (int64_t)hv * a.dim_v + 16 * NC * slice + part;
        const bool wide = ((uintptr_t)a.out | (uintptr_t)(a.out_row * sizeof(T)) | (uintptr_t)(a.dim_v * sizeof(T))) %
                              (EL * sizeof(T)) == 0;
        auto chunk = [&](int c, Ahead& x, Ahead& other) {
            sync_lds();
            if (kSets == 2 && c > 0) load_p(other);
            f32x4 o[NC];
#pragma unroll
            for (int y = 0; y < NC; ++y) o[y] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int y = 0; y < NC; ++y) {
                    u32x4 b[NO];
#pragma unroll
                    for (int m = 0; m < NO; ++m) b[m] = ssh[y][s][m][lane];
                    o[y] = mfma_terms<NT, NO, NO>(x.q[s], b, o[y]);
                }
            const f32x4 up = kDirect ? *reinterpret_cast<const f32x4*>(&gsh[c % kBufs][kDirect ? 16 * w + 4 * grp : 0]) : x.up;
#pragma unroll
            for (int y = 0; y < NC; ++y) o[y] *= up;
            if (kDelta) sync_lds();
            load_q(x);
            sync_lds();
            const bool some_bad = __any(first_bad < c * C + C);
#pragma unroll
            for (int ts = 0; ts < 2; ++ts)
#pragma unroll
                for (int y = 0; y < NC; ++y) {
                    u32x4 b[NO];
#pragma unroll
                    for (int m = 0; m < NO; ++m) b[m] = ush[y][ts][m][lane];
                    o[y] = mfma_terms<NO, NO, 3>(x.p[ts], b, o[y]);
                }
            if (kSets == 1) load_p(x);
#pragma unroll
            for (int y = 0; y < NC; ++y) o[y] *= a.scale;
            if (__builtin_expect(some_bad, 0))
#pragma unroll
                for (int y = 0; y < NC; ++y)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c * C + 16 * w + 4 * grp + e >= bad_sh[y][col]) o[y][e] = __builtin_nanf("");
#pragma unroll
            for (int y = 0; y < NC; ++y) {
                // the tile row by row (nobody else's part of LDS, and in order within a wavefront)
#pragma unroll
                for (int e = 0; e < 4; ++e) osh[w][4 * grp + e][col] = from_float<T>(o[y][e]);
                struct alignas(EL * sizeof(T)) Part {
                    T x[EL];
                };
                asm volatile("" ::: "memory");
                const Part v = *reinterpret_cast<const Part*>(&osh[w][lane / kLanes][part]);
                asm volatile("" ::: "memory");
                T* to = out + 16 * y;
                const int left = a.dim_v - (16 * NC * slice + 16 * y + part);
                if (c * C + token < len) {
                    if (wide && left >= EL) {
                        *reinterpret_cast<Part*>(to) = v;
                    } else {
#pragma unroll
                        for (int e = 0; e < EL; ++e)
                            if (e < left) to[e] = v.x[e];
                    }
                }
            }
            out += C * a.out_row;
            if (kBufs == 1) sync_lds();
        };
        for (int c = 0; c < nc; c += kSets) {
            chunk(c, set[0], set[kSets - 1]);
            if (kSets == 2 && c + 1 < nc) chunk(c + 1, set[kSets - 1], set[0]);
        }
        return;
    }

    // the state: lane holds rows state_row(tile, grp) .. + 3 of column j0 + 16 x
    const size_t head_state = ((size_t)slot * a.heads_v + hv) * a.dim_k * a.dim_v;
    // (with one step along dim_k two of the wavefronts have no tile; else the compiler has to know that all do: it leaves
    // too few wait states between a matrix product, a branch around the next one, and the first use of the result)
    auto has_tile = [&](int t) { return KS >= 2 || w * TPW + t < 2 * KS; };
    f32x4 S[NC][TPW];
    auto each_state = [&](auto&& f) {
#pragma unroll
        for (int x = 0; x < NC; ++x)
#pragma unroll
            for (int t = 0; t < TPW; ++t) {
                const int i = state_row(w * TPW + t, grp), j = j0 + 16 * x;
                if (j < a.dim_v && i < a.dim_k && has_tile(t))
                    f(S[x][t], head_state + (((size_t)(j / 4) * (a.dim_k / 4) + i / 4) * 4 + j % 4) * 4);
            }
    };
#pragma unroll
    for (int x = 0; x < NC; ++x)
#pragma unroll
        for (int t = 0; t < TPW; ++t) S[x][t] = f32x4{0, 0, 0, 0};
    if (a.state_in)
        each_state([&](f32x4& s, size_t i) { s = *reinterpret_cast<const f32x4*>(a.state_in + i); });
    u32x4 tf[2][3];
    const T* vp[NC][4];
    T v[NC][4];
    f32x4 up, down;
    float last;
    const T* vbase = static_cast<const T*>(a.v) + first * a.v_row + (int64_t)hv * a.dim_v;
    auto load_t = [&] {
        if (!kDelta || kDirect) return;
        const u32x4* p = reinterpret_cast<const u32x4*>(at.t) + tri_tile(w, 0) * 3 * 64 + lane;
#pragma unroll
        for (int m = 0; m < 3; ++m) tf[0][m] = p[m * 64];
        if (w >= 2)
#pragma unroll
            for (int m = 0; m < 3; ++m) tf[1][m] = p[(3 + m) * 64];
    };
    auto load_v = [&](int c) {
        if (kDirect) return;
#pragma unroll
        for (int x = 0; x < NC; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (c == 0 || c == nc - 1)
                    vp[x][e] = vbase + min(c * C + 16 * w + 4 * grp + e, len - 1) * a.v_row +
                               min(j0 + 16 * x, a.dim_v - 1);
                else
                    vp[x][e] += C * a.v_row;
                v[x][e] = *vp[x][e];
            }
        if (kDelta) up = *reinterpret_cast<const f32x4*>(at.up + 16 * w + 4 * grp);
    };
    auto load_down = [&] {
        if (kDirect) return;
        down = *reinterpret_cast<const f32x4*>(at.down + 16 * w + 4 * grp);
        last = at.last[0];
    };
    auto put_state = [&] {
#pragma unroll
        for (int x = 0; x < NC; ++x)
#pragma unroll
            for (int t = 0; t < TPW; ++t)
                if (has_tile(t)) {
                    u32x2 y[3];
                    split4(S[x][t], y);
#pragma unroll
                    for (int m = 0; m < 3; ++m) half(ssh[x][(w * TPW + t) / 2][m], w * TPW + t) = y[m];
                }
    };
#pragma unroll
    for (int m = 0; m < 3; ++m) tf[1][m] = u32x4{0, 0, 0, 0};
    if (nc > 0) {
        load_v(0);
        load_t();
        load_down();
    }
    put_state();
    if (w == 0 && grp == 0)
#pragma unroll
        for (int x = 0; x < NC; ++x) bad_sh[x][col] = first_bad = 0x7fffffff;
    for (int c = 0; c < nc; ++c) {
        const int nx = min(c + 1, nc - 1);
        // Whether any of these is not finite (or their sum is not: then each is looked at).
        auto any_bad = [](const f32x4(&r)[NC]) {
            float sum = 0.0f;
#pragma unroll
            for (int x = 0; x < NC; ++x) sum += (r[x][0] + r[x][1]) + (r[x][2] + r[x][3]);
            return __any(!finite(sum));
        };
        // Zeros for r where `by` is not finite.
        auto leave_out = [&](f32x4(&r)[NC], const f32x4(&by)[NC]) {
#pragma unroll
            for (int x = 0; x < NC; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!finite(by[x][e])) {
                        atomicMin(&bad_sh[x][col], c * C + 16 * w + 4 * grp + e);
                        atomicMin(&first_bad, c * C);
                        r[x][e] = 0.0f;
                    }
        };
        if (c + 1 < nc) L::next(a, at);
        const char* kt = ksh[c % kBufs];
        sync_lds();
        if constexpr (kDirect) {
            const float* g = &gsh[c % kBufs][16 * w + 4 * grp];
            up = *reinterpret_cast<const f32x4*>(g);
            down = *reinterpret_cast<const f32x4*>(g + C);
            last = gsh[c % kBufs][2 * C];
#pragma unroll
            for (int x = 0; x < NC; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[x][e] = *reinterpret_cast<const T*>(vsh[c % kBufs] + (16 * w + 4 * grp + e) * kVRow + (16 * x + col) * 2);
        }
        f32x4 u[NC], into[NC];
        if constexpr (kDelta) {
            // R = V - 2^g K S0
            f32x4 ks[NC][2];
#pragma unroll
            for (int x = 0; x < NC; ++x) ks[x][0] = ks[x][1] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u32x4 kf[NT];
                K::rows(kt, w, s, lane, kf);
#pragma unroll
                for (int x = 0; x < NC; ++x) {
                    u32x4 b[3];
#pragma unroll
                    for (int m = 0; m < 3; ++m) b[m] = ssh[x][s][m][lane];
                    ks[x][s % 2] = mfma_terms<NT, 3, 3>(kf, b, ks[x][s % 2]);
                }
            }
            f32x4 rhs[NC];
            float poison[NC];  // NaN for a column whose state ends here
#pragma unroll
            for (int x = 0; x < NC; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    rhs[x][e] = __builtin_fmaf(-up[e], ks[x][0][e] + ks[x][1][e], to_float<T>(v[x][e]));
            const bool bad = any_bad(rhs);
            if (__builtin_expect(bad, 0)) {
#pragma unroll
                for (int x = 0; x < NC; ++x) {
                    const f32x4 z = rhs[x] * 0.0f;
                    poison[x] = (z[0] + z[1]) + (z[2] + z[3]);
                }
                leave_out(rhs, rhs);
            }
#pragma unroll
            for (int x = 0; x < NC; ++x) {
                u32x2 y[3];
                split4(rhs[x], y);
#pragma unroll
                for (int m = 0; m < 3; ++m) half(rsh[x][w / 2][m], w) = y[m];
            }
            load_v(nx);
            sync_lds();
            f32x4 u2[NC][2];
            u32x4 b[NC][2][3];
#pragma unroll
            for (int x = 0; x < NC; ++x)
#pragma unroll
                for (int ts = 0; ts < 2; ++ts) {
                    u2[x][ts] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int m = 0; m < 3; ++m) b[x][ts][m] = rsh[x][ts][m][lane];
                }
            if constexpr (kDirect) {
                const u32x4* p = reinterpret_cast<const u32x4*>(tsh[c % 2]) + tri_tile(w, 0) * 3 * 64 + lane;
#pragma unroll
                for (int m = 0; m < 3; ++m) tf[0][m] = p[m * 64];
                if (w >= 2)
#pragma unroll
                    for (int m = 0; m < 3; ++m) tf[1][m] = p[(3 + m) * 64];
            }
#pragma unroll
            for (int z = 2; z >= 0; --z)  // the pairs of terms, the chains side by side
#pragma unroll
                for (int y = 0; y <= z; ++y)
#pragma unroll
                    for (int ts = 0; ts < 2; ++ts)
#pragma unroll
                        for (int x = 0; x < NC; ++x) u2[x][ts] = mfma(tf[ts][y], b[x][ts][z - y], u2[x][ts]);
            load_t();
#pragma unroll
            for (int x = 0; x < NC; ++x) {
                u[x] = u2[x][0] + u2[x][1];
                into[x] = u[x] * down;
            }
            if (__builtin_expect(bad, 0))
#pragma unroll
                for (int x = 0; x < NC; ++x) into[x] += poison[x];
        } else {
#pragma unroll
            for (int x = 0; x < NC; ++x) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    u[x][e] = c * C + 16 * w + 4 * grp + e < len ? to_float<T>(v[x][e]) : 0.0f;
                into[x] = u[x] * down;
            }
            // (a bf16 that is finite fits; a float32 may fit only after its decay)
            if (__builtin_expect(any_bad(into) || (NT == 3 && any_bad(u)), 0)) {
                leave_out(u, into);
                if constexpr (NT == 3) {
#pragma unroll
                    for (int x = 0; x < NC; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!finite(u[x][e])) into[x][e] = __builtin_nanf("");
                    leave_out(u, u);
                }
            }
            load_v(nx);
        }
#pragma unroll
        for (int x = 0; x < NC; ++x) {
            u32x2 y[NO], d[3];
            split4(into[x], d);
#pragma unroll
            for (int m = 0; m < 3; ++m) half(dsh[x][w / 2][m], w) = d[m];
            split4(u[x], y);
#pragma unroll
            for (int m = 0; m < NO; ++m) half(ush[x][w / 2][m], w) = y[m];
        }
        const float keep = last;
        load_down();
        sync_lds();
        // S0 <- 2^(g_C) S0 + K^T (2^(g_C - g) U)
#pragma unroll
        for (int x = 0; x < NC; ++x)
#pragma unroll
            for (int t = 0; t < TPW; ++t) S[x][t] *= keep;
#pragma unroll
        for (int ts = 0; ts < 2; ++ts) {
            u32x4 b[NC][3];
#pragma unroll
            for (int x = 0; x < NC; ++x)
#pragma unroll
                for (int m = 0; m < 3; ++m) b[x][m] = dsh[x][ts][m][lane];
#pragma unroll
            for (int t = 0; t < TPW; ++t)
                if (has_tile(t)) {
                    u32x4 kf[NT];
                    K::columns(kt, w * TPW + t, ts, lane, kf);
#pragma unroll
                    for (int x = 0; x < NC; ++x) S[x][t] = mfma_terms<NT, 3, 3>(kf, b[x], S[x][t]);
                }
        }
        put_state();
        if (kBufs == 1) sync_lds();
    }
    each_state([&](const f32x4& s, size_t i) { *reinterpret_cast<f32x4*>(a.state_out + i) = s; });
}

// ---- token by token -------------------------------------------------------------------
// A wavefront as four rows of 16 lanes, two registers at a time: what both have in the lower and in the upper
// half, or in the even and in the odd rows.
struct Pair {
    float a, b;
};
__device__ __forceinline__ Pair swap32(float x, float y) {  // {x's | y's lower half, x's | y's upper half}
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}
__device__ __forceinline__ Pair swap16(float x, float y) {  // {x's | y's even rows, x's | y's odd rows}
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}
template <int N>
__device__ __forceinline__ float turned(float x) {  // by N lanes in each row
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x120 + N, 15, 15, true));
}
// x summed over the 16 lanes of a column (lane % 4): one value in every lane, four the value of its row in each.
__device__ __forceinline__ float over_lanes(const float (&x)[1]) {
    Pair p = swap32(x[0], x[0]);
    p = swap16(p.a + p.b, p.a + p.b);
    float y = p.a + p.b;
    y += turned<8>(y);
    return y + turned<4>(y);
}
__device__ __forceinline__ float over_lanes(const float (&x)[4]) {
    const Pair p = swap32(x[0], x[2]), q = swap32(x[1], x[3]);
    const Pair r = swap16(p.a + p.b, q.a + q.b);
    float y = r.a + r.b;
    y += turned<8>(y);
    return y + turned<4>(y);
}
// The rows' values to every lane.
__device__ __forceinline__ void to_lanes(float x, float (&y)[1]) { y[0] = x; }
__device__ __forceinline__ void to_lanes(float x, float (&y)[4]) {
    const Pair r = swap16(x, x), p = swap32(r.a, r.a), q = swap32(r.b, r.b);
    y[0] = p.a, y[1] = q.a, y[2] = p.b, y[3] = q.b;
}

// With the old state S: u = b (v - a S^T k), out = scale (a S^T q + (k.q) u), S <- a S + k u^T:
// one pass over the state, whose bytes bound one token (256 sequences of 16 heads of 128: 87 us, 6.2 TB/s).  A
// wavefront has G groups of four value columns; lane 4 g + l has rows 4 (g + 16 n) .. + 3 of column l of
// each, one 16-byte load and store each, 1 KiB a wavefront.  The sums over lanes stay in registers, and four
// columns' share their steps (each by itself, through LDS: 95 us; 16 tokens of 64 sequences 73 us, each by itself 92).
// kStream: past the caches, for states that would not be found there again.
// kText: the sequences of up to short_to tokens of a prompt call, the state in registers from token to token
// and kAhead tokens' rows on their way; else one token a sequence.
template <int NI, int G, bool kStream, bool kText, class T>
__global__ __launch_bounds__(256) void gdn_token_kernel(gdn_dev_args a, int groups, int short_to) {
    constexpr int kAhead = kText ? 4 : 1;
    using Four = std::conditional_t<sizeof(T) == 2, u32x2, f32x4>;  // four elements as they are in memory
    const int lane = threadIdx.x & 63, l = lane & 3, g = lane >> 2;
    const int unit = blockIdx.x * 4 + (threadIdx.x >> 6);  // (sequence, head, run of G column groups)
    const int runs = (groups + G - 1) / G, per_seq = a.heads_v * runs;
    const int seq = __builtin_amdgcn_readfirstlane(unit / per_seq);
    if (seq >= a.n_seq) return;
    const int hv = __builtin_amdgcn_readfirstlane(unit % per_seq / runs), jg0 = unit % runs * G;
    int first = seq, len = 1;
    if (kText) {
        span(a, seq, first, len);
        if (len > short_to) return;
    }
    const int slot = slot_of(a, seq);
    if (kText && a.zero_rest) zero_ends<T>(a, seq, first, len, hv, 4 * jg0, 4 * G, lane, 64);
    if (__builtin_expect(slot < 0, 0)) {  // (rare)
        if (a.zero_rest) zero_rows<T>(a, first, first + len, hv, 4 * jg0, 4 * G, lane, 64);
        return;
    }
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
            if (jg0 + m < groups && ig < ng && a.state_in) {
                const f32x4* at = reinterpret_cast<const f32x4*>(a.state_in + head_state) + ((jg0 + m) * ng + ig) * 4 + l;
                S[m][n] = kStream ? __builtin_nontemporal_load(at) : *at;
            }
        }
    // the column that this lane has a token's v and output of: in a row of lanes that of the row's group
    const int group = jg0 + (G == 4 ? g >> 2 : 0), col = 4 * min(group, groups - 1) + l;
    const bool writes = (G == 4 ? g & 3 : g) == 0 && group < groups;
    struct Token {
        Four k[NI], q[NI];
        T v;
        float al, be;
    } tok[kAhead];
    auto load = [&](int t, Token& x) {
        const int64_t row = first + (kText ? min(t, len - 1) : 0);
        const T* q = static_cast<const T*>(a.q) + row * a.q_row + (int64_t)hk * a.dim_k;
        const T* k = static_cast<const T*>(a.k) + row * a.k_row + (int64_t)hk * a.dim_k;
        const T* v = static_cast<const T*>(a.v) + row * a.v_row + (int64_t)hv * a.dim_v;
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            const int i = 4 * min(g + 16 * n, ng - 1);
            __builtin_memcpy(&x.k[n], k + i, sizeof(Four));
            __builtin_memcpy(&x.q[n], q + i, sizeof(Four));
        }
        x.v = v[col];
        x.al = a.alpha[row * a.gate_row + hv];
        x.be = a.beta ? a.beta[row * a.gate_row + hv] : 0.0f;
    };
    auto four = [&](const Four& x, int n) {
        f32x4 y;
        if constexpr (sizeof(T) == 2)
            y = f32x4{__uint_as_float(x[0] << 16), __uint_as_float(x[0] & 0xffff0000u), __uint_as_float(x[1] << 16),
                      __uint_as_float(x[1] & 0xffff0000u)};
        else
            y = x;
        return g + 16 * n < ng ? y : f32x4{0, 0, 0, 0};
    };
    auto take = [&](int t, const Token& x) {
        f32x4 kf[NI], qf[NI];
        float qk[1] = {0.0f}, kv[G], qs[G];
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            kf[n] = four(x.k[n], n);
            qf[n] = four(x.q[n], n);
#pragma unroll
            for (int e = 0; e < 4; ++e) qk[0] = __builtin_fmaf(kf[n][e], qf[n][e], qk[0]);
        }
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
        float u = to_float<T>(x.v), us[G];
        if (a.beta) u = x.be * (u - x.al * over_lanes(kv));
        const float o = a.scale * __builtin_fmaf(over_lanes(qk), u, x.al * over_lanes(qs));
        if (writes) static_cast<T*>(a.out)[(int64_t)(first + t) * a.out_row + (int64_t)hv * a.dim_v + col] = from_float<T>(o);
        to_lanes(u, us);
#pragma unroll
        for (int m = 0; m < G; ++m)
#pragma unroll
            for (int n = 0; n < NI; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[m][n][e] = __builtin_fmaf(kf[n][e], us[m], x.al * S[m][n][e]);
    };
    if constexpr (kText) {
        if (len > 0) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j) load(j, tok[j]);
            for (int t = 0; t < len; t += kAhead) {
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
                    if (t + j < len) {
                        take(t + j, tok[j]);
                        load(t + j + kAhead, tok[j]);
                    }
            }
        }
    } else {
        load(0, tok[0]);
        take(0, tok[0]);
    }
#pragma unroll
    for (int m = 0; m < G; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            const int ig = g + 16 * n;
            if (jg0 + m < groups && ig < ng) {
                f32x4* at = reinterpret_cast<f32x4*>(a.state_out + head_state) + ((jg0 + m) * ng + ig) * 4 + l;
                if (kStream)
                    __builtin_nontemporal_store(S[m][n], at);
                else
                    *at = S[m][n];
            }
        }
}

bool rows_of_16(const void* p, int64_t row, int dim, int es) {
    return ((uintptr_t)p | (uintptr_t)(row * es) | (uintptr_t)(dim * es)) % 16 == 0;
}

template <int KS, int NT, bool kDelta>
hipError_t launch_prompt(const gdn_dev_args& a, const GdnWork& w, hipStream_t s) {
    using T = std::conditional_t<NT == 1, uint16_t, float>;
    const int es = NT == 1 ? 2 : 4;
    const bool full_q = a.dim_k == 32 * KS && rows_of_16(a.q, a.q_row, a.dim_k, es);
    const bool full_k = a.dim_k == 32 * KS && rows_of_16(a.k, a.k_row, a.dim_k, es);
    const bool direct = NT == 1 && full_q && full_k && rows_of_16(a.v, a.v_row, a.dim_v, es) &&
                        a.k_row < 1 << 24 && a.v_row < 1 << 24;  // (offsets of 64 rows in 32 bits)
    gdn_chunk_kernel<KS, NT, kDelta>
        <<<dim3((unsigned)(w.places * a.heads_v)), 256, 0, s>>>(a, w.n_chunks, w.short_to, full_q, full_k, direct);
    auto scan = [&](auto nc, auto from_inputs) {
        constexpr int NC = decltype(nc)::value;
        const int slices = (a.dim_v + 16 * NC - 1) / (16 * NC);
        gdn_scan_kernel<KS, NT, NC, kDelta, decltype(from_inputs)::value, T>
            <<<dim3((unsigned)((size_t)a.n_seq * a.heads_v * slices)), 576, 0, s>>>(a, w.n_chunks, slices, w.short_to);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, KS <= 4 ? 2 : 1>;
    using Direct = std::integral_constant<bool, NT == 1>;
    // 16 columns a workgroup while the workgroups have a compute unit each (they hold most of its LDS):
    // the shortest chain; else 32, which load K, T and P half as often.  Sequences of 1024 tokens, 16 heads
    // of 128, bf16 with the delta rule, 16 | 32 columns: 2 sequences 44 | 56 us, 3 72 | 59, 16 486 | 284.
    const bool two = (size_t)a.n_seq * a.heads_v * ((a.dim_v + 15) / 16) > 256;
    if (direct)
        two ? scan(Two(), Direct()) : scan(One(), Direct());
    else
        two ? scan(Two(), std::false_type()) : scan(One(), std::false_type());
    return hipGetLastError();
}

template <int KS>
hipError_t launch_prompt_of(const gdn_dev_args& a, const GdnWork& w, hipStream_t s) {
    if (a.dtype == QWEN_BF16)
        return a.beta ? launch_prompt<KS, 1, true>(a, w, s) : launch_prompt<KS, 1, false>(a, w, s);
    return a.beta ? launch_prompt<KS, 3, true>(a, w, s) : launch_prompt<KS, 3, false>(a, w, s);
}

template <int NI, int G, bool kStream, bool kText>
hipError_t launch_tokens(const gdn_dev_args& a, int short_to, hipStream_t s) {
    const int groups = a.dim_v / 4;
    const size_t units = (size_t)a.n_seq * a.heads_v * ((groups + G - 1) / G);
    const dim3 grid((unsigned)((units + 3) / 4));
    if (a.dtype == QWEN_BF16)
        gdn_token_kernel<NI, G, kStream, kText, uint16_t><<<grid, 256, 0, s>>>(a, groups, short_to);
    else
        gdn_token_kernel<NI, G, kStream, kText, float><<<grid, 256, 0, s>>>(a, groups, short_to);
    return hipGetLastError();
}

template <int G, bool kStream, bool kText>
hipError_t launch_tokens_of(const gdn_dev_args& a, int short_to, hipStream_t s) {
    if (a.dim_k <= 64) return launch_tokens<1, G, kStream, kText>(a, short_to, s);
    if (a.dim_k <= 128) return launch_tokens<2, G, kStream, kText>(a, short_to, s);
    return launch_tokens<4, G, kStream, kText>(a, short_to, s);
}

// Token by token: every sequence's one (kText false), or those sequences of a prompt call that have up to
// short_to.
template <bool kText>
hipError_t tokens(const gdn_dev_args& a, int short_to, hipStream_t s) {
    // Four value columns a wavefront while there are few, to have more of them at work: 4 | 8 | 16 sequences of
    // 16 heads of 128 3.6 | 4.9 | 7.3 us, and 16 tokens of each 12.7 | 23 | 41; sixteen columns, four loads in
    // flight a lane and as many sums over the lanes for four times the columns: 3.8 | 4.6 | 6.4 and 14 | 19 | 26.
    if ((size_t)a.n_seq * a.heads_v * a.dim_v <= 8192) return launch_tokens_of<1, false, kText>(a, short_to, s);
    // States of 128 MiB and more, with other layers' before they are next wanted, are not left in the 256 MiB
    // of last-level cache: 256 sequences in turn over four pools 88 us for 103 (one pool again and again: 87 for 80).
    if ((size_t)a.n_seq * a.heads_v * a.dim_k * a.dim_v * 4 < (size_t)128 << 20)
        return launch_tokens_of<4, false, kText>(a, short_to, s);
    return launch_tokens_of<4, true, kText>(a, short_to, s);
}

}  // namespace

hipError_t gdn_launch_prompt(const gdn_dev_args& a, const GdnWork& w, hipStream_t s) {
    if (w.short_to >= 0) {
        const hipError_t e = tokens<true>(a, w.short_to, s);
        if (e != hipSuccess || a.rows <= w.short_to) return e;
    }
    switch (w.ks) {
        case 1: return launch_prompt_of<1>(a, w, s);
        case 2: return launch_prompt_of<2>(a, w, s);
        case 4: return launch_prompt_of<4>(a, w, s);
        default: return launch_prompt_of<8>(a, w, s);
    }
}

hipError_t gdn_launch_step(const gdn_dev_args& a, hipStream_t s) { return tokens<false>(a, 1, s); }
