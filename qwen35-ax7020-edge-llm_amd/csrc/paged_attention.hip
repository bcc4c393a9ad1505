// paged_attention.hip -- attention over a paged cache: single tokens, prompts and trees of
// drafted tokens (attn_dev_paged).
//
//   o = sum_j w_j v_j / sum_j w_j,  w_j = 2^(c q . k_j - m),  c = scale log2 e
//
// One pass over the keys with the running maximum m.  A tile of rows holds the tokens of a sequence with
// the query heads of one key head; its keys come to LDS in tiles, pages in any order, one tile ahead.  Products are
// turned round (K Q^T, V^T W^T), so that a lane holds scores, weights and outputs of one row: the weights
// are the next product's operand as they lie, maxima and sums need two exchanges between lanes.
//
// The tiles of keys of all tiles of rows are one long axis, divided evenly over the workgroups: a batch of
// ragged lengths fills the device to the end, and one long sequence is shared by all.  A workgroup whose share begins
// or ends inside a tile of rows leaves its maxima, sums and outputs, which attn_join_kernel joins in a fixed order.
#include "bf16_terms.h"
#include "paged_attention.h"

namespace {

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void global_void;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using lds_s16x4 = __attribute__((address_space(3))) s16x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -INFINITY;  // the maximum of no scores
__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }  // below 2^-126: 0

// 16 bytes that are read for keys that do not exist and elements past the head's: their weights are 0, but 0 times
// what lies in a free page need not be.
__device__ const uint4 kZeros = {0, 0, 0, 0};

// A tile of rows that this workgroup's share ends in, and begins (AttnPlan::desc_at).
struct AttnDesc {
    int there;   // 0: none
    int first;   // the sequence's first row
    int m0;      // first row of the tile
    int count;   // rows that the sequence has
    int head;    // key head
    int last;    // the workgroup that ends it
    int pad[2];
};

// ---- which tiles -----------------------------------------------------------------------
// Places of tiles of rows: with starts, tile t of sequence s at starts[s] group / rows + s + t, different for
// every tile; else those of each sequence one after the other.
struct Tile {
    int seq, first, count, m0;  // the sequence, its first row, group times its tokens, the tile's first row of those
    int held, places;           // tokens before the call's, places that exist (both as int32: 2^30 at most)
    int tiles;                  // of keys (0: nothing to do)
};

struct Shape {
    const attn_dev_args& a;
    const AttnPlan& p;
    __device__ int64_t places() const {
        if (!a.starts) return (int64_t)a.n_seq * each();
        return (int64_t)a.rows * p.group / p.rows + a.n_seq;
    }
    __device__ int each() const { return (int)(((int64_t)(a.rows / a.n_seq) * p.group + p.rows - 1) / p.rows); }
    __device__ int64_t first_place(int s) const {
        return (int64_t)min(max(a.starts[s], 0), a.rows) * p.group / p.rows + s;
    }
    __device__ Tile tile(int64_t place) const {
        Tile t{};
        int64_t in;
        if (a.starts) {
            int lo = 0, hi = a.n_seq;
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (first_place(mid) <= place)
                    lo = mid;
                else
                    hi = mid;
            }
            t.seq = lo;
            in = place - first_place(lo);
        } else {
            const int n = each();
            t.seq = n == 1 ? (int)place : (int)(place / n);
            in = place - (int64_t)t.seq * n;
        }
        const Span span = span_of(a.starts, a.rows, a.n_seq, t.seq);
        t.first = span.first;
        t.count = span.count * p.group;
        const int64_t m0 = in * p.rows;
        if (in < 0 || m0 >= t.count) return t;
        t.m0 = (int)m0;
        t.held = a.cached[t.seq];
        if (t.held < 0) {
            t.tiles = a.zero_rest ? 1 : 0;
            return t;
        }
        const int room = a.table_pages * a.page;  // (up to 2^30)
        const int last = min(t.count, t.m0 + p.rows) - 1;
        const int seen = a.mask ? span.count : last / p.group + 1;
        t.places = (int)min((int64_t)t.held + seen, (int64_t)room);
        t.held = min(t.held, 1 << 30);
        t.tiles = max(1, (t.places + p.keys - 1) / p.keys);
        return t;
    }
};

__device__ __forceinline__ int64_t wave_sum(int64_t x) {
#pragma unroll
    for (int i = 1; i < 64; i *= 2) x += __shfl_xor(x, i);
    return x;
}

// This workgroup's share: from which tile of keys on, how many.
struct Share {
    int64_t place, total;  // the place it begins in; tiles of keys of the call
    int64_t from, to;      // of those
    int64_t before;        // tiles of the places before
    int workers;           // workgroups with a share
};

// By one wavefront: the tiles of all places are counted, then the place is looked for in which the share begins.
__device__ Share share_of(const Shape& sh, int* held, int least) {
    const int lane = threadIdx.x & 63, heads = sh.a.heads_k;
    const int64_t n = sh.places();
    int64_t sum = 0;
    for (int64_t at = lane; at < n; at += 64) {
        const int t = sh.tile(at).tiles;
        if (at < ATTN_HELD) held[at] = t;
        sum += t;
    }
    Share r{};
    r.total = wave_sum(sum) * heads;
    r.workers = (int)min((int64_t)gridDim.x, max((int64_t)1, r.total / least));
    r.from = (int64_t)blockIdx.x * r.total / r.workers;
    r.to = (int64_t)(blockIdx.x + 1) * r.total / r.workers;
    if ((int)blockIdx.x >= r.workers) r.from = r.to = 0;
    if (r.from >= r.to) return r;
    int64_t before = 0;
    for (int64_t base = 0; base < n; base += 64) {
        const int64_t at = base + lane;
        int64_t mine = 0;
        if (at < n) mine = (int64_t)(at < ATTN_HELD ? held[at] : sh.tile(at).tiles) * heads;
        int64_t upto = mine;
#pragma unroll
        for (int i = 1; i < 64; i *= 2) {
            const int64_t x = __shfl_up(upto, i);
            if (lane >= i) upto += x;
        }
        const uint64_t over = __ballot(before + upto > r.from);
        if (over) {
            const int l = __builtin_ctzll(over);
            r.place = base + l;
            r.before = before + __shfl(upto - mine, l);
            return r;
        }
        before += __shfl(upto, 63);
    }
    return r;
}

__device__ __forceinline__ float pair_max(float x) {  // over the lanes of a row: those 16 apart
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

template <class T>
__device__ __forceinline__ bool odd_bits(u32x4 x);  // some element is not finite
template <>
__device__ __forceinline__ bool odd_bits<float>(u32x4 x) {
    bool r = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= (x[i] & 0x7f800000u) == 0x7f800000u;
    return r;
}
template <>
__device__ __forceinline__ bool odd_bits<uint16_t>(u32x4 x) {
    bool r = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= (x[i] & 0x7f800000u) == 0x7f800000u || (x[i] & 0x7f80u) == 0x7f80u;
    return r;
}
__device__ __forceinline__ bool is_odd(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ float finite(float x) { return is_odd(x) ? 0.0f : x; }
__device__ __forceinline__ float kind_of(float x) {
    return !is_odd(x) ? 0.0f : __float_as_uint(x) << 9 ? 4096.0f : x > 0 ? 1.0f : 64.0f;
}
// A sum of up to 32 kinds to what those values add up to.
__device__ __forceinline__ void add_kinds(f32x4& o, f32x4 kinds) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int x = (int)kinds[e], plus = x & 63, minus = x >> 6 & 63;
        const float y = x >= 4096 || (plus && minus) ? NAN : plus ? INFINITY : minus ? -INFINITY : 0.0f;
        o[e] += y;
    }
}

// ---- the pass over the keys ------------------------------------------------------------
// T: uint16_t (bf16) or float.  D: elements of a head, padded.  RB blocks of 16 rows a wavefront, W wavefronts,
// BN keys a tile.  A step is 32 keys: products of 16 keys by 16 rows by 32 (bf16) or 4 (float32) elements.
template <class T, int D, int RB, int W, int BN>
struct Pass {
    static constexpr bool kBf16 = sizeof(T) == 2;
    static constexpr int E = 16 / sizeof(T);          // elements of a 16-byte part
    static constexpr int kRow = D * sizeof(T);        // bytes of a key in LDS
    static constexpr int kParts = kRow / 16;
    static constexpr int kTile = BN * kRow;           // a tile of keys, or of values
    static constexpr int kStage = 2 * kTile;
    static constexpr int kLoads = kTile / 1024 / W;   // wave instructions of a wavefront for a tile of keys
    static_assert(kTile % (1024 * W) == 0 && BN % 32 == 0 && BN <= 64, "every wavefront copies the same share");
    static constexpr int kQ = D / (4 * E);  // a lane's parts of a row of q
    static constexpr int kOut = D / 16;     // a lane's outputs of a row, in fours
    static constexpr int kFlip = D == 64 ? 4 : 8;  // 32-byte parts of a bf16 value that change places (v_swizzle)

    static constexpr bool kTight = W == 8 && D == 256;  // little room in 256 registers

    const attn_dev_args& a;
    Divisor page;
    int group;
    char* lds;
    int lane, wave;
    Tile t;
    const char* kbase;
    const char* vbase;
    int first_token, last_token;  // of the wavefront's rows (last_token < 0: it has none)
    int token[RB];                // of the lane's rows
    u32x4 q[RB][kQ];
    f32x4 o[RB][kOut];
    float m[RB], l[RB];  // maximum of the scores as they are, this lane's part of the sum
    float c;

    // Positions of a key's parts in LDS: eight keys' parts of one place, which lanes of K Q^T read together, and
    // the 32 bytes of each of eight keys that ds_read_tr16_b64 reads lie in different banks.
    static __device__ int k_swizzle(int r) { return r & 7; }
    static __device__ int v_swizzle(int r) { return !kBf16 ? r & 7 : (D == 64 ? r >> 1 & 3 : r & 7) << 1; }

    // Output e of f of a lane's row is element out_at(f, e); four of them are next to each other.
    // (float32: 16 bytes of a value are the left operands of four products, so that a product's 16
    // rows are four elements apart)
    __device__ int quad_at(int f) const {
        const int g = lane >> 4;
        return kBf16 ? 16 * f + 4 * g : 64 * (f / 4) + 16 * g + 4 * (f % 4);
    }
    static __device__ float quad_of(const f32x4 (&x)[kOut], int f, int e) {
        return kBf16 ? x[f][e] : x[f / 4 * 4 + e][f % 4];
    }

    __device__ void begin(const Tile& tile, int head) {
        t = tile;
        kbase = static_cast<const char*>(a.key_cache) + head * a.cache_head * (int64_t)sizeof(T);
        vbase = static_cast<const char*>(a.value_cache) + head * a.cache_head * (int64_t)sizeof(T);
        const int r0 = t.m0 + wave * RB * 16, r1 = min(r0 + RB * 16, t.count) - 1;
        first_token = r0 / group;
        last_token = r0 < t.count ? r1 / group : -1;
        const bool vec = ((uintptr_t)a.q | (uint64_t)a.q_row * sizeof(T) | (uint64_t)a.q_head * sizeof(T)) % 16 == 0;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const int r = min(r0 + 16 * b + (lane & 15), t.count - 1);  // rows past the end: the last one's, not stored
            token[b] = r / group;
            const T* from = static_cast<const T*>(a.q) + (int64_t)(t.first + token[b]) * a.q_row +
                            (int64_t)(head * group + r % group) * a.q_head;
#pragma unroll
            for (int k = 0; k < kQ; ++k) {
                const int d = (k * 4 + (lane >> 4)) * E;
                q[b][k] = u32x4{0, 0, 0, 0};
                if (d < a.dim) {
                    if (vec)
                        q[b][k] = *reinterpret_cast<const u32x4*>(from + d);
                    else
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if constexpr (kBf16)
                                q[b][k][j] = from[d + 2 * j] | (uint32_t)from[d + 2 * j + 1] << 16;
                            else
                                q[b][k][j] = __float_as_uint(from[d + j]);
                        }
                }
            }
            m[b] = kNone;
            l[b] = 0;
#pragma unroll
            for (int f = 0; f < kOut; ++f) o[b][f] = f32x4{0, 0, 0, 0};
        }
    }

    // Where key j of the sequence is (elements), -1 nowhere.
    __device__ int64_t key_at(int j) const {
        if (j >= t.places) return -1;
        const uint32_t n = divide((uint32_t)j, page);
        const int id = a.tables[t.seq * a.table_row + n];
        return (unsigned)id < (unsigned)a.pages ? id * a.cache_page + ((uint32_t)j - n * a.page) * a.cache_token : -1;
    }

    // Starts the copies of a tile whose keys are at `at` (key i's in lane i): 1 KiB a wave instruction, to consecutive
    // bytes of LDS; the parts' positions are in the addresses.  WHOLE: every key exists, heads have D elements.
    template <bool WHOLE>
    __device__ __forceinline__ void copy_of(int stage, int64_t at) const {
        const char* zeros = reinterpret_cast<const char*>(&kZeros);
        char* to = lds + stage * kStage;
        int lane = this->lane;
        if (kTight || !WHOLE) asm volatile("" : "+v"(lane));  // (addresses are not kept in registers across the loop)
        const int part = lane % kParts;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int n = wave * kLoads + i, r = n * (64 / kParts) + lane / kParts;
            const int64_t from = __shfl(at, r) * (int64_t)sizeof(T);
            const int kp = part ^ k_swizzle(r), vp = part ^ v_swizzle(r);
            const char* ks = WHOLE || (from >= 0 && kp * E < a.dim) ? kbase + from + kp * 16 : zeros;
            const char* vs = WHOLE || (from >= 0 && vp * E < a.dim) ? vbase + from + vp * 16 : zeros;
            __builtin_amdgcn_global_load_lds((global_void*)ks, (lds_void*)(to + n * 1024), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((global_void*)vs, (lds_void*)(to + kTile + n * 1024), 16, 0, 0);
        }
    }
    __device__ __forceinline__ void copy(int stage, int64_t at) const {
        if (a.dim == D && __all(at >= 0))
            copy_of<true>(stage, at);
        else
            copy_of<false>(stage, at);
    }
    static __device__ void sync() {  // LDS alone: copies stay in flight
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    static __device__ void arrived() {  // every copy is in LDS, for all wavefronts; their reads are done
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }

    // Which of the 32 keys from k0 on row b of this lane sees, of those that exist.
    __device__ uint32_t seen(int b, int k0, uint32_t there) const {
        if (!a.mask) {
            const int upto = t.held + token[b] - k0;
            return upto < 0 ? 0 : upto >= 31 ? there : there & ((2u << upto) - 1);
        }
        const int j = k0 - t.held;
        if (j <= -32) return there;
        const int32_t* words = a.mask + (int64_t)(t.first + token[b]) * a.mask_words;
        if (j < 0) {
            const uint32_t w = a.mask_words > 0 ? words[0] : 0;
            return there & (w << -j | ((1u << -j) - 1));
        }
        const int n = j >> 5, sh = j & 31;
        const uint32_t lo = n < a.mask_words ? words[n] : 0, hi = n + 1 < a.mask_words ? words[n + 1] : 0;
        return there & (uint32_t)(((uint64_t)hi << 32 | lo) >> sh);
    }

    // Byte of LDS, from a step's first key on, of the values that product f reads with ds_read_tr16_b64: lane n of 16
    // reads 8 bytes of key 4 g + n / 4 (and of that 16 keys on), and gets element n of four keys.
    __device__ __forceinline__ int tr_at() const {
        const int n = lane & 15, r = 4 * (lane >> 4) + (n >> 2);
        return r * kRow + (v_swizzle(r) ^ (n >> 1 & 1)) * 16 + (n & 1) * 8;
    }
    static __device__ __forceinline__ u32x4 tr_read(const char* v, int at, int f) {
        const char* x = v + (at ^ f % kFlip * 32) + f / kFlip * (kFlip * 32);
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)x));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(x + 16 * kRow)));
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
    // float32: parts 16 f + lane % 16 of key 16 (i / 4) + 4 g + i % 4
    __device__ __forceinline__ f32x4 row_read(const char* v, int i, int f) const {
        const int r = 16 * (i / 4) + 4 * (lane >> 4) + i % 4;
        return *reinterpret_cast<const f32x4*>(v + r * kRow + ((16 * f + (lane & 15)) ^ v_swizzle(r)) * 16);
    }

    // O += the values of 32 keys (from v on) times their weights.
    __device__ __forceinline__ void add_values(const char* v, const float (&w)[RB][2][4], const u32x4 (&wb)[RB]) {
        if constexpr (kBf16) {
            int at = tr_at();
            asm volatile("" : "+v"(at));  // (one operation a product, not a register each)
#pragma unroll
            for (int f = 0; f < kOut; ++f) {
                const u32x4 y = tr_read(v, at, f);
#pragma unroll
                for (int b = 0; b < RB; ++b) o[b][f] = mfma(y, wb[b], o[b][f]);
            }
        } else {
#pragma unroll
            for (int f = 0; f < kOut / 4; ++f)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const f32x4 y = row_read(v, i, f);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int b = 0; b < RB; ++b)
                            o[b][4 * f + j] = mfma4(y[j], w[b][i / 4][i % 4], o[b][4 * f + j]);
                }
        }
    }

    // The values of 32 keys (from v on) that are not finite, to the rows that see them: counted by a product, their kinds
    // (1 infinity, 64 minus infinity, 4096 NaN) with 1 for a key that is seen.
    __device__ __forceinline__ void add_odd(const char* v, int k0, uint32_t there) {
        const int g = lane >> 4;
        float see[RB][8];
        u32x4 seeb[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const uint32_t sees = seen(b, k0, there) >> (4 * g);
#pragma unroll
            for (int i = 0; i < 8; ++i) see[b][i] = (float)(sees >> (16 * (i / 4) + i % 4) & 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) seeb[b][i] = round2(see[b][2 * i], see[b][2 * i + 1]);
        }
        const int at = kBf16 ? tr_at() : 0;
#pragma unroll
        for (int f = 0; f < (kBf16 ? kOut : kOut / 4); ++f) {
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (kBf16) {
                u32x4 y = tr_read(v, at, f);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    y[j] = round2(kind_of(__uint_as_float(y[j] << 16)), kind_of(__uint_as_float(y[j] & 0xffff0000u)));
#pragma unroll
                for (int b = 0; b < RB; ++b) add_kinds(o[b][f], mfma(y, seeb[b], f32x4{0, 0, 0, 0}));
            } else {
                f32x4 kinds[RB][4] = {};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const f32x4 y = row_read(v, i, f);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int b = 0; b < RB; ++b) kinds[b][j] = mfma4(kind_of(y[j]), see[b][i], kinds[b][j]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int b = 0; b < RB; ++b) add_kinds(o[b][4 * f + j], kinds[b][j]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }

    // A tile of which some row does not see every key: a value that is not finite must not reach such a row as 0 times it.
    // If there are any, those rows that see them get them here, and 0 takes their place.
    __device__ void clean(int stage, int k0, uint64_t there, int* flags) {
        char* v = lds + stage * kStage + kTile;
        bool odd = false;
        for (int i = wave * 64 + lane; i < BN * kParts; i += 64 * W)
            odd |= odd_bits<T>(*reinterpret_cast<const u32x4*>(v + i * 16));
        const bool mine = __any(odd);
        if (lane == 0) flags[wave] = mine;
        sync();
        int any = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) any |= flags[i];
        if (__builtin_amdgcn_readfirstlane(any)) {
            if (last_token >= 0)
#pragma unroll 1
                for (int i = 0; i < BN / 32; ++i) add_odd(v + 32 * i * kRow, k0 + 32 * i, (uint32_t)(there >> 32 * i));
            sync();
            for (int i = wave * 64 + lane; i < BN * kParts; i += 64 * W) {
                u32x4 x = *reinterpret_cast<const u32x4*>(v + i * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (kBf16)
                        x[j] = round2(finite(__uint_as_float(x[j] << 16)), finite(__uint_as_float(x[j] & 0xffff0000u)));
                    else
                        x[j] = __float_as_uint(finite(__uint_as_float(x[j])));
                }
                *reinterpret_cast<u32x4*>(v + i * 16) = x;
            }
        }
        sync();  // (and the flags can be written again)
    }

    // The keys k0 .. k0 + 31, at rows k .. of the tile in `stage`.
    __device__ __forceinline__ void step(int stage, int k, int k0, uint32_t there) {
        const char* ks = lds + stage * kStage;
        const char* vs = ks + kTile;
        const int n = lane & 15, g = lane >> 4;
        int at[2];  // parts 4 i + g of a key: eight of them change places
#pragma unroll
        for (int i = 0; i < 2; ++i) at[i] = n * kRow + ((4 * i + g) ^ k_swizzle(n)) * 16;
        f32x4 s[RB][2];
#pragma unroll
        for (int b = 0; b < RB; ++b) s[b][0] = s[b][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kQ; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(ks + (k + 16 * h) * kRow + at[i % 2] + i / 2 * 128);
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    if constexpr (kBf16) {
                        s[b][h] = mfma(x, q[b][i], s[b][h]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            s[b][h] = mfma4(__uint_as_float(x[j]), __uint_as_float(q[b][i][j]), s[b][h]);
                    }
                }
            }
        // scores and the maximum before any branch: the first use of the products
        float top[RB];
        const bool all = there == 0xffffffffu && (a.mask ? k0 + 32 <= t.held : k0 + 31 <= t.held + first_token);
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const uint32_t bits = (all ? 0xffffffffu : seen(b, k0, there)) >> (4 * g);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(bits >> (16 * (i / 4) + i % 4) & 1)) s[b][i / 4][i % 4] = kNone;
            const f32x4 x = s[b][0], y = s[b][1];
            top[b] = pair_max(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]))));
        }
        bool grows = false;
#pragma unroll
        for (int b = 0; b < RB; ++b) grows |= top[b] > m[b];
        if (__any(grows)) {
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const float now = fmaxf(m[b], top[b]);
                const float f = m[b] == kNone ? 1.0f : exp2_raw(m[b] * c - now * c);  // (nothing yet but clean()'s)
                m[b] = now;
                l[b] *= f;
#pragma unroll
                for (int i = 0; i < kOut; ++i) o[b][i] *= f;
            }
        }
        float w[RB][2][4];
        u32x4 wb[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const float mc = m[b] == kNone ? 0.0f : m[b] * c;
#pragma unroll
            for (int i = 0; i < 8; ++i) w[b][i / 4][i % 4] = exp2_raw(__builtin_fmaf(s[b][i / 4][i % 4], c, -mc));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = w[b][i / 2][i % 2 * 2], y = w[b][i / 2][i % 2 * 2 + 1];
                if (kBf16) {
                    wb[b][i] = round2(x, y);
                    x = __uint_as_float(wb[b][i] << 16);
                    y = __uint_as_float(wb[b][i] & 0xffff0000u);
                }
                l[b] += x;
                l[b] += y;
            }
        }
        add_values(vs + k * kRow, w, wb);
    }

    // The tiles of keys k0 .. k1 - 1 of this tile of rows.
    __device__ void run(int k0, int k1, int* flags) {
        arrived();  // (the tile of rows before is done with LDS)
        int64_t next = key_at(k0 * BN + lane % BN);
        copy(0, next);
        uint64_t there = __ballot(next >= 0);
        next = k0 + 1 < k1 ? key_at((k0 + 1) * BN + lane % BN) : -1;
        for (int k = k0; k < k1; ++k) {
            const uint64_t now = there;
            const int stage = (k - k0) & 1;
            arrived();
            if (k + 1 < k1) {
                copy(stage ^ 1, next);
                there = __ballot(next >= 0);
                if (k + 2 < k1) next = key_at((k + 2) * BN + lane % BN);
            }
            if (now != ~0ull || (a.mask ? (k + 1) * BN > t.held : (k + 1) * BN - 1 > t.held + t.m0 / group))
                clean(stage, k * BN, now, flags);
#pragma unroll
            for (int i = 0; i < BN / 32; ++i) {
                const int from = k * BN + 32 * i;
                if (last_token >= 0 && (a.mask || from <= t.held + last_token)) step(stage, 32 * i, from, (uint32_t)(now >> 32 * i));
            }
        }
    }
};

template <class T>
__device__ __forceinline__ void store4(T* to, const float (&x)[4], bool vec) {
    if (vec) {
        if constexpr (sizeof(T) == 2)
            *reinterpret_cast<u32x2*>(to) = u32x2{round2(x[0], x[1]), round2(x[2], x[3])};
        else
            *reinterpret_cast<f32x4*>(to) = f32x4{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = from_float<T>(x[e]);
    }
}
template <class T>
__device__ __forceinline__ bool quads(const attn_dev_args& a) {  // four elements of out can be stored at once
    return ((uintptr_t)a.out | (uint64_t)a.out_row * sizeof(T) | (uint64_t)a.out_head * sizeof(T)) % (4 * sizeof(T)) == 0;
}

template <class T, int D, int RB, int W, int BN>
__global__ __launch_bounds__(64 * W) void attn_kernel(attn_dev_args a, AttnPlan p, Divisor page, int least) {
    using P = Pass<T, D, RB, W, BN>;
    __shared__ __attribute__((aligned(1024))) char lds[2 * P::kStage];
    __shared__ int held[ATTN_HELD];
    __shared__ Share share_sh;
    __shared__ int flags[W];
    const Shape shape{a, p};
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave == 0) {
        const Share s = share_of(shape, held, least);
        if (threadIdx.x == 0) share_sh = s;
    }
    __syncthreads();
    const Share share = share_sh;
    AttnDesc* desc = reinterpret_cast<AttnDesc*>(static_cast<char*>(a.work) + p.desc_at) + blockIdx.x;
    float2* stats = reinterpret_cast<float2*>(static_cast<char*>(a.work) + p.stat_at);
    f32x4* parts = reinterpret_cast<f32x4*>(static_cast<char*>(a.work) + p.part_at);
    AttnDesc left{};
    P pass{a, page, p.group, lds, (int)(threadIdx.x & 63), wave};
    pass.c = a.scale * kLog2e;
    int64_t at = share.from, place = share.place, before = share.before;
    const int64_t places = shape.places();
    const bool vec = quads<T>(a);
    while (at < share.to && place < places) {
        const Tile t = shape.tile(place);
        const int64_t in = at - before, all = (int64_t)t.tiles * a.heads_k;
        if (in >= all) {
            before += all;
            ++place;
            continue;
        }
        const int head = (int)(in / t.tiles), k0 = (int)(in - (int64_t)head * t.tiles);
        const int k1 = (int)min((int64_t)t.tiles, k0 + (share.to - at));
        at += k1 - k0;
        pass.begin(t, head);
        if (t.held >= 0) pass.run(k0, k1, flags);
        asm volatile("s_nop 7\n\ts_nop 7" ::: "memory");  // the last products' results, whatever way the loop was left
        if (k0 == 0 && k1 < t.tiles)
            left = AttnDesc{1, t.first, t.m0, t.count, head,
                            (int)(((at - k1 + t.tiles) * share.workers - 1) / share.total)};
        const int n = threadIdx.x & 15, slot = 2 * blockIdx.x + (k0 == 0);
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const int block = wave * RB + b, r = t.m0 + 16 * block + n;
            const float sum = pair_sum(pass.l[b]);
            if (r >= t.count) continue;
            if (k0 == 0 && k1 == t.tiles) {
                const float f = sum == 0 ? 0.0f : 1.0f / sum;
                T* to = static_cast<T*>(a.out) + (int64_t)(t.first + r / p.group) * a.out_row +
                        (int64_t)(head * p.group + r % p.group) * a.out_head;
#pragma unroll
                for (int i = 0; i < P::kOut; ++i) {
                    const int d = pass.quad_at(i);
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = sum == 0 ? 0.0f : P::quad_of(pass.o[b], i, e) * f;
                    if (d < a.dim) store4(to + d, x, vec);
                }
            } else {
                if (threadIdx.x % 64 < 16) stats[(int64_t)slot * p.rows + 16 * block + n] = float2{pass.m[b] * pass.c, sum};
                f32x4* to = parts + ((int64_t)slot * (p.rows / 16) + block) * P::kOut * 64 + (threadIdx.x & 63);
#pragma unroll
                for (int i = 0; i < P::kOut; ++i) to[i * 64] = pass.o[b][i];
            }
        }
    }
    if (threadIdx.x == 0) *desc = left;
}

// The parts of a tile of rows, 16 rows and 64 elements to a workgroup: its first part is the last of workgroup
// blockIdx.x, the others are the first of those that follow.  Four wavefronts take every fourth.
template <class T, int D>
__global__ __launch_bounds__(256) void attn_join_kernel(attn_dev_args a, AttnPlan p) {
    const AttnDesc d = reinterpret_cast<const AttnDesc*>(static_cast<const char*>(a.work) + p.desc_at)[blockIdx.x];
    const int block = blockIdx.y, m0 = d.m0 + 16 * block;
    if (!d.there || m0 >= d.count) return;
    constexpr int kOut = D / 16;
    const float2* stats = reinterpret_cast<const float2*>(static_cast<const char*>(a.work) + p.stat_at);
    const f32x4* parts = reinterpret_cast<const f32x4*>(static_cast<const char*>(a.work) + p.part_at);
    __shared__ f32x4 sums[4][4][64];
    __shared__ float2 tops[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, first = blockIdx.x;
    const bool mine = m0 + n < d.count;
    f32x4 o[4] = {};
    float m = kNone, l = 0;
    if (mine)
        for (int w = first + wave; w <= d.last; w += 4) {
            const int slot = w == first ? 2 * first + 1 : 2 * w;
            const float2 s = stats[(int64_t)slot * p.rows + 16 * block + n];
            const f32x4* from = parts + (((int64_t)slot * (p.rows / 16) + block) * kOut + 4 * blockIdx.z) * 64 + lane;
            const float now = fmaxf(m, s.x);
            if (now == kNone) continue;
            const float f = exp2_raw(m - now), e = exp2_raw(s.x - now);
            m = now;
            l = l * f + s.y * e;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = o[i] * f + from[i * 64] * e;
        }
    tops[wave][lane] = float2{m, l};
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][i][lane] = o[i];
    __syncthreads();
    if (!mine) return;
    // each wavefront a quarter: its own four outputs of the lane's row
    float top = kNone;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, tops[w][lane].x);
    float sum = 0, x[4] = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float2 s = tops[w][lane];
        const float f = s.x == kNone ? 0.0f : exp2_raw(s.x - top);
        sum += s.y * f;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += (sizeof(T) == 2 ? sums[w][wave][lane][e] : sums[w][e][lane][wave]) * f;
    }
    const float f = 1.0f / sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = sum == 0 ? 0.0f : x[e] * f;
    const int g = lane >> 4, at = 64 * blockIdx.z + (sizeof(T) == 2 ? 16 * wave + 4 * g : 16 * g + 4 * wave);
    const int r = m0 + n;
    T* to = static_cast<T*>(a.out) + (int64_t)(d.first + r / p.group) * a.out_row +
            (int64_t)(d.head * p.group + r % p.group) * a.out_head;
    if (at < a.dim) store4(to + at, x, quads<T>(a));
}

template <class T, int D, int RB, int W, int BN>
hipError_t launch(const attn_dev_args& a, const AttnPlan& p, hipStream_t s) {
    attn_kernel<T, D, RB, W, BN><<<dim3((unsigned)p.grid), 64 * W, 0, s>>>(a, p, divisor(a.page), 1);
    attn_join_kernel<T, D><<<dim3((unsigned)p.grid, (unsigned)(p.rows / 16), D / 64), 256, 0, s>>>(a, p);
    return hipGetLastError();
}

template <int D>
hipError_t launch_bf16(const attn_dev_args& a, const AttnPlan& p, hipStream_t s) {
    if (p.blocks == 1) return launch<uint16_t, D, 1, 1, 32>(a, p, s);
    switch (p.waves) {
        case 1: return launch<uint16_t, D, 2, 1, 32>(a, p, s);
        case 2: return launch<uint16_t, D, 2, 2, 32>(a, p, s);
        case 4: return launch<uint16_t, D, 2, 4, 32>(a, p, s);
        default: return launch<uint16_t, D, 2, 8, 64>(a, p, s);
    }
}
template <int D>
hipError_t launch_f32(const attn_dev_args& a, const AttnPlan& p, hipStream_t s) {
    switch (p.waves) {
        case 1: return launch<float, D, 1, 1, 32>(a, p, s);
        case 2: return launch<float, D, 1, 2, 32>(a, p, s);
        case 4: return launch<float, D, 1, 4, 32>(a, p, s);
        default: return launch<float, D, 1, 8, 32>(a, p, s);
    }
}

}  // namespace

hipError_t attn_launch_paged(const attn_dev_args& a, const AttnPlan& p, hipStream_t s) {
    if (a.dtype == QWEN_BF16)
        return p.dim == 64 ? launch_bf16<64>(a, p, s) : p.dim == 128 ? launch_bf16<128>(a, p, s) : launch_bf16<256>(a, p, s);
    return p.dim == 64 ? launch_f32<64>(a, p, s) : p.dim == 128 ? launch_f32<128>(a, p, s) : launch_f32<256>(a, p, s);
}
