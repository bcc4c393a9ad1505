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
// The tiles of keys of all tiles of rows, and some more for what a tile of rows costs by itself, are one long axis,
// divided evenly over the workgroups: a batch of ragged lengths fills the device to the end, and one long sequence is
// shared by all.  A workgroup whose share begins or ends inside a tile of rows leaves its maxima, sums and outputs,
// which attn_join_kernel joins in a fixed order.
#include <type_traits>

#include "bf16_terms.h"
#include "paged_attention.h"

namespace {

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void global_void;
typedef __attribute__((address_space(1))) const char global_char;  // (where a pointer is one of two, the compiler has to be told)
using s16x4 = __attribute__((ext_vector_type(4))) short;
using lds_s16x4 = __attribute__((address_space(3))) s16x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -INFINITY;  // the maximum of no scores
constexpr uint32_t kNowhere = 0xffffffffu;
// A row's maximum is raised, and what it has so far scaled down to it, only by a score that is this much above it:
// weights then are up to 2^8, and float32 sums have the same bits.  (Each of 32 rows raises its own: without slack
// nearly every 32 keys of the first thousand.)
constexpr float kSlack = 8;
__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }  // below 2^-126: 0

// 16 bytes that are read for keys that do not exist and elements past the head's: their weights are 0, but 0 times
// what lies in a free page need not be.
__device__ const uint4 kZeros[64] = {};  // (attn_step_kernel: a whole key's or value's)

// 16 bytes a lane from `from` to 1 KiB of LDS, the same `to` in all lanes.  (The builtin of this instruction makes the
// compiler wait for all copies in flight before the next read of LDS, whichever buffer that is from. Whoever reads
// waits for itself: Pass::arrived.)
__device__ __forceinline__ void copy_to_lds(global_char* from, char* to) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void*)to);
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(at) : "memory");
}

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
    int cost;                   // on the axis that is divided: and AttnPlan::extra
};

struct Shape {
    const attn_dev_args& a;
    const AttnPlan& p;
    // (rows group is up to 2^28, a tile's rows are a power of two)
    __device__ int tiles_of(int rows) const { return (rows * p.group) >> p.rows_log; }
    __device__ int places() const { return a.starts ? tiles_of(a.rows) + a.n_seq : a.n_seq * p.each; }
    __device__ int first_place(int s) const { return tiles_of(min(max(a.starts[s], 0), a.rows)) + s; }
    // The last sequence whose first place is not past this one.
    __device__ int seq_of(int place) const {
        int lo = 0, hi = a.n_seq;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (first_place(mid) <= place)
                lo = mid;
            else
                hi = mid;
        }
        return lo;
    }
    // The same for places (of any lanes) that are up to 64 sequences past lo, by a load of all lanes and exchanges
    // between them; lo + 64 if they are more (1,024 sequences, two at work: a search in memory for every place 81 us,
    // so 58).
    __device__ __forceinline__ int seq_from(int lo, int place) const {
        const int next = lo + 1 + (threadIdx.x & 63), first = next < a.n_seq ? first_place(next) : INT32_MAX;
        int past = 0;
#pragma unroll
        for (int i = 32; i; i /= 2)
            if (__shfl(first, past + i - 1) <= place) past += i;
        return lo + past + (__shfl(first, past) <= place);
    }
    __device__ Tile tile(int place) const { return tile(place, a.starts ? seq_of(place) : 0); }
    __device__ Tile tile(int place, int seq) const {  // (seq: with starts)
        Tile t{};
        int in = 0;
        if (a.starts) {
            t.seq = seq;
            in = place - first_place(seq);
        } else if (p.each == 1) {
            t.seq = place;
        } else {
            t.seq = place / p.each;
            in = place - t.seq * p.each;
        }
        const Span span = span_of(a.starts, a.rows, a.n_seq, t.seq);
        t.first = span.first;
        t.count = span.count * p.group;
        if (in < 0 || in > (t.count - 1) >> p.rows_log) return t;  // (without rows: -1)
        t.m0 = in << p.rows_log;
        t.held = a.cached[t.seq];
        if (t.held < 0) {
            t.tiles = t.cost = a.zero_rest ? 1 : 0;
            return t;
        }
        const int room = a.pages ? a.table_pages * a.page : 0;  // (up to 2^30)
        const int last = min(t.count, t.m0 + p.rows) - 1;
        const int seen = a.mask ? span.count : last / p.group + 1;
        t.places = (int)min((int64_t)t.held + seen, (int64_t)room);
        t.held = min(t.held, 1 << 30);
        t.tiles = max(1, (t.places + p.keys - 1) / p.keys);
        t.cost = t.tiles + p.extra;
        return t;
    }
};

template <class T>
__device__ __forceinline__ T uniform(T x) {  // the same in all lanes: to scalar registers
    int w[sizeof(T) / 4];
    __builtin_memcpy(w, &x, sizeof(T));
#pragma unroll
    for (size_t i = 0; i < sizeof(T) / 4; ++i) w[i] = __builtin_amdgcn_readfirstlane(w[i]);
    __builtin_memcpy(&x, w, sizeof(T));
    return x;
}

// This workgroup's share: from which tile of keys on, how many.
struct Share {
    int64_t total;     // tiles of keys of the call
    int64_t from, to;  // of those
    int64_t before;    // tiles of the places before
    int place;         // the place it begins in
    int seq;           // a sequence that is not past that place's
    int workers;       // workgroups with a share
};

__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {  // (a division of 64 bits is 20 times one of 32)
    return (x | y) >> 32 ? x / y : (uint32_t)x / (uint32_t)y;
}

// By every wavefront for itself: the tiles of all places are counted (a chunk of 64 at a time: 2^25 each at most), then
// the place is looked for in which the share begins.
__device__ Share share_of(const Shape& sh, int* held, int least) {
    const int lane = threadIdx.x & 63, heads = sh.a.heads_k;
    const int n = sh.places();
    auto scan = [&](uint32_t mine) {  // tiles of the chunk's places up to this one
#pragma unroll
        for (int i = 1; i < 64; i *= 2) {
            const uint32_t x = __shfl_up(mine, i);
            if (lane >= i) mine += x;
        }
        return mine;
    };
    int64_t sum = 0;
    uint32_t upto = 0, mine = 0;
    int seq = 0, far = 0;  // the sequence of the last place so far, and of the last one of `held`
    for (int base = 0; base < n; base += 64) {
        const int at = base + lane;
        if (base == ATTN_HELD) far = seq;
        const int own = sh.a.starts ? sh.seq_from(seq, at) : 0;
        mine = at < n ? sh.tile(at, own).cost : 0;
        seq = __shfl(own, 63);
        if (at < ATTN_HELD) held[at] = mine;
        upto = scan(mine);
        sum += (uint32_t)__shfl(upto, 63);
    }
    Share r{};
    r.total = sum * heads;
    r.workers = (int)min((int64_t)gridDim.x, max((int64_t)1, quotient(r.total, least)));
    r.from = quotient(blockIdx.x * r.total, r.workers);
    r.to = quotient((blockIdx.x + 1) * r.total, r.workers);
    if ((int)blockIdx.x >= r.workers) r.from = r.to = 0;
    if (r.from >= r.to) return r;
    int64_t before = 0;
    seq = far;
    for (int base = 0; base < n; base += 64) {
        if (n > 64) {
            const int at = base + lane;
            if (base >= ATTN_HELD) {
                const int own = sh.a.starts ? sh.seq_from(seq, at) : 0;
                mine = at < n ? sh.tile(at, own).cost : 0;
                r.seq = seq;
                seq = __shfl(own, 63);
            } else {
                mine = at < n ? held[at] : 0;
            }
            upto = scan(mine);
        }
        const uint64_t over = __ballot((before + upto) * heads > r.from);
        if (over) {
            const int l = __builtin_ctzll(over);
            r.place = base + l;
            r.before = (before + (uint32_t)__shfl(upto - mine, l)) * heads;
            return r;
        }
        before += (uint32_t)__shfl(upto, 63);
    }
    return r;
}

// The first place after this one that has something to do: a batch's skipped and empty sequences, 64 at a time.
__device__ __forceinline__ int place_after(const Shape& sh, const int* held, int place) {
    const int lane = threadIdx.x & 63, n = sh.places();
    for (int base = place + 1; base < n; base += 64) {
        const int at = base + lane;
        const uint64_t some = __ballot(at < n && (at < ATTN_HELD ? held[at] : sh.tile(at).cost) > 0);
        if (some) return base + __builtin_ctzll(some);
    }
    return n;
}

// The sequence of a place that lies further on than lo's.
__device__ __forceinline__ int next_seq(const Shape& sh, int lo, int place) {
    const int seq = __builtin_amdgcn_readfirstlane(sh.seq_from(lo, place));
    return seq < lo + 64 ? seq : __builtin_amdgcn_readfirstlane(sh.seq_of(place));
}

// Where key j of a sequence is, in units of the cache's strides (AttnPlan), kNowhere if it does not exist.
__device__ __forceinline__ uint32_t key_at(const attn_dev_args& a, const AttnUnits& u, const Tile& t, int j) {
    if (j >= t.places) return kNowhere;
    const uint32_t n = divide((uint32_t)j, u.divisor);
    const int id = a.tables[t.seq * a.table_row + n];
    return (unsigned)id < (unsigned)a.pages ? (uint32_t)id * u.page + ((uint32_t)j - n * a.page) * u.token : kNowhere;
}
__device__ __forceinline__ global_char* in_cache(global_char* base, uint32_t at, const AttnUnits& u) {
    return base + ((uint64_t)at << u.log);
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

__device__ __forceinline__ float sum2(uint32_t pair, float x) {  // x + both of a pair of bf16
    using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, 0x3f803f80u), x, false);
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
// FULL: heads have D elements.
template <class T, int D, int RB, int W, int BN, bool FULL>
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

    // Eight wavefronts leave each 256 registers: outputs and queries of 32 rows of 256 bf16 elements are 192 of them.
    static constexpr bool kTight = W == 8 && D == 256;

    const attn_dev_args& a;
    AttnUnits units;
    int group;
    char* lds;
    int lane, wave;
    Tile t;
    global_char* kbase;
    global_char* vbase;
    int kv_head, last_token;  // last of the wavefront's rows (below 0: it has none)
    u32x4 q[RB][kQ];
    f32x4 o[RB][kOut];
    float m[RB], l[RB];  // maximum of the scores (in base 2), or up to kSlack less, and this lane's part of the sum
    float c;

    // Positions of a key's parts in LDS.  16 lanes whose 16 bytes are read at once have to have them in different
    // sixteenths of 256 bytes: those of K Q^T, with parts 4 i and 4 i + 1 of eight keys each, change places
    // by their key; the 32 bytes of each of eight keys that ds_read_tr16_b64 reads too.  float32 values are read along the
    // key.  (Among eight parts only, every read of keys met itself: 1,159 us for 1,149 of the prompt below.)
    static constexpr int kTurn = kParts < 16 ? 8 : 16;
    static __device__ int k_swizzle(int r) { return r & (kTurn - 1); }
    static __device__ int v_swizzle(int r) { return !kBf16 ? 0 : (D == 64 ? r >> 1 & 3 : r & 7) << 1; }

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

    __device__ __forceinline__ void begin(const Tile& tile, int head) {
        t = tile;
        kv_head = head;
        kbase = (global_char*)a.key_cache + head * a.cache_head * (int64_t)sizeof(T);
        vbase = (global_char*)a.value_cache + head * a.cache_head * (int64_t)sizeof(T);
        const int r0 = t.m0 + wave * RB * 16, r1 = min(r0 + RB * 16, t.count) - 1;
        last_token = r0 < t.count ? r1 / group : -1;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            m[b] = kNone;
            l[b] = 0;
#pragma unroll
            for (int f = 0; f < kOut; ++f) o[b][f] = f32x4{0, 0, 0, 0};
        }
    }
    __device__ __forceinline__ int token_of(int b) const {  // rows past the end: the last one, not stored
        return min(t.m0 + (wave * RB + b) * 16 + (lane & 15), t.count - 1) / group;
    }
    __device__ __forceinline__ void load_q() {
        const bool vec = ((uintptr_t)a.q | (uint64_t)a.q_row * sizeof(T) | (uint64_t)a.q_head * sizeof(T)) % 16 == 0;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const int r = min(t.m0 + (wave * RB + b) * 16 + (lane & 15), t.count - 1);
            const T* from = static_cast<const T*>(a.q) + (int64_t)(t.first + r / group) * a.q_row +
                            (int64_t)(kv_head * group + r % group) * a.q_head;
#pragma unroll
            for (int k = 0; k < kQ; ++k) {
                const int d = (k * 4 + (lane >> 4)) * E;
                u32x4 x = {0, 0, 0, 0};
                if (d < a.dim) {
                    if (vec)
                        x = *reinterpret_cast<const u32x4*>(from + d);
                    else
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if constexpr (kBf16)
                                x[j] = from[d + 2 * j] | (uint32_t)from[d + 2 * j + 1] << 16;
                            else
                                x[j] = __float_as_uint(from[d + j]);
                        }
                }
                q[b][k] = x;
            }
        }
    }

    __device__ uint32_t key_at(int j) const { return ::key_at(a, units, t, j); }

    // Starts the copies of a tile whose keys are at `at` (key i's in lane i): 1 KiB a wave instruction, to consecutive
    // bytes of LDS; the parts' positions are in the addresses.  The first place stands for keys that do not exist: no
    // row sees them, and clean() takes care that their values do no harm.
    __device__ __forceinline__ void copy(int stage, uint32_t at) const {
        if (at == kNowhere) at = 0;
        global_char* zeros = (global_char*)kZeros;
        char* to = lds + stage * kStage;
        int lane = this->lane;
        if (kTight || !FULL) asm volatile("" : "+v"(lane));  // (addresses are not kept in registers across the loop)
        const int part = lane % kParts;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int n = wave * kLoads + i, r = n * (64 / kParts) + lane / kParts;
            const uint32_t from = __shfl(at, r);
            const int kp = part ^ k_swizzle(r), vp = part ^ v_swizzle(r);
            global_char* ks = FULL || kp * E < a.dim ? in_cache(kbase, from, units) + kp * 16 : zeros;
            global_char* vs = FULL || vp * E < a.dim ? in_cache(vbase, from, units) + vp * 16 : zeros;
            copy_to_lds(ks, to + n * 1024);
            copy_to_lds(vs, to + kTile + n * 1024);
        }
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
            const int upto = t.held + token_of(b) - k0;
            return upto < 0 ? 0 : upto >= 31 ? there : there & ((2u << upto) - 1);
        }
        const int j = k0 - t.held;
        if (j <= -32) return there;
        const int32_t* words = a.mask + (int64_t)(t.first + token_of(b)) * a.mask_words;
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
    static __device__ __forceinline__ int tr_at(int lane) {
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
        return *reinterpret_cast<const f32x4*>(v + r * kRow + (16 * f + (lane & 15)) * 16);
    }

    // The operands of the step's products, read kDeep - 1 ahead of them.  Keys: part 4 i + g of keys 16 h + lane % 16.
    // Values (operand t of kValues): bf16 a product's, 32 keys by 16 elements; float32 four products', four keys by 64
    // elements.
    static constexpr int kDeep = kBf16 && !kTight ? 4 : 3;
    static constexpr int kKeys = 2 * kQ, kValues = kBf16 ? kOut : 2 * kOut;
    using Operand = u32x4;
    static __device__ __forceinline__ Operand read_key(const char* k, int at, int t) {
        const int i = t / 2, h = t % 2;  // (kTurn parts change places with one another)
        return *reinterpret_cast<const Operand*>(k + (at ^ i % (kTurn / 4) * 64) + 16 * h * kRow + i / (kTurn / 4) * (kTurn * 16));
    }
    __device__ __forceinline__ Operand read_value(const char* v, int at, int t) const {
        if constexpr (kBf16) return tr_read(v, at, t);
        return __builtin_bit_cast(Operand, row_read(v, t % 8, t / 8));
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
        const int at = kBf16 ? tr_at(lane) : 0;
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

    // A tile of which some row does not see every key: a value that is not finite must not reach such a row as 0 times
    // it. If there are any, those rows that see them get them here, and 0 takes their place.
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

    // The keys k0 .. k0 + 31, at rows k .. of the tile in `stage`.  ALL: every row sees every one of them.
    template <bool ALL>
    __device__ __forceinline__ void step(int stage, int k, int k0, uint32_t there) {
        const char* ks = lds + stage * kStage;
        const char* vs = ks + kTile;
        // (before the products: no branch stands between them and the first use of their results)
        uint32_t sees[RB];
        if (!ALL)
#pragma unroll
            for (int b = 0; b < RB; ++b) sees[b] = seen(b, k0, there) >> (4 * (this->lane >> 4));
        int lane = this->lane;
        if (kTight) asm volatile("" : "+v"(lane));  // (addresses are made again, not kept)
        const int at = (lane & 15) * kRow + ((lane >> 4) ^ k_swizzle(lane & 15)) * 16;
        ks += k * kRow;
        vs += k * kRow;
        Operand x[kDeep];
#pragma unroll
        for (int i = 0; i < kDeep - 1; ++i) x[i] = read_key(ks, at, i);
        f32x4 s[RB][2];
#pragma unroll
        for (int b = 0; b < RB; ++b) s[b][0] = s[b][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kKeys; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            if (i + kDeep - 1 < kKeys) x[(i + kDeep - 1) % kDeep] = read_key(ks, at, i + kDeep - 1);
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                f32x4& z = s[b][i % 2];
                if constexpr (kBf16) {
                    z = mfma(x[i % kDeep], q[b][i / 2], z);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        z = mfma4(__uint_as_float(x[i % kDeep][j]), __uint_as_float(q[b][i / 2][j]), z);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        int vat = kBf16 ? tr_at(lane) : 0;
        asm volatile("" : "+v"(vat));  // (one operation an operand, not a register each)
#pragma unroll
        for (int i = 0; i < kDeep - 1; ++i) x[i] = read_value(vs, vat, i);
        float top[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s[b][i / 4][i % 4] *= c;
                if (!ALL && !(sees[b] >> (16 * (i / 4) + i % 4) & 1)) s[b][i / 4][i % 4] = kNone;
            }
            const f32x4 x = s[b][0], y = s[b][1];
            top[b] = pair_max(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]))));
        }
        bool grows = false;
#pragma unroll
        for (int b = 0; b < RB; ++b) grows |= top[b] > m[b] + kSlack;
        if (__any(grows)) {
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const float now = fmaxf(m[b], top[b]);
                const float f = m[b] == kNone ? 1.0f : exp2_raw(m[b] - now);  // (nothing yet but clean()'s)
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
            const float most = m[b] == kNone ? 0.0f : m[b];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[b][i / 4][i % 4] = exp2_raw(s[b][i / 4][i % 4] - most);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = w[b][i / 2][i % 2 * 2], y = w[b][i / 2][i % 2 * 2 + 1];
                // bf16 weights, off by 2^-8 of each at the most, for the bf16 product with the values (float32 products
                // reach an eighth of its rate): against 64 bits the output is off by 2.1e-3 to 2.2e-3 of its norm, its own
                // rounding alone by 1.7e-3.  The sum takes the rounded ones, so that equal weights leave no error.
                if constexpr (kBf16) {
                    wb[b][i] = round2(x, y);
                    l[b] = sum2(wb[b][i], l[b]);
                } else {
                    l[b] += x;
                    l[b] += y;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            if (i + kDeep - 1 < kValues) x[(i + kDeep - 1) % kDeep] = read_value(vs, vat, i + kDeep - 1);
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                if constexpr (kBf16) {
                    o[b][i] = mfma(x[i % kDeep], wb[b], o[b][i]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f32x4& z = o[b][i / 8 * 4 + j];
                        z = mfma4(__uint_as_float(x[i % kDeep][j]), w[b][i % 8 / 4][i % 4], z);
                    }
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }

    // A run of tiles of keys, a tile ahead.
    int ahead, end, stage;  // the tile whose copy is in flight or done, the first that is not wanted, where it goes
    uint32_t next;          // places of the tile after it
    uint64_t exist;         // its keys that exist
    __device__ __forceinline__ void start(int k0, int k1) {
        arrived();  // (whoever used LDS before is done)
        ahead = k0, end = k1, stage = 0;
        next = key_at(k0 * BN + lane % BN);
        copy(0, next);
        exist = __ballot(next != kNowhere);
        if (k0 + 1 < k1) next = key_at((k0 + 1) * BN + lane % BN);
    }
    __device__ __forceinline__ uint64_t take() {  // tile `ahead` is in LDS -> its keys that exist; the next one is on its way
        const uint64_t now = exist;
        arrived();
        ++ahead;
        stage ^= 1;
        if (ahead < end) {
            copy(stage, next);
            exist = __ballot(next != kNowhere);
            if (ahead + 1 < end) next = key_at((ahead + 1) * BN + lane % BN);
        }
        return now;
    }
    // The products of tile k, in the stage that take() left.
    template <bool ALL>
    __device__ __forceinline__ void steps(int k, uint64_t now) {
#pragma unroll 1
        for (int i = 0; i < BN / 32; ++i) {
            const int from = k * BN + 32 * i;
            if (last_token >= 0 && (ALL || a.mask || from <= t.held + last_token))
                step<ALL>(stage ^ 1, 32 * i, from, (uint32_t)(now >> 32 * i));
        }
    }

    // The tiles of keys k0 .. k1 - 1 of this tile of rows: first those that every row sees, in a loop without masks (but
    // for those with absent pages: they come last).
    __device__ __forceinline__ void run(int k0, int k1, int* flags) {
        if (t.places == 0) return;
        const int seen_by_all = min(a.mask ? t.held : t.held + t.m0 / group + 1, t.places);
        const int full = min(max(seen_by_all / BN, k0), k1);
        int rest = full;
        start(k0, k1);
        load_q();
        for (int k = k0; k < full; ++k) {
            const uint64_t now = take();
            if (now == ~0ull)
                steps<true>(k, now);
            else
                rest = min(rest, k);
        }
        if (full == k1 && rest == full) return;
        load_q();  // (again, so that what the masks need does not push it out of the first loop's registers)
#pragma unroll 1
        for (int part = 0; part < 2; ++part) {
            const int from = part ? rest : full, to = part ? full : k1;
            if (part && from < to) start(from, to);
            for (int k = from; k < to; ++k) {
                const uint64_t now = take();
                if (k < full && now == ~0ull) continue;
                clean(stage ^ 1, k * BN, now, flags);
                steps<false>(k, now);
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

// What bounds it.  Many rows: what a step does one after the other (a prompt of 16,384 tokens, 8 heads of 256, bf16:
// 1.15 ms for 1.1 TFLOP, 0.96 PFLOP/s; matrix cores 42 % of the time, other vector instructions 32, LDS 23).  A step of
// 32 keys by 32 rows of 256 elements is 64 products, 32 KiB from LDS, 16 exponentials a lane and a maximum over lanes;
// two wavefronts a SIMD take turns with them, for more there are no registers.  Tens of rows on thousands of keys: the copies'
// latency and the parts (1,500 drafted tokens of 48 sequences on 100,000 keys, 4 key heads of 128: 79 us for 205 MB, 2.6
// TB/s); one sequence: the latency of finding its share, of a few tiles of keys and of the join (26 tokens on 6,000: 22
// us and 7).  float32: the 16 x 16 x 4 products, 59 % of the time (9 prompts, 3,001 tokens on 5,000, 80 of 128 elements
// used: 87 us).
template <class T, int D, int RB, int W, int BN, bool FULL>
__global__ __launch_bounds__(64 * W) void attn_kernel(attn_dev_args a, AttnPlan p, AttnUnits units) {
    using P = Pass<T, D, RB, W, BN, FULL>;
    __shared__ __attribute__((aligned(1024))) char lds[2 * P::kStage];
    __shared__ int held[ATTN_HELD];
    __shared__ int flags[W];
    const Shape shape{a, p};
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Share share = uniform(share_of(shape, held, p.least));
    AttnDesc* desc = reinterpret_cast<AttnDesc*>(static_cast<char*>(a.work) + p.desc_at) + blockIdx.x;
    float2* stats = reinterpret_cast<float2*>(static_cast<char*>(a.work) + p.stat_at);
    f32x4* parts = reinterpret_cast<f32x4*>(static_cast<char*>(a.work) + p.part_at);
    AttnDesc left{};
    P pass{a, units, p.group, lds, (int)(threadIdx.x & 63), wave};
    pass.c = a.scale * kLog2e;
    int64_t at = share.from, before = share.before;
    int place = share.place, seq = share.seq;
    const int places = shape.places();
    const bool vec = quads<T>(a);
    while (at < share.to && place < places) {
        if (a.starts) seq = next_seq(shape, seq, place);
        const Tile t = uniform(shape.tile(place, seq));
        const int64_t in = at - before, all = (int64_t)t.cost * a.heads_k;
        if (in >= all) {
            before += all;
            place = __builtin_amdgcn_readfirstlane(place_after(shape, held, place));
            continue;
        }
        const int head = (int)quotient(in, t.cost), c0 = (int)(in - (int64_t)head * t.cost);
        const int c1 = (int)min((int64_t)t.cost, c0 + (share.to - at));
        at += c1 - c0;
        const int k0 = max(c0 - (t.cost - t.tiles), 0), k1 = c1 - (t.cost - t.tiles);
        if (k0 >= k1) continue;
        pass.begin(t, head);
        if (t.held >= 0) pass.run(k0, k1, flags);
        asm volatile("s_nop 7\n\ts_nop 7" ::: "memory");  // the last products' results, whatever way the loop was left
        if (k0 == 0 && k1 < t.tiles)
            left = AttnDesc{1, t.first, t.m0, t.count, head,
                            min((int)quotient((at - c1 + t.cost) * share.workers - 1, share.total), share.workers - 1)};
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
                if (threadIdx.x % 64 < 16) stats[(int64_t)slot * p.rows + 16 * block + n] = float2{pass.m[b], sum};
                f32x4* to = parts + ((int64_t)slot * (p.rows / 16) + block) * P::kOut * 64 + (threadIdx.x & 63);
#pragma unroll
                for (int i = 0; i < P::kOut; ++i) to[i * 64] = pass.o[b][i];
            }
        }
    }
    if (threadIdx.x == 0) {
        *desc = left;
        reinterpret_cast<int*>(static_cast<char*>(a.work) + p.flag_at)[blockIdx.x] = left.there;
    }
}

// The workgroup whose share ends in the tile of rows that a workgroup joins: workgroup blockIdx.x; or (p.shared: few
// tiles, and only so many workgroups) the blockIdx.x-th that left one, by their flags.  -1: none.
template <int THREADS>
__device__ __forceinline__ int first_of(const attn_dev_args& a, const AttnPlan& p) {
    const int* flags = reinterpret_cast<const int*>(static_cast<const char*>(a.work) + p.flag_at);
    if (!p.shared) return flags[blockIdx.x] ? (int)blockIdx.x : -1;
    constexpr int kRounds = (ATTN_MOST + THREADS - 1) / THREADS, kWaves = THREADS / 64;
    __shared__ uint64_t sets[kRounds * kWaves];
    bool there[kRounds];
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
        const int at = i * THREADS + threadIdx.x;
        there[i] = at < p.grid && flags[at];
    }
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
        const uint64_t set = __ballot(there[i]);
        if (threadIdx.x % 64 == 0) sets[i * kWaves + threadIdx.x / 64] = set;
    }
    __syncthreads();
    // (a wavefront's lane has a set of 64 flags)
    const int lane = threadIdx.x & 63;
    uint64_t set = lane < kRounds * kWaves ? sets[lane] : 0;
    static_assert(kRounds * kWaves <= 64, "a lane for each set");
    int upto = __popcll(set);
    const int mine = upto;
#pragma unroll
    for (int i = 1; i < kRounds * kWaves; i *= 2) {
        const int x = __shfl_up(upto, i);
        if (lane >= i) upto += x;
    }
    const uint64_t over = __ballot(upto > (int)blockIdx.x);
    if (!over) return -1;
    const int l = __builtin_ctzll(over);
    int left = (int)blockIdx.x - (upto - mine);
    while (left-- > 0 && lane == l) set &= set - 1;
    return l * 64 + __shfl(lane == l ? __builtin_ctzll(set | 1ull << 63) : 0, l);
}

// The parts of a tile of rows, 16 rows to a workgroup: its first part is the last of workgroup first_of(), the others
// are the first of those that follow.  A wavefront has 64 elements of the rows and every G-th part, kAtOnce of them in
// flight; Z wavefronts side by side, D / 64 / Z workgroups.  Bound by the parts' latency where there are few tiles (7
// us for one sequence's 26 tokens in 200 parts), else by their bytes (48 trees: 13 us, a prompt of 16,384 tokens 29).
constexpr int kAtOnce = 4;
template <class T, int D, int G, int Z>
__global__ __launch_bounds__(64 * Z * G) void attn_join_kernel(attn_dev_args a, AttnPlan p) {
    const int first = first_of<64 * Z * G>(a, p);
    if (first < 0) return;
    const AttnDesc d = reinterpret_cast<const AttnDesc*>(static_cast<const char*>(a.work) + p.desc_at)[first];
    const int block = blockIdx.y, m0 = d.m0 + 16 * block;
    if (m0 >= d.count) return;
    constexpr int kOut = D / 16;
    const float2* stats = reinterpret_cast<const float2*>(static_cast<const char*>(a.work) + p.stat_at);
    const f32x4* parts = reinterpret_cast<const f32x4*>(static_cast<const char*>(a.work) + p.part_at);
    __shared__ f32x4 sums[G > 1 ? G - 1 : 1][Z][4][64];
    __shared__ float2 tops[G][Z][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15;
    const int at_z = wave % Z, z = Z * blockIdx.z + at_z, group = wave / Z;
    f32x4 o[4] = {};
    float m = kNone, l = 0;
    if (m0 + n < d.count)
        for (int w0 = first + group; w0 <= d.last; w0 += G * kAtOnce) {
            // (a part past the last: the last again, with no weight)
            float2 s[kAtOnce];
            f32x4 x[kAtOnce][4];
            float now = m;
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const int w = min(w0 + G * j, d.last), slot = w == first ? 2 * first + 1 : 2 * w;
                s[j] = stats[(int64_t)slot * p.rows + 16 * block + n];
                const f32x4* from = parts + (((int64_t)slot * (p.rows / 16) + block) * kOut + 4 * z) * 64 + lane;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[j][i] = from[i * 64];
            }
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j)
                if (w0 + G * j <= d.last) now = fmaxf(now, s[j].x);
            const float f = m == kNone ? 1.0f : exp2_raw(m - now);
            m = now;
            l *= f;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] *= f;
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                if (w0 + G * j > d.last) break;
                const float e = s[j].x == kNone ? 1.0f : exp2_raw(s[j].x - now);  // (values that are not finite alone)
                l += s[j].y * e;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] += x[j][i] * e;
            }
        }
    if constexpr (G > 1) {
        tops[group][at_z][lane] = float2{m, l};
        if (group)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[group - 1][at_z][i][lane] = o[i];
        __syncthreads();
        if (group) return;
        float top = kNone;
#pragma unroll
        for (int g = 0; g < G; ++g) top = fmaxf(top, tops[g][at_z][lane].x);
        const float f = m == kNone ? 1.0f : exp2_raw(m - top);
        l *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= f;
#pragma unroll 3
        for (int g = 1; g < G; ++g) {
            const float2 s = tops[g][at_z][lane];
            const float e = s.x == kNone ? 1.0f : exp2_raw(s.x - top);
            l += s.y * e;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += sums[g - 1][at_z][i][lane] * e;
        }
    }
    const int r = m0 + n, g = lane >> 4;
    if (r >= d.count) return;
    const float f = 1.0f / l;
    T* to = static_cast<T*>(a.out) + (int64_t)(d.first + r / p.group) * a.out_row +
            (int64_t)(d.head * p.group + r % p.group) * a.out_head;
    const bool vec = quads<T>(a);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // (Pass::quad_at)
        const int at = 64 * z + (sizeof(T) == 2 ? 16 * i + 4 * g : 16 * g + 4 * i);
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = l == 0 ? 0.0f : (sizeof(T) == 2 ? o[i][e] : o[e][i]) * f;
        if (at < a.dim) store4(to + at, x, vec);
    }
}

// ---- few rows ----------------------------------------------------------------------------
// Up to 16 rows on a key head: bound by the cache's bytes (64 sequences of 4,096 keys, 2 key heads of 256, bf16: 537 MB
// in 108 us, 5.0 TB/s, where a kernel that only reads the same pages took 88; 139 us when the keys came through LDS), or
// where they are few by the latency of a share (one sequence: 11 us).  Every wavefront has keys of its own, 16 at a time, straight to registers:
// as the left operands of K Q^T and, with float32 weights and values widened, of V^T W^T, whose 16 by 16 by 4 products
// take a lane's 16 bytes of a value as that many products' operands.  (bf16 products of V would need its transpose,
// from LDS: the float32 ones are a third of the time that the bytes take.)  The wavefronts' outputs meet in LDS at the
// end. FULL: heads have D elements.
template <class T, int D, bool FULL>
struct Few {
    static constexpr bool kBf16 = sizeof(T) == 2;
    static constexpr int W = 4;
    static constexpr int E = 16 / sizeof(T);
    static constexpr int kQ = D / (4 * E);               // a lane's parts of a key
    static constexpr int kN = D / 16 < E ? D / 16 : E;   // elements of a lane's part of a value, next to each other
    static constexpr int kV = D / (16 * kN);             // such parts
    static constexpr int kPitch = D + 4;                 // floats of a row in LDS
    using VPart = std::conditional_t<kN * sizeof(T) == 16, u32x4, u32x2>;

    const attn_dev_args& a;
    AttnUnits units;
    int lane, wave;
    Tile t;
    global_char* kbase;
    global_char* vbase;
    const u32x4* q;  // in LDS: part k of lane l at [k][l]
    int token;       // of the lane's row
    f32x4 o[kV][kN];
    float m, l, c;
    u32x4 kr[kQ];
    VPart vr[4][kV];

    __device__ uint32_t key_at(int j) const { return ::key_at(a, units, t, j); }
    // Lane n of 16 reads key n; parts past the head's elements are read as the first and zeroed.
    __device__ __forceinline__ void load_keys(uint32_t at) {
        const int g = lane >> 4;
        using Part = __attribute__((address_space(1))) const u32x4;
        global_char* from = at == kNowhere ? (global_char*)kZeros : in_cache(kbase, at, units);
#pragma unroll
        for (int i = 0; i < kQ; ++i) kr[i] = *(Part*)(from + (FULL || (4 * i + g) * E < a.dim ? (4 * i + g) * 16 : 0));
    }
    // Lane n of 16, group g: elements of key 4 g + i, which is at `at` of lane 4 g + i.
    __device__ __forceinline__ global_char* value_at(uint32_t at, int i) const {
        const uint32_t x = __shfl(at, 4 * (lane >> 4) + i);
        return x == kNowhere ? (global_char*)kZeros : in_cache(vbase, x, units);
    }
    __device__ __forceinline__ void load_value(global_char* from, int i) {
#pragma unroll
        for (int f = 0; f < kV; ++f) {
            const int d = (16 * f + (lane & 15)) * kN;
            vr[i][f] = *(__attribute__((address_space(1))) const VPart*)(from + (FULL || d < a.dim ? d : 0) * (int)sizeof(T));
        }
    }
    __device__ __forceinline__ float value(int i, int f, int j) const {
        if constexpr (!kBf16) return __uint_as_float(vr[i][f][j]);
        const uint32_t x = vr[i][f][j / 2];
        return __uint_as_float(j % 2 ? x & 0xffff0000u : x << 16);
    }

    // Which of the 16 keys from k0 on the lane's row sees, of those that exist (Pass::seen).
    __device__ uint32_t seen(int k0, uint32_t there) const {
        if (!a.mask) {
            const int upto = t.held + token - k0;
            return upto < 0 ? 0 : upto >= 15 ? there : there & ((2u << upto) - 1);
        }
        const int j = k0 - t.held;
        if (j <= -16) return there;
        const int32_t* words = a.mask + (int64_t)(t.first + token) * a.mask_words;
        if (j < 0) {
            const uint32_t w = a.mask_words > 0 ? words[0] : 0;
            return there & (w << -j | ((1u << -j) - 1));
        }
        const int n = j >> 5, sh = j & 31;
        const uint32_t lo = n < a.mask_words ? words[n] : 0, hi = n + 1 < a.mask_words ? words[n + 1] : 0;
        return there & (uint32_t)(((uint64_t)hi << 32 | lo) >> sh);
    }

    // The 16 keys from k0 on, in the registers; next: where the wavefront's next ones are, whose loads begin as soon as
    // the products have read a register.  ALL: every row sees every key.
    template <bool ALL, bool MORE>
    __device__ __forceinline__ void step(int k0, uint32_t there, uint32_t next) {
        const int g = lane >> 4;
        // (before the products, as in Pass::step)
        const uint32_t sees = ALL ? 0xffffu : seen(k0, there);
        f32x4 s = {0, 0, 0, 0};
        if constexpr (kBf16) {
#pragma unroll
            for (int i = 0; i < kQ; ++i) {
                u32x4 x = kr[i];
                if (!FULL) x = (4 * i + g) * E < a.dim ? x : u32x4{0, 0, 0, 0};
                s = mfma(x, q[i * 64 + lane], s);
            }
        } else {
            f32x4 part[4] = {};  // (a product waits for the one before in its sum)
#pragma unroll
            for (int i = 0; i < kQ; ++i) {
                const f32x4 x = __builtin_bit_cast(f32x4, kr[i]), y = __builtin_bit_cast(f32x4, q[i * 64 + lane]);
                const bool in = FULL || (4 * i + g) * E < a.dim;
#pragma unroll
                for (int j = 0; j < 4; ++j) part[j] = mfma4(in ? x[j] : 0.0f, y[j], part[j]);
            }
            s = (part[0] + part[1]) + (part[2] + part[3]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] *= c;
            if (!ALL && !(sees >> (4 * g + i) & 1)) s[i] = kNone;
        }
        const float top = pair_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
        global_char* from[4];
        if (MORE) {
            __builtin_amdgcn_sched_barrier(0);
            load_keys(next);
#pragma unroll
            for (int i = 0; i < 4; ++i) from[i] = value_at(next, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__any(top > m + kSlack)) {
            const float now = fmaxf(m, top);
            const float f = m == kNone ? 1.0f : exp2_raw(m - now);  // (nothing yet but values that are not finite)
            m = now;
            l *= f;
#pragma unroll
            for (int i = 0; i < kV; ++i)
#pragma unroll
                for (int j = 0; j < kN; ++j) o[i][j] *= f;
        }
        const float most = m == kNone ? 0.0f : m;
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = exp2_raw(s[i] - most);
            l += w[i];
        }
        if (!ALL) clean(sees);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int f = 0; f < kV; ++f)
#pragma unroll
                for (int j = 0; j < kN; ++j) o[f][j] = mfma4(value(i, f, j), w[i], o[f][j]);
            if (MORE) {
                __builtin_amdgcn_sched_barrier(0);
                load_value(from[i], i);
            }
        }
    }

    // Values that are not finite: to the rows that see them, and 0 in their place (Pass::clean).
    __device__ __forceinline__ void clean(uint32_t sees) {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int f = 0; f < kV; ++f)
#pragma unroll
                for (int j = 0; j < kN; ++j) odd |= is_odd(value(i, f, j));
        if (!__any(odd)) return;
        float see[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) see[i] = (float)(sees >> (4 * (lane >> 4) + i) & 1);
#pragma unroll
        for (int f = 0; f < kV; ++f) {
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                __builtin_amdgcn_sched_barrier(0);
                f32x4 kinds = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 4; ++i) kinds = mfma4(kind_of(value(i, f, j)), see[i], kinds);
                add_kinds(o[f][j], kinds);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < kN * (int)sizeof(T) / 4; ++j) {
                    if constexpr (kBf16)
                        vr[i][f][j] = round2(finite(value(i, f, 2 * j)), finite(value(i, f, 2 * j + 1)));
                    else
                        vr[i][f][j] = __float_as_uint(finite(value(i, f, j)));
                }
        }
    }
    int group;

    // The tiles of 64 keys k0 .. k1 - 1: keys 16 wave .. of each.  First those that every row sees, in a loop without
    // masks; then the rest (the last ones, and those of absent pages), one by one.
    __device__ __forceinline__ void run(int k0, int k1) {
        const int n = lane & 15;
        auto first = [&](int k) { return k * 16 * W + 16 * wave; };
        auto load = [&](uint32_t at) {
            load_keys(at);
#pragma unroll
            for (int i = 0; i < 4; ++i) load_value(value_at(at, i), i);
        };
        const int spare = min(a.mask ? t.held : t.held + t.m0 / group + 1, t.places) - 16 - 16 * wave;
        const int full = min(max(spare < 0 ? 0 : spare / (16 * W) + 1, k0), k1);
        int rest = full;
        if (k0 < full) {
            // Tables are read two tiles ahead, before the next tile's loads: waiting for them waits for nothing newer.
            uint32_t at = key_at(first(k0) + n), next = k0 + 1 < full ? key_at(first(k0 + 1) + n) : kNowhere;
            load(at);
            int k = k0;
            auto turn = [&](auto more) {
                const uint32_t after = k + 2 < full ? key_at(first(k + 2) + n) : kNowhere;
                if (__all(at != kNowhere)) {
                    step<true, decltype(more)::value>(first(k), 0xffff, next);
                } else {
                    rest = min(rest, k);
                    if (decltype(more)::value) load(next);
                }
                at = next;
                next = after;
                ++k;
            };
            while (k + 1 < full) turn(std::true_type{});
            turn(std::false_type{});  // (apart: with a branch around its loads the compiler would wait for them at once)
        }
        for (int k = rest; k < k1; ++k) {
            const uint32_t at = key_at(first(k) + n), there = (uint32_t)__ballot(at != kNowhere) & 0xffff;
            if (there == 0 || (k < full && there == 0xffff)) continue;
            load(at);
            step<false, false>(first(k), there, kNowhere);
        }
    }
};

// Four consecutive elements of a row of out.
template <class T>
__device__ __forceinline__ void store_row(const attn_dev_args& a, int group, int first, int r, int head, int d, const float (&x)[4]) {
    if (d >= a.dim) return;
    T* to = static_cast<T*>(a.out) + (int64_t)(first + r / group) * a.out_row + (int64_t)(head * group + r % group) * a.out_head + d;
    store4(to, x, quads<T>(a));
}

template <class T, int D, bool FULL>
__global__ __launch_bounds__(256, 2) void attn_step_kernel(attn_dev_args a, AttnPlan p, AttnUnits units) {
    using P = Few<T, D, FULL>;
    __shared__ int held[ATTN_HELD];
    __shared__ u32x4 q[P::kQ * 64];
    __shared__ float2 tops[P::W][16];
    __shared__ __attribute__((aligned(16))) float sums[P::W][16][P::kPitch];
    const Shape shape{a, p};
    const Share share = uniform(share_of(shape, held, p.least));
    AttnDesc* desc = reinterpret_cast<AttnDesc*>(static_cast<char*>(a.work) + p.desc_at) + blockIdx.x;
    float2* stats = reinterpret_cast<float2*>(static_cast<char*>(a.work) + p.stat_at);
    float* parts = reinterpret_cast<float*>(static_cast<char*>(a.work) + p.part_at);
    AttnDesc left{};
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    P few{a, units, lane, wave};
    few.c = a.scale * kLog2e;
    few.q = q;
    few.group = p.group;
    int64_t at = share.from, before = share.before;
    int place = share.place, seq = share.seq;
    const int places = shape.places();
    while (at < share.to && place < places) {
        if (a.starts) seq = next_seq(shape, seq, place);
        const Tile t = uniform(shape.tile(place, seq));
        const int64_t in = at - before, all = (int64_t)t.cost * a.heads_k;
        if (in >= all) {
            before += all;
            place = __builtin_amdgcn_readfirstlane(place_after(shape, held, place));
            continue;
        }
        const int head = (int)quotient(in, t.cost), c0 = (int)(in - (int64_t)head * t.cost);
        const int c1 = (int)min((int64_t)t.cost, c0 + (share.to - at));
        at += c1 - c0;
        const int k0 = max(c0 - (t.cost - t.tiles), 0), k1 = c1 - (t.cost - t.tiles);
        if (k0 >= k1) continue;
        if (k0 == 0 && k1 < t.tiles)
            left = AttnDesc{1, t.first, t.m0, t.count, head,
                            min((int)quotient((at - c1 + t.cost) * share.workers - 1, share.total), share.workers - 1)};
        // q to LDS, a part a thread at a time
        const int rows = min(16, t.count - t.m0);
        few.t = t;
        few.token = (t.m0 + min(n, rows - 1)) / p.group;
        few.kbase = (global_char*)a.key_cache + head * a.cache_head * (int64_t)sizeof(T);
        few.vbase = (global_char*)a.value_cache + head * a.cache_head * (int64_t)sizeof(T);
        const bool vec = ((uintptr_t)a.q | (uint64_t)a.q_row * sizeof(T) | (uint64_t)a.q_head * sizeof(T)) % 16 == 0;
        for (int i = wave; i < P::kQ; i += P::W) {
            const int r = t.m0 + min(n, rows - 1), d = (4 * i + g) * P::E;
            const T* from = static_cast<const T*>(a.q) + (int64_t)(t.first + r / p.group) * a.q_row +
                            (int64_t)(head * p.group + r % p.group) * a.q_head + d;
            u32x4 x = {0, 0, 0, 0};
            if (d < a.dim) {
                if (vec)
                    x = *reinterpret_cast<const u32x4*>(from);
                else
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if constexpr (P::kBf16)
                            x[j] = from[2 * j] | (uint32_t)from[2 * j + 1] << 16;
                        else
                            x[j] = __float_as_uint(from[j]);
                    }
            }
            q[i * 64 + lane] = x;
        }
        few.m = kNone;
        few.l = 0;
#pragma unroll
        for (int f = 0; f < P::kV; ++f)
#pragma unroll
            for (int j = 0; j < P::kN; ++j) few.o[f][j] = f32x4{0, 0, 0, 0};
        __syncthreads();
        if (t.held >= 0) few.run(k0, k1);
        asm volatile("s_nop 7\n\ts_nop 7" ::: "memory");  // the last products' results, whatever way the loop was left
        // a row's maximum over the wavefronts, and what each has, scaled to it
        const float sum = pair_sum(few.l);
        if (g == 0) tops[wave][n] = float2{few.m, sum};
        __syncthreads();
        float top = kNone;
#pragma unroll
        for (int w = 0; w < P::W; ++w) top = fmaxf(top, tops[w][n].x);
        const float f = few.m == kNone ? 1.0f : exp2_raw(few.m - top);
        if (n < rows)
#pragma unroll
            for (int v = 0; v < P::kV; ++v)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < P::kN; j += 4)
                        *reinterpret_cast<f32x4*>(&sums[wave][n][(16 * v + 4 * g + e) * P::kN + j]) =
                            f32x4{few.o[v][j][e], few.o[v][j + 1][e], few.o[v][j + 2][e], few.o[v][j + 3][e]} * f;
        __syncthreads();
        const int slot = 2 * blockIdx.x + (k0 == 0);
        for (int i = threadIdx.x; i < rows * (D / 4); i += 256) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            f32x4 x = {0, 0, 0, 0};
            float most = kNone, all_l = 0;
#pragma unroll
            for (int w = 0; w < P::W; ++w) {
                x += *reinterpret_cast<const f32x4*>(&sums[w][r][d]);
                most = fmaxf(most, tops[w][r].x);
            }
#pragma unroll
            for (int w = 0; w < P::W; ++w) {
                const float2 s = tops[w][r];
                all_l += s.x == kNone ? s.y : s.y * exp2_raw(s.x - most);  // (no maximum: no sum, or every score NaN)
            }
            if (k0 == 0 && k1 == t.tiles) {
                const float y = 1.0f / all_l;
                float z[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) z[e] = all_l == 0 ? 0.0f : x[e] * y;
                store_row<T>(a, p.group, t.first, t.m0 + r, head, d, z);
            } else {
                *reinterpret_cast<f32x4*>(parts + ((int64_t)slot * 16 + r) * D + d) = x;
                if (d == 0) stats[slot * 16 + r] = float2{most, all_l};
            }
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        *desc = left;
        reinterpret_cast<int*>(static_cast<char*>(a.work) + p.flag_at)[blockIdx.x] = left.there;
    }
}

// The parts of a row, a row to a workgroup: D / 4 lanes have every G-th part, kAtOnce of them in flight.  Latency: 5 us.
template <class T, int D, int G>
__global__ __launch_bounds__(G * (D / 4)) void attn_step_join_kernel(attn_dev_args a, AttnPlan p) {
    const int first = first_of<G * (D / 4)>(a, p);
    if (first < 0) return;
    const AttnDesc d = reinterpret_cast<const AttnDesc*>(static_cast<const char*>(a.work) + p.desc_at)[first];
    const int r = blockIdx.y;
    if (d.m0 + r >= d.count) return;
    const float2* stats = reinterpret_cast<const float2*>(static_cast<const char*>(a.work) + p.stat_at);
    const float* parts = reinterpret_cast<const float*>(static_cast<const char*>(a.work) + p.part_at);
    __shared__ f32x4 sums[G][D / 4];
    __shared__ float2 tops[G];
    const int lane = threadIdx.x % (D / 4), group = threadIdx.x / (D / 4);
    f32x4 o = {0, 0, 0, 0};
    float m = kNone, l = 0;
    for (int w0 = first + group; w0 <= d.last; w0 += G * kAtOnce) {
        float2 s[kAtOnce];
        f32x4 x[kAtOnce];
        float now = m;
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {  // (past the last: the last again, with no weight)
            const int w = min(w0 + G * j, d.last), slot = w == first ? 2 * first + 1 : 2 * w;
            s[j] = stats[slot * 16 + r];
            x[j] = *reinterpret_cast<const f32x4*>(parts + ((int64_t)slot * 16 + r) * D + 4 * lane);
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
            if (w0 + G * j <= d.last) now = fmaxf(now, s[j].x);
        const float f = m == kNone ? 1.0f : exp2_raw(m - now);
        m = now;
        l *= f;
        o *= f;
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            if (w0 + G * j > d.last) break;
            const float e = s[j].x == kNone ? 1.0f : exp2_raw(s[j].x - now);  // (values that are not finite alone)
            l += s[j].y * e;
            o += x[j] * e;
        }
    }
    sums[group][lane] = o;
    if (lane == 0) tops[group] = float2{m, l};
    __syncthreads();
    if (group) return;
    float top = kNone, all = 0;
#pragma unroll
    for (int w = 0; w < G; ++w) top = fmaxf(top, tops[w].x);
    f32x4 x = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < G; ++w) {
        const float e = tops[w].x == kNone ? 1.0f : exp2_raw(tops[w].x - top);
        all += tops[w].y * e;
        x += sums[w][lane] * e;
    }
    const float y = 1.0f / all;
    float z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = all == 0 ? 0.0f : x[e] * y;
    store_row<T>(a, p.group, d.first, d.m0 + r, d.head, 4 * lane, z);
}

template <class T, int D>
hipError_t launch_step(const attn_dev_args& a, const AttnPlan& p, hipStream_t s) {
    const AttnUnits units = attn_units(a);
    if (a.dim == D)
        attn_step_kernel<T, D, true><<<dim3((unsigned)p.grid), 256, 0, s>>>(a, p, units);
    else
        attn_step_kernel<T, D, false><<<dim3((unsigned)p.grid), 256, 0, s>>>(a, p, units);
    const dim3 grid((unsigned)(p.shared ? p.shared : p.grid), (unsigned)std::min(16, p.rows_most));
    if (p.shared)
        attn_step_join_kernel<T, D, 16><<<grid, 4 * D, 0, s>>>(a, p);
    else
        attn_step_join_kernel<T, D, 4><<<grid, D, 0, s>>>(a, p);
    return hipGetLastError();
}

template <class T, int D, int RB, int W, int BN>
hipError_t launch(const attn_dev_args& a, const AttnPlan& p, hipStream_t s) {
    const AttnUnits units = attn_units(a);
    if (a.dim == D)
        attn_kernel<T, D, RB, W, BN, true><<<dim3((unsigned)p.grid), 64 * W, 0, s>>>(a, p, units);
    else
        attn_kernel<T, D, RB, W, BN, false><<<dim3((unsigned)p.grid), 64 * W, 0, s>>>(a, p, units);
    const unsigned blocks = (std::min(p.rows, p.rows_most) + 15) / 16;
    if (p.shared)
        attn_join_kernel<T, D, 16, 1><<<dim3(p.shared, blocks, D / 64), 1024, 0, s>>>(a, p);
    else
        attn_join_kernel<T, D, 1, D / 64><<<dim3(p.grid, blocks), D, 0, s>>>(a, p);
    return hipGetLastError();
}

template <int D>
hipError_t launch_bf16(const attn_dev_args& a, const AttnPlan& p, hipStream_t s) {
    if (p.few) return launch_step<uint16_t, D>(a, p, s);
    if (p.waves == 2) return launch<uint16_t, D, 2, 2, 32>(a, p, s);
    if constexpr (D < 256)
        if (p.waves == 4) return launch<uint16_t, D, 2, 4, 32>(a, p, s);
    return launch<uint16_t, D, 2, 8, 64>(a, p, s);
}
template <int D>
hipError_t launch_f32(const attn_dev_args& a, const AttnPlan& p, hipStream_t s) {
    if (p.few) return launch_step<float, D>(a, p, s);
    switch (p.waves) {
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
