// attn.h -- what the attention kernels share: a call's arguments, a sequence's bounds, the LDS tile of
// token rows and the MFMA operands read from it.
//
// Products. Scores and probabilities are kept transposed, S^T [keys, queries] = K . Q^T, by
// v_mfma_f32_32x32x16_bf16: a lane's 16 results of a 32 x 32 tile then belong to one query (column
// lane % 32), at the keys 8 (i / 4) + 4 (lane / 32) + i % 4. A query's maximum and sum are a lane's own
// values and one exchange with lane ^ 32, and the probabilities, rounded to bf16, already lie as the B
// operand of the next product, O^T = V^T . P^T: of the 16 keys of a k step a lane holds 4h .. 4h+3 and
// 8+4h .. 8+4h+3 (h = lane / 32), and since a product's reduction may run in any order, the A operand
// V^T is read in that same order: two transposed LDS reads (ds_read_b64_tr_b16) of four keys each. No
// probability passes through LDS. The backward's products use the same two shapes.
//
// Rows. Query heads that share a key head are walked as one list of rows: row r is the head r % G of
// the group at token r / G. A tile of 128 rows then reads each key once for all its heads, and under a
// causal mask it spans 128 / G tokens.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <utility>

#include "../../include/r97q.h"
#include "iqr_device.h"

namespace r97q {
namespace attn {

using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using s16x8 = __attribute__((ext_vector_type(8))) short;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMostSplits = 256;  // ranges of the keys that the forward's join adds
constexpr int64_t kMostHeads = 1 << 23;  // query heads in all the sequences

// workgroups of `threads` in a launch's first dimension: their threads in all stay below 2^32. The kernels' tile loops take
// what a grid cut short leaves.
constexpr int64_t most_groups(int threads) { return 0xFFFFFFFFLL / threads; }
static_assert(most_groups(256) >= kMostHeads, "a workgroup for every head");

// one tensor of heads: element (b, t, h, d) at data[b * bs + t * ts + h * hs + d]
struct Heads {
    uint8_t* data;
    int64_t bs, ts, hs;
    int32_t f32;  // elements are f32 (outputs), else bf16
};

struct Args {
    Heads q, k, v, o;    // o: the forward's output, written there and read in the backward
    Heads d_o, dq, dk, dv;
    float* lse;          // [b][h][Lq], packed: [h][q_tokens]
    float* base;         // backward: the log-sum-exp in base 2 (0 for a row that sees nothing), laid out as lse
    float* delta;        // and minus the sum over d of dO * O
    // the backward cut over the other side's steps where its grids are small: partial sums in f32, added in order
    int32_t q_splits, k_splits;
    int64_t kv_slots;    // rows of one dk or dv partial
    float *dq_part, *dk_part, *dv_part;  // [splits][slots][d]
    // dS^T kept between the launches, bf16: a query head's row of `pitch` tokens for each key; null: computed again
    uint16_t* ds;
    int64_t pitch;
    int32_t batch, hq, hk, g, d;
    int32_t lq, lk;      // tokens of a sequence (packed: of the longest)
    const int32_t* q_starts;
    const int32_t* kv_starts;
    const int32_t* kv_lens;
    int64_t q_tokens, kv_tokens;
    int32_t causal;
    int32_t window;      // 0: none
    float scale;         // of the scores
    // the forward split over the keys: ranges of `chunk` keys, each one's unnormalised sums in f32 and (m, l)
    int32_t splits, chunk;
    int32_t together;    // heads an XCD takes at a time
    int64_t slots;       // rows of one range: every query head's
    float* part;         // [splits][slots][d]
    float2* stats;       // [splits][slots]
    // a paged cache: k and v are pools of pages (bs: values from page to page, ts: from token to token in one), and a sequence's
    // tokens lie in the pages that its row of the table names
    const int32_t* table;
    int64_t table_stride;
    int32_t pages, max_pages, page_shift;
    int32_t held;        // the longest sequence's keys, for the plan
};

// What the launches are cut by: tiles of `tile` rows or keys in all sequences together, and a sequence's tokens. Packed
// sequences go by their tokens in all, not by the longest.
inline int64_t all_tiles(bool packed, int64_t tokens, int64_t len, int64_t batch, int64_t each, int64_t tile) {
    return packed ? (tokens * each + tile - 1) / tile : batch * ((len * each + tile - 1) / tile);
}
inline int64_t mean_len(bool packed, int64_t tokens, int64_t len, int64_t batch) { return packed ? (tokens + batch - 1) / batch : len; }

// one sequence: its tokens' places and counts. Starts and lengths come from device memory, so they are
// clamped to the tensors: nothing is read or written past them whatever they hold.
struct Seq {
    int32_t b;
    int32_t q_base, k_base;  // token offsets (packed) into the whole tensors; 0 in the dense form
    int32_t lq, lk, off;     // off: query i stands at key position i + off
};

__device__ __forceinline__ int64_t clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// the same value, but what follows from it is computed here: otherwise the many comparisons with the head's width
// that a row's loads and stores make are computed once, before the loop, and held in registers through it
__device__ __forceinline__ int fresh(int x) {
    asm volatile("" : "+s"(x));
    return x;
}
__device__ __forceinline__ int fresh_lane(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ Seq sequence(const Args& a, int b) {
    Seq s;
    s.b = b;
    s.q_base = s.k_base = 0;
    s.lq = a.lq;
    s.lk = a.lk;
    if (a.q_starts) {  // starts are int32: a tensor's tokens past 2^31 - 1 are out of their reach
        s.q_base = (int)clamp64(uniform(a.q_starts[b]), 0, a.q_tokens);
        s.lq = (int)clamp64(uniform(a.q_starts[b + 1]), s.q_base, a.q_tokens > s.q_base ? a.q_tokens : s.q_base) - s.q_base;
        // a key head's rows stay inside 31 bits whatever the starts hold
        const int most = 0x7FFFFF00 / a.g;
        if (s.lq > most) s.lq = most;
    }
    if (a.kv_starts) {
        s.k_base = (int)clamp64(uniform(a.kv_starts[b]), 0, a.kv_tokens);
        s.lk = (int)clamp64(uniform(a.kv_starts[b + 1]), s.k_base, a.kv_tokens > s.k_base ? a.kv_tokens : s.k_base) - s.k_base;
        if (s.lk > 0x7FFFFF00) s.lk = 0x7FFFFF00;
    } else if (a.kv_lens) {
        s.lk = (int)clamp64(uniform(a.kv_lens[b]), 0, a.lk);
    }
    s.off = s.lk - s.lq;
    return s;
}

// the sequence's first token of head h
__device__ __forceinline__ uint8_t* q_at(const Heads& t, const Args& a, const Seq& s, int h) {
    const int64_t e = (a.q_starts ? s.q_base * t.ts : s.b * t.bs) + h * t.hs;
    return t.data + (t.f32 ? 4 * e : 2 * e);
}
__device__ __forceinline__ uint8_t* kv_at(const Heads& t, const Args& a, const Seq& s, int h) {
    const int64_t e = (a.kv_starts ? s.k_base * t.ts : s.b * t.bs) + h * t.hs;
    return t.data + (t.f32 ? 4 * e : 2 * e);
}
// where a row's log-sum-exp (and delta) lies
__device__ __forceinline__ int64_t stat_at(const Args& a, const Seq& s, int h, int token) {
    return a.q_starts ? h * a.q_tokens + s.q_base + token : ((int64_t)s.b * a.hq + h) * a.lq + token;
}

// Which key head of which sequence a workgroup of a one-dimensional grid takes, and which part of it (the first parts
// have the most work). Workgroups go to the 8 XCDs in turn, each with its own L2: where the heads divide evenly, an XCD
// takes `together` of its heads at a time, as many as its L2 holds the keys and values of, part by part, then the next.
struct Place {
    int bh, part;
    __device__ __forceinline__ Place(int nb, int together) {
        const int w = blockIdx.x, parts = gridDim.x / nb;
        if (nb % 8 == 0) {
            const int i = w / 8, group = i / (together * parts), j = i - group * together * parts;
            const int left = nb / 8 - group * together, heads = left < together ? left : together;
            part = j / heads;
            bh = w % 8 + 8 * (group * together + (j - part * heads));
        } else {
            part = w / nb;
            bh = w - part * nb;
        }
    }
};
// a key's row of a partial sum
__device__ __forceinline__ int64_t kv_slot(const Args& a, const Seq& s, int hk, int key) {
    return a.kv_starts ? hk * a.kv_tokens + s.k_base + key : ((int64_t)s.b * a.hk + hk) * a.lk + key;
}

// the kept dS^T: where the row of a head's key begins, at the sequence's token 0. Packed sequences begin on 64 tokens.
__device__ __forceinline__ uint16_t* ds_at(const Args& a, const Seq& s, int head, int key) {
    const int64_t row = a.kv_starts ? head * a.kv_tokens + s.k_base + key : ((int64_t)s.b * a.hq + head) * a.lk + key;
    const int64_t col = a.q_starts ? (s.q_base + 63LL) / 64 * 64 + 64LL * s.b : 0;
    return a.ds + row * a.pitch + col;
}
// dK's and dV's tiles of RT tokens for 128 keys from w0: the first one's token, a multiple of RT, and the tokens' end
__device__ __forceinline__ void tokens_of(const Args& a, const Seq& s, int w0, int rt, int& t0, int& t1) {
    const int wend = w0 + 127 < s.lk ? w0 + 127 : s.lk - 1;
    t0 = 0;
    t1 = s.lq;
    if (a.causal) t0 = (int)clamp64((int64_t)w0 - s.off, 0, s.lq) / rt * rt;
    if (a.window) t1 = (int)clamp64((int64_t)wend + a.window - s.off, t0, s.lq);
    if (w0 >= s.lk) t1 = t0;
}

// the keys [lo, hi) that some of the queries at tokens [t0, t1] see (hi <= lo: none), and [all_lo, all_hi)
// that all of them see
struct Keys {
    int lo, hi, all_lo, all_hi;
};
__device__ __forceinline__ Keys keys_of(const Args& a, const Seq& s, int t0, int t1) {
    Keys k = {0, s.lk, 0, s.lk};
    if (a.causal) {
        k.hi = (int)clamp64((int64_t)t1 + s.off + 1, 0, s.lk);
        k.all_hi = (int)clamp64((int64_t)t0 + s.off + 1, 0, s.lk);
    }
    if (a.window) {
        k.lo = (int)clamp64((int64_t)t0 + s.off - a.window + 1, 0, s.lk);
        k.all_lo = (int)clamp64((int64_t)t1 + s.off - a.window + 1, 0, s.lk);
    }
    return k;
}

// instructions stay on their side
__device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0); }
__device__ __forceinline__ f32x16 mfma(bf16x8 x, bf16x8 y, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
}
// The same with the accumulator in the accumulation registers (ACC: a kernel of one wave a SIMD, whose other registers are
// all taken). In assembly because the compiler otherwise moves operands and sums back and forth between the two files.
// It does not see the instruction's latency: the operands are written a product or more before, the sums are read only
// after settled().
template <bool ACC>
__device__ __forceinline__ void add_product(bf16x8 x, bf16x8 y, f32x16& c) {
    if constexpr (ACC)
        asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(x), "v"(y));
    else
        c = mfma(x, y, c);
}
// fragments settle in whole registers, or their words are gathered anew for every product
template <int N>
__device__ __forceinline__ void settle(bf16x8 (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}
// the sums may be read from here on, each after its own settle_sum(): otherwise all are copied out at once, and what
// else is held has to leave the registers
template <bool ACC>
__device__ __forceinline__ void settled() {
    if constexpr (ACC) asm volatile("s_nop 15\n\ts_nop 15");
}
template <bool ACC>
__device__ __forceinline__ void settle_sum(f32x16& c) {
    if constexpr (ACC) {
        pin();
        asm volatile("" : "+a"(c));
    }
}
__device__ __forceinline__ bf16x8 as_bf16x8(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
    bf16x2 v = {(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, v);
}
// a 32 x 32 tile's 16 values of a lane, rounded to bf16: B operands of the two 16-deep k steps
__device__ __forceinline__ void pack_tile(const f32x16& p, bf16x8 (&out)[2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack_bf16(p[8 * c + 2 * j], p[8 * c + 2 * j + 1]);
        out[c] = as_bf16x8(w);
    }
}
// max and sum of the lanes 32 apart, in both of them. (The swap's two results are taken as values first:
// a bit cast of a vector's element reads element 0.)
__device__ __forceinline__ void pair_of(float x, float& lo, float& hi) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = s[0], b = s[1];
    lo = __builtin_bit_cast(float, a);
    hi = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float pair_max(float x) {
    float lo, hi;
    pair_of(x, lo, hi);
    return fmaxf(lo, hi);
}
__device__ __forceinline__ float pair_sum(float x) {
    float lo, hi;
    pair_of(x, lo, hi);
    return lo + hi;
}

// ---------------------------------------------------------------- LDS tiles of token rows
// Rows of D bf16 values. A row's 16-byte chunks are stored at chunk ^ f(row): the 16 rows that 16 lanes
// of a row read (ds_read_b128) take at one chunk, and the 4 rows x 64 bytes that 32 lanes of a
// transposed read take, then lie on different banks. Rows of 128 bytes share a 256-byte bank line two
// by two, so there f goes by the row's pair.
template <int D>
struct Tile {
    static constexpr int RB = 2 * D;       // bytes a row
    static constexpr int CH = D / 8;       // chunks a row
    static __device__ __forceinline__ int f(int row) {
        if constexpr (D == 64) return ((row >> 1) & 1) << 2 | ((row >> 2) & 3);
        return (row & 3) << 2 | ((row >> 2) & 3);
    }
    static __device__ __forceinline__ int at(int row, int chunk) { return row * RB + ((chunk ^ f(row)) << 4); }
    // rows [r0, r0 + 32) as an MFMA operand along d: row r0 + lane % 32, elements 16 c + 8 h .. + 8
    static __device__ __forceinline__ bf16x8 rows(const uint8_t* t, int r0, int c, int lane) {
        return as_bf16x8(*reinterpret_cast<const u32x4*>(t + at(r0 + (lane & 31), 2 * c + (lane >> 5))));
    }
    // rows [r0, r0 + 16) as an MFMA operand along the rows, for the columns 32 db + lane % 32: rows
    // 4h .. 4h+3 and 8+4h .. 8+4h+3
    static __device__ __forceinline__ bf16x8 cols(const uint8_t* t, int r0, int db, int lane) {
        const int l = lane & 15, row = r0 + 4 * (lane >> 5) + (l >> 2);
        const int chunk = 4 * db + 2 * ((lane >> 4) & 1) + ((l & 3) >> 1), in = 8 * (l & 1);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(t + at(row, chunk) + in));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(t + at(row + 8, chunk) + in));
        const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        return __builtin_bit_cast(bf16x8, v);
    }
};

// The same operands by LDS address, for the loops that place every instruction themselves. Tiles start on 1024 bytes,
// so a chunk's place differs from the first chunk's by an exclusive or of the address: one register a lane and
// operand kind, and one or two vector instructions a read.
template <int D>
struct Frags {
    static constexpr int RB = 2 * D;
    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
    // offsets in a tile: rows(), and cols()
    static __device__ __forceinline__ uint32_t row0(int lane) { return Tile<D>::at(lane & 31, lane >> 5); }
    static __device__ __forceinline__ uint32_t col0(int lane) {
        const int l = lane & 15;
        return Tile<D>::at(4 * (lane >> 5) + (l >> 2), 2 * ((lane >> 4) & 1) + ((l & 3) >> 1)) + 8 * (l & 1);
    }
    // rows [r0, r0 + 32), elements 16 c + 8 h .. + 8
    template <int R0, int C>
    static __device__ __forceinline__ bf16x8 rows(uint32_t at0) {
        constexpr int per = D == 64 ? 4 : 8;
        return as_bf16x8(*(lds_u32x4*)(uintptr_t)((at0 ^ (32 * (C % per))) + (C / per) * 256 + R0 * RB));
    }
    // rows R0 + 4h .. and R0 + 8 + 4h .., columns 32 DB + lane % 32
    template <int R0, int DB>
    static __device__ __forceinline__ bf16x8 cols(uint32_t at0) {
        constexpr int per = D == 64 ? 2 : 4;
        const uint32_t lo = at0 ^ (64 * (DB % per)), hi = at0 ^ (64 * (DB % per) + 32);
        constexpr int off = (DB / per) * 256 + R0 * RB;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(lo + off));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(hi + off + 8 * RB));
        const s16x8 v = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        return __builtin_bit_cast(bf16x8, v);
    }
};
// f(0), f(1), .. f(N - 1) with constant indices, unrolled
template <class F, int... I>
__device__ __forceinline__ void steps_of(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void steps(F&& f) {
    steps_of(f, std::make_integer_sequence<int, N>{});
}
// a 32 x 32 tile's values e and e + 1 (e even) as a word of its B operands
__device__ __forceinline__ void pack_two(const f32x16& x, int e, u32x4 (&out)[2]) { out[e >> 3][(e & 7) >> 1] = pack_bf16(x[e], x[e + 1]); }

// ---------------------------------------------------------------- memory -> LDS
// Rows of tokens in memory as a buffer that ends with the last token in use: a load past it, like one of the
// columns past the head's d, gives zeros, so nothing past a sequence is read and no row needs a clamp.
constexpr uint32_t kNowhere = 0x80000000u;  // an offset past every buffer's end
struct Rows {
    uint64_t p;          // the next tile's first token
    uint32_t ts, tail;   // bytes a token, and of the head in use
    int left;            // tokens in use from there on
    // from token row0 of `rows` on; ts2: bytes a token
    __device__ __forceinline__ Rows(const uint8_t* base, int64_t ts2, int row0, int rows, int d)
        : p(reinterpret_cast<uint64_t>(base) + row0 * ts2), ts((uint32_t)ts2), tail(2 * d), left(rows - row0) {}
    __device__ __forceinline__ void step(int tokens) {
        p += (uint64_t)ts * (uint32_t)tokens;
        left -= tokens;
    }
    // a tile of R tokens
    template <int R>
    __device__ __forceinline__ u32x4 buffer() const {
        const uint32_t whole = (R - 1) * ts + tail, part = left > 0 ? (uint32_t)(left - 1) * ts + tail : 0u;
        return (u32x4){(uint32_t)uniform((int)p), (uint32_t)uniform((int)(p >> 32)), (uint32_t)uniform((int)(left >= R ? whole : part)), 0x00020000u};
    }
};

// the LDS address of a pointer into LDS
__device__ __forceinline__ uint32_t lds_at(const void* p) {
    return (uint32_t)uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p);
}
// 64 pieces of 16 bytes, a lane's at `off` of the buffer, to LDS dst + 16 lane. In assembly because the compiler would
// wait for every such load before the next LDS read; the waits are landed()'s, at the loops' barriers. m0 is not put
// back: nothing else in these kernels uses it.
__device__ __forceinline__ void load_piece(const u32x4& buf, uint32_t off, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(buf), "s"(dst));
}
// 64 values of 4 bytes
__device__ __forceinline__ void load_words(const u32x4& buf, uint32_t off, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(off), "s"(buf), "s"(dst));
}
// all but the newest N loads have landed in LDS
template <int N = 0>
__device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// The same of a sequence's tokens in pages. A wave holds 64 entries of the sequence's row of the table, a lane's each: tiles
// begin at multiples of their size, so a tile's pages are of one such block. The next 64 wait in LDS, loaded like the tiles
// (an ordinary load on its way through the loop would have every step wait for all that it has asked for). An entry outside
// the pool reads as zeros, like a token past the end. The keys' walk leads, and loads the entries for the values' too, which
// is at most two tiles behind: less than a block.
constexpr int kTableBytes = 2 * 64 * 4;  // of LDS, a wave
struct PageTable {
    u32x4 row;             // the sequence's row of the table
    uint32_t area, pos;    // the wave's LDS; the next tile's first token
    int from, end;         // tokens to read
    int shift, pages;
    bool leads;
    uint32_t block;
    int ent;               // the lane's entry of the block
    __device__ __forceinline__ PageTable(const Args& a, const Seq& s, int row0, int from_, int rows, uint32_t lds, bool leads_)
        : area(lds), pos(row0), from(from_), end(rows), shift(a.page_shift), pages(a.pages), leads(leads_) {
        const uint64_t p = reinterpret_cast<uint64_t>(a.table + s.b * a.table_stride);
        row = (u32x4){(uint32_t)uniform((int)p), (uint32_t)uniform((int)(p >> 32)), (uint32_t)uniform(4 * a.max_pages), 0x00020000u};
        block = pos >> shift >> 6;
        if (leads) {
            fetch(block);
            fetch(block + 1);
            landed();
        }
        take();
    }
    __device__ __forceinline__ void fetch(uint32_t b) const { load_words(row, 256 * b + 4 * (threadIdx.x & 63), area + 256 * (b & 1)); }
    __device__ __forceinline__ void take() {
        ent = *(__attribute__((address_space(3))) const volatile int*)(uintptr_t)(area + 256 * (block & 1) + 4 * (threadIdx.x & 63));
    }
    __device__ __forceinline__ int size() const { return 1 << shift; }
    __device__ __forceinline__ void step(int tokens) { pos += tokens; }
    __device__ __forceinline__ bool turn() {
        const uint32_t b = pos >> shift >> 6;
        if (b == block) return false;
        block = b;
        take();
        if (leads) fetch(b + 1);
        return true;
    }
    __device__ __forceinline__ uint32_t entry(uint32_t at) const { return __builtin_amdgcn_readlane(ent, (int)(at >> shift) & 63); }
};
// How a pool's pages are reached: one buffer with a page's offset in it, where the pool is less than 2 GiB, a tile's page looked
// up once (kWholePages: they hold a tile) or a wave's piece at a time (kSmallPages: of a tile's first one on); else a piece's
// page as a buffer of its own (kFarPages). What a step does for it counts, since no product runs beside it: 2048 tokens over
// 16384, 16 over 4 heads of 128, 277 us over rows, 286 over pages of 64, of 16 and of 8 some 2% more (275 in two ranges); with every piece's page
// and bounds worked out in scalars 374 (64), and with the next entries an ordinary load 415.
enum { kWholePages, kSmallPages, kFarPages };
constexpr uint32_t kNearBytes = 0x7FFFFFF0u;  // a near pool's end at most: an offset for entries outside the pool
template <int MODE>
struct PageRows : PageTable {
    u32x4 pool;            // near: the pool from the head on
    uint64_t base, page;   // the head in page 0; bytes from page to page
    uint32_t ts, tail;
    __device__ __forceinline__ PageRows(const Args& a, const Seq& s, const Heads& t, int h, int row0, int from_, int rows, int d,
                                        uint32_t lds, bool leads_)
        : PageTable(a, s, row0, from_, rows, lds, leads_), base(reinterpret_cast<uint64_t>(t.data) + 2 * h * t.hs), page(2 * t.bs),
          ts((uint32_t)(2 * t.ts)), tail(2 * d) {
        if constexpr (MODE != kFarPages) {
            const uint32_t n = pages > 0 ? (uint32_t)(pages - 1) * (uint32_t)page + (uint32_t)(size() - 1) * ts + tail : 0u;
            pool = (u32x4){(uint32_t)uniform((int)base), (uint32_t)uniform((int)(base >> 32)), (uint32_t)uniform((int)n), 0x00020000u};
            place();
        }
    }
    // near: the entry as an offset
    __device__ __forceinline__ void place() {
        ent = (uint32_t)ent < (uint32_t)pages ? (int)((uint32_t)ent * (uint32_t)page) : (int)kNearBytes;
    }
    __device__ __forceinline__ void turn() {
        if (!PageTable::turn()) return;
        if constexpr (MODE != kFarPages) place();
    }
    // the buffer of the tile's tokens first .. first + R - 1, in one page, at the tile's offsets
    template <int R>
    __device__ __forceinline__ u32x4 buffer(int first) const {
        const uint32_t at = pos + first, e = entry(at);
        const int left = end - (int)at;
        const uint64_t p = base + (uint64_t)e * page + (int64_t)((int)(at & (size() - 1)) - first) * ts;
        const uint32_t n = (uint32_t)(first + (left < R ? left : R) - 1) * ts + tail;
        return (u32x4){(uint32_t)uniform((int)p), (uint32_t)uniform((int)(p >> 32)),
                       (uint32_t)uniform(e < (uint32_t)pages && left > 0 ? (int)n : 0), 0x00020000u};
    }
};

// ROWS rows from memory into a tile, by THREADS threads: a piece's place in LDS is its thread's, so the swizzle
// is in which chunk of the row a thread loads.
template <int D, int ROWS, int THREADS>
struct Loader {
    static constexpr int CH = Tile<D>::CH, N = ROWS * CH / THREADS;  // pieces a thread
    static_assert(N * THREADS == ROWS * Tile<D>::CH, "whole pieces");
    uint32_t off[N];
    __device__ __forceinline__ Loader(int64_t ts2, int d, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int p = tid + THREADS * i, row = p / Tile<D>::CH, ch = (p % Tile<D>::CH) ^ Tile<D>::f(row);
            off[i] = 8 * ch < d ? (uint32_t)(row * ts2) + 16 * ch : kNowhere;
        }
    }
    // dst: the tile's LDS address + 1024 * the wave's index
    __device__ __forceinline__ void load(const Rows& r, uint32_t dst) const {
        const u32x4 b = r.template buffer<ROWS>();
#pragma unroll
        for (int i = 0; i < N; ++i) load_piece(b, off[i], dst + 16 * THREADS * i);
    }
    // The same from pages; w0: the wave's first thread. FIRST: the tile may hold tokens that no query sees.
    template <bool FIRST, int MODE>
    __device__ __forceinline__ void load_pages(PageRows<MODE>& r, int w0, uint32_t dst) const {
        r.turn();
        if constexpr (MODE == kFarPages) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const u32x4 b = r.template buffer<64 / CH>((w0 + THREADS * i) / CH);
                load_piece(b, FIRST && row_of(i, w0) < r.from - (int)r.pos ? kNowhere : off[i], dst + 16 * THREADS * i);
            }
            return;
        }
        const int left = r.end - (int)r.pos;
        if constexpr (MODE == kWholePages) {
            const uint32_t e = r.entry(r.pos), add = e == kNearBytes ? e : e + (r.pos & (r.size() - 1)) * r.ts;
            const uint32_t last = add + (uint32_t)(left - 1) * r.ts + r.tail;
            u32x4 b = r.pool;
            b[2] = (uint32_t)uniform((int)(left >= ROWS || (left > 0 && last >= b[2]) ? b[2] : left > 0 ? last : 0u));
#pragma unroll
            for (int i = 0; i < N; ++i)
                load_piece(b, FIRST && row_of(i, w0) < r.from - (int)r.pos ? kNowhere : off[i] + add, dst + 16 * THREADS * i);
            return;
        }
        uint32_t add[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {  // the piece's page, and back from the tile's beginning, which is a page's, to that page's
            const int page = ((w0 + THREADS * i) / CH) >> r.shift;
            add[i] = r.entry(r.pos + (page << r.shift)) - (uint32_t)(page << r.shift) * r.ts;
        }
        if (!FIRST && left >= ROWS) {
#pragma unroll
            for (int i = 0; i < N; ++i) load_piece(r.pool, off[i] + add[i], dst + 16 * THREADS * i);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = row_of(i, w0);
                load_piece(r.pool, row < r.from - (int)r.pos || row >= left ? kNowhere : off[i] + add[i], dst + 16 * THREADS * i);
            }
        }
    }
    __device__ __forceinline__ static int row_of(int i, int w0) { return (w0 + (int)(threadIdx.x & 63) + THREADS * i) / CH; }
};

// A row's values as B operands: 16 c + 8 h .. + 8 of the head, zeros past d and for rows outside. `row` is a row that may
// be read whether or not it is valid, so that the loads go out together.
template <int D>
__device__ __forceinline__ void load_row(const uint8_t* row, bool valid, int d, int lane, bf16x8 (&out)[D / 16]) {
    u32x4 w[D / 16];
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
        const int e = 16 * c + 8 * (lane >> 5);
        w[c] = *reinterpret_cast<const u32x4*>(row + (e < d ? 2 * e : 0));
    }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
        const bool on = valid && 16 * c + 8 * (lane >> 5) < d;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[c][j] = on ? w[c][j] : 0u;
        out[c] = as_bf16x8(w[c]);
    }
}

// a 32 x 32 tile's bf16 words, as B operands, back to rows: the lane's column holds rows 16 c + 8 h .. + 7 in 16 bytes
__device__ __forceinline__ u32x4 rows_of(const u32x4& w) {
    u32x4 r;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const auto s = __builtin_amdgcn_permlane32_swap(w[j], w[2 + j], false, false);
        r[j] = s[0];
        r[2 + j] = s[1];
    }
    return r;
}

// A lane's 16 values of one 32-column block of an output row (columns 8e + 4h + 0..3 of the block, e = 0..3),
// times f, to the row at column d0: 16 bytes a store. Both lanes of a row call it; on: the row is written.
__device__ __forceinline__ void store_block(uint8_t* row, bool f32, bool on, int d0, int d, int h, const f32x16& x, float f) {
    if (f32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = d0 + 8 * e + 4 * h;
            const float4 v = {x[4 * e] * f, x[4 * e + 1] * f, x[4 * e + 2] * f, x[4 * e + 3] * f};
            if (on && c < d) *reinterpret_cast<float4*>(row + 4 * c) = v;
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e += 2) {  // the two lanes exchange: columns 8e .. 8e + 7 in the lower, the next 8 in the upper
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const auto s = __builtin_amdgcn_permlane32_swap(pack_bf16(x[4 * e + 2 * j] * f, x[4 * e + 2 * j + 1] * f),
                                                            pack_bf16(x[4 * e + 4 + 2 * j] * f, x[4 * e + 5 + 2 * j] * f), false, false);
            w[j] = s[0];
            w[2 + j] = s[1];
        }
        const int c = d0 + 8 * e + 8 * h;
        if (on && c < d) *reinterpret_cast<u32x4*>(row + 2 * c) = w;
    }
}

// products between an LDS operand's read and its use in the loops that place every instruction
constexpr int kAhead = 4;
// step i of `len` steps from `from`: the elements [lo, hi) of 16 that belong to it, in pairs
constexpr int pair_from(int i, int from, int len) { return i < from ? 0 : i >= from + len ? 16 : 2 * (8 * (i - from) / len); }

// the backward's factor on the scores, in base 2. With a scale of zero a factor that leaves nothing of a finite score; so a masked score
// is an infinity of the other sign, and its exponential zero.
__device__ __forceinline__ float back_scale(const Args& a) { return a.scale == 0.0f ? 0x1p-126f : a.scale * kLog2e; }

}  // namespace attn
}  // namespace r97q
