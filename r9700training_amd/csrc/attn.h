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

#include "../../include/r97q.h"
#include "iqr_device.h"

namespace r97q {
namespace attn {

using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using s16x8 = __attribute__((ext_vector_type(8))) short;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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
    float* delta;        // backward: sum over d of dO * O, laid out as lse
    int32_t batch, hq, hk, g, d;
    int64_t lq, lk;      // tokens of a sequence (packed: of the longest)
    const int32_t* q_starts;
    const int32_t* kv_starts;
    const int32_t* kv_lens;
    int64_t q_tokens, kv_tokens;
    int32_t causal;
    int64_t window;      // 0: none
    float scale;         // of the scores
    // the split forward: partial results of a row tile's key ranges
    int32_t splits;
    int32_t tiles;       // row tiles in the grid
    float* part;         // [split][b][h][Lq][D] f32, then (m, l) pairs [split][b][h][Lq]
};

// one sequence: its tokens' places and counts. Starts and lengths come from device memory, so they are
// clamped to the tensors: nothing is read or written past them whatever they hold.
struct Seq {
    int64_t q_base, k_base;  // token offsets (packed) into the whole tensors; 0 in the dense form
    int64_t b;
    int64_t lq, lk, off;     // off: query i stands at key position i + off
};

__device__ __forceinline__ int64_t clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

__device__ __forceinline__ Seq sequence(const Args& a, int b) {
    Seq s;
    s.b = b;
    s.q_base = s.k_base = 0;
    s.lq = a.lq;
    s.lk = a.lk;
    if (a.q_starts) {
        s.q_base = clamp64(a.q_starts[b], 0, a.q_tokens);
        s.lq = clamp64(a.q_starts[b + 1], s.q_base, a.q_tokens) - s.q_base;
    }
    if (a.kv_starts) {
        s.k_base = clamp64(a.kv_starts[b], 0, a.kv_tokens);
        s.lk = clamp64(a.kv_starts[b + 1], s.k_base, a.kv_tokens) - s.k_base;
    } else if (a.kv_lens) {
        s.lk = clamp64(a.kv_lens[b], 0, a.lk);
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
__device__ __forceinline__ int64_t stat_at(const Args& a, const Seq& s, int h, int64_t token) {
    return a.q_starts ? h * a.q_tokens + s.q_base + token : (s.b * a.hq + h) * a.lq + token;
}

// keys [lo, hi) that queries at tokens [t0, t1] may see (hi <= lo: none)
__device__ __forceinline__ void key_range(const Args& a, const Seq& s, int64_t t0, int64_t t1, int64_t& lo, int64_t& hi) {
    lo = 0;
    hi = s.lk;
    if (a.causal) hi = clamp64(t1 + s.off + 1, 0, s.lk);
    if (a.window) lo = clamp64(t0 + s.off - a.window + 1, 0, s.lk);
}

__device__ __forceinline__ f32x16 mfma(bf16x8 x, bf16x8 y, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
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

// ROWS rows of a tile on their way from memory through a workgroup's registers. Rows past the last one
// repeat it and columns past the head's d repeat the first chunk: what lies there is multiplied by zeros,
// masked or not stored, and comes from values that some row sees.
template <int D, int ROWS, int THREADS>
struct Stage {
    static constexpr int N = ROWS * Tile<D>::CH / THREADS;  // 16-byte pieces a thread
    static_assert(N * THREADS == ROWS * Tile<D>::CH, "whole pieces");
    u32x4 x[N];
    // base: the sequence's token 0 of the head; ts2: bytes a token
    __device__ __forceinline__ void load(const uint8_t* base, int64_t ts2, int64_t row0, int64_t last, int d, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int p = tid + THREADS * i, row = p / Tile<D>::CH, ch = p % Tile<D>::CH;
            const int64_t r = row0 + row < last ? row0 + row : last;
            x[i] = *reinterpret_cast<const u32x4*>(base + r * ts2 + (8 * ch < d ? 16 * ch : 0));
        }
    }
    __device__ __forceinline__ void store(uint8_t* t, int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int p = tid + THREADS * i;
            *reinterpret_cast<u32x4*>(t + Tile<D>::at(p / Tile<D>::CH, p % Tile<D>::CH)) = x[i];
        }
    }
};

// a row's values as B operands: 16 c + 8 h .. + 8 of the head, zeros past d and for rows outside
template <int D>
__device__ __forceinline__ void load_row(const uint8_t* row, bool valid, int d, int lane, bf16x8 (&out)[D / 16]) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
        const int e = 16 * c + 8 * (lane >> 5);
        u32x4 w = {0, 0, 0, 0};
        if (valid && e < d) w = *reinterpret_cast<const u32x4*>(row + 2 * e);
        out[c] = as_bf16x8(w);
    }
}

// four consecutive values of a row (d0 a multiple of 4; d a multiple of 8)
__device__ __forceinline__ void store4(uint8_t* row, bool f32, int d0, float x, float y, float z, float w) {
    if (f32) {
        float4 v = {x, y, z, w};
        *reinterpret_cast<float4*>(row + 4 * d0) = v;
    } else {
        uint2 v = {pack_bf16(x, y), pack_bf16(z, w)};
        *reinterpret_cast<uint2*>(row + 2 * d0) = v;
    }
}

}  // namespace attn
}  // namespace r97q
