// recurrence.hip -- a gated linear recurrence over long sequences, forward and backward.
//
//   s = sigmoid(gate), a = e^(-rate s), q = 1 - a^2, w = sigmoid(input_gate) x,  h_t = a_t h_(t-1) + sqrt(q_t) w_t
// and with l_t the cotangent of h_t and all that follows from it, l_t = dh_t + a_(t+1) l_(t+1):
//   dlog a = l a (h_(t-1) - a w / sqrt(q)),  drate = -sum s dlog a,  dgate = -rate s (1 - s) dlog a,
//   dx = l sqrt(q) sigmoid(i),  dinput_gate = dx x (1 - sigmoid(i)),  dh0 = a_1 l_1.
//
// A span of tokens acts on the state before it as h -> A h + H, and on the cotangent after it as m -> A m + M (m_t = a_t l_t),
// with one A = e^-(sum of rate s). So a workgroup walks a sequence's tokens for 64 channels (a row's 128 or 256 bytes) in
// tiles: a thread a few tokens one after the other for the channels of one 16-byte piece, a wave's groups of lanes and the
// workgroup's waves joined by their spans, the tile's end carried to the next tile. Each value is read and written once, which
// is the bound: a tile's loads are out while the tile before is worked on.
//
// A wave's join. Lane (g, c) holds span g of the VC channels of piece c. A transposition of registers against the lanes'
// bits 3 .. 5 (swaps of lane halves and rows, no LDS) gives each lane all the wave's spans of one channel: a scan there is
// VC multiply-adds, a wave's 64 channels one a lane, and one float2 a lane goes to the other waves.
//
// Few sequences and channels over many tokens leave compute units idle: then the tokens are cut into ranges, a first launch
// forms the ranges' spans, and each workgroup of the second begins from those before its own (behind, in the backward). The
// ranges' inputs are then read twice.
//
// Measured, us and TB/s of the tensors read and written once (a copy of 1 GiB reaches 5.0), with a gate on the input:
//                        bf16 forward   backward     f32 forward    backward
//   8 x 2048 x 2048         68  4.0     121  3.9      118  4.6      217  4.3     256 workgroups, no ranges
//   8 x 2048 x 2047         72  3.7     123  3.8      109  4.9      230  4.1     rows of every alignment
//   8 x 2048 x 1024         53  2.5      75  3.2       84  3.2      135  3.5     two ranges
//   1 x 16384 x 2048       116  2.3     151  3.1      194  2.8      268  3.5     eight ranges
//   32 x 16 x 4096          10  1.6      21  1.4       13  2.7       27  2.2     a thread a sequence
//   512 x 2048 x 3         116  0.2     438  0.1      131  0.4      542  0.2     value by value
// The value-by-value backward with a gate on the input spills (238 registers of f32, 67 of bf16): it serves rows of less than a
// piece, tokens more than 2^20 values apart and, forward, odd widths in place.
//
// Numbers. All is f32 but the inputs' and outputs' type. A state may last for thousands of tokens of decays next to one,
// where an error with a sign adds up: a wave's A is formed from the sum of its logarithms, by 1 minus a polynomial where it
// is near one, one token's decay that a state is carried through by its distance from one (carry_of), and 1 - a^2 by
// 2 a sinh(rate s).
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/r97q.h"
#include "iqr_device.h"
#include "status.h"

namespace r97q {
namespace scan {
namespace {

using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using b16x2 = __attribute__((ext_vector_type(2))) __bf16;

constexpr int kWaves = 8, kThreads = 64 * kWaves, kSlab = 64, kChunk = R97Q_RECURRENCE_CHUNK;
constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = 1.9259629911266175e-8f, kLn2 = 0.6931471805599453f;

struct Rows {  // [batch, tokens, channels] or packed [tokens, channels], channels consecutive
    uint8_t* p;
    int64_t bs, ts;
};

struct Args {
    Rows x, g, i, h;              // i.p null: no gate on the input. h: the forward's output, the backward's d_h
    Rows dx, dg, di;
    const float* rate;
    const float* first;           // the state before (h0), or the cotangent behind (d_last); may be null
    float* last;                  // the state behind (last), or the cotangent before (dh0); may be null
    float* states;                // the states before tokens 0, kChunk, 2 kChunk, .. of every sequence; may be null
    const int32_t* starts;
    int64_t tokens, len;
    int32_t batch, channels;
    int32_t ranges, fine;         // ranges, and the spans of one
    int64_t range_len, span_len;
    float2* spans;                // [batch][ranges * fine][channels]
    float* kept;                  // [batch][channels]: `first`, where `last` may be written over it
    int32_t few;                  // a thread a sequence
    int32_t dealt;                // the grid is one-dimensional, an XCD's workgroups neighbours (deal())
    float* drate;                 // [batch * ranges][channels], or the sum itself where that is one row
};

// a sequence's place
struct Span {
    int64_t base, len;
    int64_t state;                // its first row of states
};
__device__ __forceinline__ int64_t clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }
__device__ __forceinline__ Span span_of(const Args& a, int b) {
    Span s = {0, a.len, b * ((a.len + kChunk - 1) / kChunk)};
    if (a.starts) {  // starts come from device memory: clamped to the tensors
        s.base = clamp64(__builtin_amdgcn_readfirstlane(a.starts[b]), 0, a.tokens);
        s.len = clamp64(__builtin_amdgcn_readfirstlane(a.starts[b + 1]), s.base, a.tokens) - s.base;
        s.state = s.base / kChunk + b;
    }
    return s;
}
__device__ __forceinline__ uint32_t fresh(uint32_t x) {
    asm volatile("" : "+s"(x));
    return x;
}
constexpr uint32_t kNowhere = 0x80000000u;  // an offset past every buffer's end

// ---------------------------------------------------------------- pieces of 16 bytes
// A piece may lie anywhere: the memory takes loads and stores of every alignment, so rows of odd widths go by pieces too.
template <class T>
constexpr int kVC = 16 / (int)sizeof(T);
template <class T>
using Loose = u32x4 __attribute__((aligned(sizeof(T))));
template <class T>
__device__ __forceinline__ float value(const u32x4& v, int j) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, (uint32_t)v[j]);
    else return __builtin_bit_cast(float, j & 1 ? v[j >> 1] & 0xFFFF0000u : v[j >> 1] << 16);
}
template <class T>
__device__ __forceinline__ u32x4 pack(const float* x) {
    u32x4 v;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __builtin_bit_cast(uint32_t, x[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const b16x2 w = {(__bf16)x[2 * j], (__bf16)x[2 * j + 1]};
            v[j] = __builtin_bit_cast(uint32_t, w);
        }
    }
    return v;
}
// One of a sequence's tensors, in tiles of `rows` tokens. WIDE: a tile is a buffer that ends with its last token, so a load past
// it gives zeros and a store past it is dropped, every tile has as many of both (nothing waits for a store whose number the
// compiler cannot know), and an offset is 32 bits. Else value by value, the last token and channel again past the end.
template <class T, bool WIDE>
struct Io;
template <class T>
struct Io<T, true> {
    uint64_t base;
    uint32_t ts, row, off;  // bytes a token; of a row; the thread's first piece in a tile
    __device__ __forceinline__ Io(const Rows& t, const Args& a, const Span& s, int b, int first, int c0, bool mine)
        : base(reinterpret_cast<uint64_t>(t.p) + (a.starts ? s.base * t.ts : b * t.bs) * sizeof(T)), ts((uint32_t)(t.ts * sizeof(T))),
          row((uint32_t)(a.channels * sizeof(T))), off(mine ? first * ts + c0 * (uint32_t)sizeof(T) : kNowhere) {}
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(int64_t t0, int64_t end, int rows) const {
        const int left = end - t0 < rows ? (int)(end - t0) : rows;
        const int bytes = left > 0 ? (int)((left - 1) * ts + row) : 0;
        return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(base + t0 * ts), 0, bytes, 0x00020000);
    }
    // (offsets are formed where they are used: held through the loop they would take a register for every token)
    __device__ __forceinline__ u32x4 load(__amdgpu_buffer_rsrc_t buf, int k) const {
        return __builtin_amdgcn_raw_buffer_load_b128(buf, off + k * fresh(ts), 0, 0);
    }
    __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t buf, int k, const u32x4& v) const {
        __builtin_amdgcn_raw_buffer_store_b128(v, buf, off + k * fresh(ts), 0, 0);
    }
};
template <class T>
struct Io<T, false> {
    struct Tile {
        T* p;          // the thread's first token
        int left;      // tokens from there to the end
    };
    T* base;
    int64_t ts;
    int first, c0, channels;
    __device__ __forceinline__ Io(const Rows& t, const Args& a, const Span& s, int b, int first_, int c0_, bool)
        : base(reinterpret_cast<T*>(t.p) + (a.starts ? s.base * t.ts : b * t.bs)), ts(t.ts), first(first_), c0(c0_), channels(a.channels) {}
    __device__ __forceinline__ Tile buffer(int64_t t0, int64_t end, int rows) const {
        const int64_t left = end - t0 - first;
        return {base + (t0 + first) * ts, left > rows ? rows : (int)left};
    }
    __device__ __forceinline__ u32x4 load(const Tile& t, int k) const {
        const T* p = t.p + (k < t.left ? k : t.left - 1) * ts;
        T x[kVC<T>];
#pragma unroll
        for (int j = 0; j < kVC<T>; ++j) x[j] = p[c0 + j < channels ? c0 + j : channels - 1];
        return __builtin_bit_cast(u32x4, x);
    }
    __device__ __forceinline__ void store(const Tile& t, int k, const u32x4& v) const {
        struct { T x[kVC<T>]; } u = __builtin_bit_cast(decltype(u), v);
        if (k < t.left)
#pragma unroll
            for (int j = 0; j < kVC<T>; ++j)
                if (c0 + j < channels) t.p[k * ts + c0 + j] = u.x[j];
    }
};

// a sequence's tensor, a token's piece at a time
template <class T, bool WIDE>
struct Piece {
    const T* base;
    int64_t ts;
    int c0, channels;
    __device__ __forceinline__ Piece(const Rows& t, const Args& a, const Span& s, int b, int c0_)
        : base(reinterpret_cast<const T*>(t.p) + (a.starts ? s.base * t.ts : b * t.bs)), ts(t.ts), c0(c0_), channels(a.channels) {}
    __device__ __forceinline__ u32x4 load(int64_t token) const {
        const T* p = base + token * ts;
        if constexpr (WIDE) return *reinterpret_cast<const Loose<T>*>(p + c0);
        T x[kVC<T>];
#pragma unroll
        for (int j = 0; j < kVC<T>; ++j) x[j] = p[c0 + j < channels ? c0 + j : channels - 1];
        return __builtin_bit_cast(u32x4, x);
    }
};

// ---------------------------------------------------------------- the gates
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// A channel's rate in base 2, at most 2^88: under any gate but one below -57 nothing is left of a state then, as without that bound,
// and the shut gate of a place past the end, which in f32 is open by e^-87, decays nothing under every rate.
__device__ __forceinline__ float rate_of(const Args& a, int c) {
    const float r = a.rate[c] * kLog2e;
    return r > 0x1p88f ? 0x1p88f : r;
}
// 1 / (1 + e^-v). The product with log2 e is off by half a step of itself, which for a far gate is more than a step of the
// result: f32's is put right (bf16's inputs are further off), gates past 87 on either side counted as 87.
template <class T>
__device__ __forceinline__ float sigmoid(float v) {
    if constexpr (sizeof(T) == 4) v = v < -87.0f ? -87.0f : v > 87.0f ? 87.0f : v;
    const float t = v * -kLog2e;
    float e = exp2_(t);
    if constexpr (sizeof(T) == 4) {
        const float r = __builtin_fmaf(-v, kLog2eLow, __builtin_fmaf(v, -kLog2e, -t));
        e = __builtin_fmaf(e, r * kLn2, e);
    }
    return __builtin_amdgcn_rcpf(1.0f + e);
}
// 1 - a^2 of a = 2^-y: 2 a sinh(y ln 2) where a is near one
__device__ __forceinline__ float room(float y, float a) {
    constexpr float l2 = kLn2 * kLn2;
    const float t = y * y;
    float p = __builtin_fmaf(t, 2.0f * kLn2 * l2 * l2 * l2 / 5040.0f, 2.0f * kLn2 * l2 * l2 / 120.0f);
    p = __builtin_fmaf(p, t, 2.0f * kLn2 * l2 / 6.0f);
    p = __builtin_fmaf(p, t, 2.0f * kLn2);
    const float near = p * y * a, far = __builtin_fmaf(-a, a, 1.0f);
    return y < 0.72f ? near : far;
}
// 2^-y, near one by its distance from it
__device__ __forceinline__ float decay_of(float y) {
    const float z = y * kLn2;
    float p = __builtin_fmaf(z, -1.0f / 5040.0f, 1.0f / 720.0f);
    p = __builtin_fmaf(z, p, -1.0f / 120.0f);
    p = __builtin_fmaf(z, p, 1.0f / 24.0f);
    p = __builtin_fmaf(z, p, -1.0f / 6.0f);
    p = __builtin_fmaf(z, p, 0.5f);
    p = __builtin_fmaf(z, -p, 1.0f);
    return z < 0.35f ? __builtin_fmaf(-z, p, 1.0f) : exp2_(-y);
}
// The same for one token's decay that a state is carried through. The exponential's value next to one is low by 0.12 half steps
// in the mean, and a state lasts for 1 / (1 - a) tokens, so below 2^-0.01, where that is more than 100, it is formed from its
// distance from one: half of decay_of's instructions, off by z^4 / 24 < 1e-10.
__device__ __forceinline__ float carry_of(float y) {
    float p = __builtin_fmaf(y, kLn2 * kLn2 * kLn2 / 6.0f, -kLn2 * kLn2 / 2.0f);
    p = __builtin_fmaf(y, p, kLn2);
    p = __builtin_fmaf(-y, p, 1.0f);
    return y < 0.01f ? p : exp2_(-y);
}

// ---------------------------------------------------------------- a wave's transposition
__device__ __forceinline__ void swap32(float& x, float& y) {
    const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y), false, false);
    const uint32_t u = s[0], v = s[1];
    x = __builtin_bit_cast(float, u);
    y = __builtin_bit_cast(float, v);
}
__device__ __forceinline__ void swap16(float& x, float& y) {
    const auto s = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y), false, false);
    const uint32_t u = s[0], v = s[1];
    x = __builtin_bit_cast(float, u);
    y = __builtin_bit_cast(float, v);
}
// lanes 8 .. 15 of a row take y of the lane 8 before into x, lanes 0 .. 7 x of the lane 8 behind into y
__device__ __forceinline__ void swap8(float& x, float& y) {
    const int u = __builtin_bit_cast(int, x), v = __builtin_bit_cast(int, y);
    x = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(u, v, 0x128, 0xF, 0xC, false));
    y = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(v, u, 0x128, 0xF, 0x3, false));
}
// Lane (g, c)'s register j to lane (j, c)'s register g, for g the lane's bits 3 .. 5 (VC 8) or 4 and 5 (VC 4). Its own inverse.
template <int VC>
__device__ __forceinline__ void transpose(float (&x)[VC]) {
#pragma unroll
    for (int j = 0; j < VC / 2; ++j) swap32(x[j], x[j + VC / 2]);
#pragma unroll
    for (int j = 0; j < VC; ++j)
        if (!(j & (VC / 4))) swap16(x[j], x[j + VC / 4]);
    if constexpr (VC == 8) {
#pragma unroll
        for (int j = 0; j < VC; j += 2) swap8(x[j], x[j + 1]);
    }
}

// what a workgroup works on
template <class T, bool WIDE>
struct Place {
    static constexpr int VC = kVC<T>, LPR = 64 / VC;
    int lane, wave, g, c0, ch, near, b, range;
    bool mine;  // the lane's piece is one: its first channel c0. WIDE: the last one ends with the last channel, over its neighbour
    bool on;    // the transposed lane's channel is one (near: one that may be read in any case)
    bool none;  // a workgroup too many
    __device__ __forceinline__ Place(const Args& a, int ranges, int range0 = 0) {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        g = lane / LPR;
        int slab = blockIdx.x, r = blockIdx.y;
        b = blockIdx.z;
        none = false;
        if (a.dealt) {
            const uint32_t slabs = (a.channels + kSlab - 1) / kSlab, i = blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8, j = i / slabs;
            none = i >= slabs * ranges * a.batch;
            slab = (int)(i - j * slabs);
            b = (int)(j / ranges);
            r = (int)(j - (uint32_t)b * ranges);
        }
        c0 = slab * kSlab + lane % LPR * VC;
        mine = c0 < a.channels;
        if (WIDE && c0 > a.channels - VC) c0 = a.channels - VC;
        ch = c0 + g;
        on = mine && ch < a.channels;
        near = on ? ch : a.channels - 1;
        range = range0 + r;
    }
};

// What comes of nothing through the spans p[0], p[step], .. (`many` of them) in order: each wave joins a share of them, their
// loads out together, and all waves join the shares. lds: a float2 for each thread; called by all of them.
__device__ __forceinline__ float through(const float2* p, int64_t step, int many, int wave, int lane, float2 (*lds)[64]) {
    constexpr int kBatch = 8;
    const int share = (many + kWaves - 1) / kWaves, end = (wave + 1) * share < many ? (wave + 1) * share : many;
    float2 own = make_float2(1.0f, 0.0f);
    for (int r = wave * share; r < end; r += kBatch) {
        float2 s[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) s[i] = p[(r + i < end ? r + i : r) * step];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (r + i < end) own = make_float2(own.x * s[i].x, __builtin_fmaf(s[i].x, own.y, s[i].y));
    }
    lds[wave][lane] = own;
    __syncthreads();
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v = __builtin_fmaf(lds[w][lane].x, v, lds[w][lane].y);
    __syncthreads();
    return v;
}

// tokens past the end: nothing enters, nothing decays
template <class T>
__device__ __forceinline__ void blank(u32x4& x, u32x4& g, u32x4& i, bool out) {
    constexpr uint32_t shut = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = out ? 0u : x[e];
        g[e] = out ? shut : g[e];
        i[e] = out ? 0u : i[e];
    }
}

// ---------------------------------------------------------------- the ranges' spans
// grid (slabs, all but one range's spans, sequences): what a part of a range makes of the state before it, or (BACK, from a and
// dh alone) of the cotangent behind it. Nothing is needed of the tokens between, so a lane's group takes a run of tokens of its
// own, with no join but one at the end, and takes each decay as carry_of forms it: over runs of 2048 tokens at rates of 1e-4 the
// state that a range begins from is off by 1 half step in the mean, with the exponential's value by 120. The span that has the
// given end (the first, or BACK the last) holds it; the forward also keeps a copy of it, since `last` may be written over it
// before every workgroup of the next launch has read it. Bound by memory: 1 x 16384 x 2048 bf16, seven ranges' gate and d_h, 41
// us, of which the vector instructions' issue (20 a value) is 17.
template <class T, bool GATED, bool WIDE, bool BACK>
__global__ __launch_bounds__(kThreads, 2) void recurrence_spans_kernel(Args a) {
    constexpr int VC = kVC<T>, TL = 2;
    __shared__ float2 spans[kWaves][64];
    const int all = a.ranges * a.fine;
    const Place<T, WIDE> at(a, all - a.fine, BACK ? a.fine : 0);
    if (at.none) return;
    const Span s = span_of(a, at.b);
    const int64_t begin = at.range * a.span_len;
    const int64_t end = BACK && at.range == all - 1 ? s.len : clamp64(begin + a.span_len, 0, s.len);
    const int64_t run = ((end - begin + kWaves * VC - 1) / (kWaves * VC)), from = begin + (at.wave * VC + at.g) * run;
    float rate[VC], y[VC], u[VC];
#pragma unroll
    for (int j = 0; j < VC; ++j) {
        rate[j] = rate_of(a, at.c0 + j < a.channels ? at.c0 + j : a.channels - 1);
        y[j] = u[j] = 0.0f;
    }
    const Piece<T, WIDE> xs(BACK ? a.h : a.x, a, s, at.b, at.c0), gs(a.g, a, s, at.b, at.c0), is(a.i, a, s, at.b, at.c0);
    struct Raw {
        u32x4 x[TL], g[TL], i[TL];
    };
    // the run's tokens k .. k + TL - 1 in the order they are taken
    auto token = [&](int64_t k) { return BACK ? from + run - 1 - k : from + k; };
    auto fetch = [&](Raw& r, int64_t k0) {
#pragma unroll
        for (int k = 0; k < TL; ++k) {
            const int64_t t = clamp64(token(k0 + k), begin, end - 1);
            r.x[k] = xs.load(t);
            r.g[k] = gs.load(t);
            if constexpr (GATED && !BACK) r.i[k] = is.load(t);
        }
    };
    auto take = [&](Raw& now, Raw& next, int64_t k0) {
        fetch(next, k0 + TL);
        __builtin_amdgcn_sched_barrier(0);
        if (k0 + TL > run || begin + run * kWaves * VC > end) {
#pragma unroll
            for (int k = 0; k < TL; ++k) blank<T>(now.x[k], now.g[k], now.i[k], k0 + k >= run || token(k0 + k) >= end);
        }
#pragma unroll
        for (int k = 0; k < TL; ++k)
#pragma unroll
            for (int j = 0; j < VC; ++j) {
                const float e = rate[j] * sigmoid<T>(value<T>(now.g[k], j)), dec = carry_of(e);
                y[j] += e;
                if constexpr (BACK) {
                    u[j] = dec * (u[j] + value<T>(now.x[k], j));
                } else {
                    float w = value<T>(now.x[k], j);
                    if constexpr (GATED) w *= sigmoid<T>(value<T>(now.i[k], j));
                    u[j] = __builtin_fmaf(dec, u[j], __builtin_amdgcn_sqrtf(room(e, dec)) * w);
                }
            }
    };
    if (begin < end) {
        Raw one, two;
        fetch(one, 0);
        for (int64_t k0 = 0; k0 < run; k0 += 2 * TL) {
            take(one, two, k0);
            if (k0 + TL < run) take(two, one, k0 + TL);
        }
    }
    transpose<VC>(y);
    transpose<VC>(u);
    float sum = 0.0f, got = 0.0f;
#pragma unroll
    for (int i = 0; i < VC; ++i) {
        const int g = BACK ? VC - 1 - i : i;
        got = __builtin_fmaf(decay_of(y[g]), got, u[g]);
        sum += y[g];
    }
    spans[at.wave][at.lane] = make_float2(sum, got);
    __syncthreads();
    if (at.wave || !at.on) return;
    const int64_t mine = (int64_t)at.b * a.channels + at.ch;
    float v = 0.0f;
    if (a.first && at.range == (BACK ? all - 1 : 0)) {
        v = a.first[mine];
        if constexpr (!BACK) a.kept[mine] = v;
    }
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const float2 p = spans[BACK ? kWaves - 1 - i : i][at.lane];
        v = __builtin_fmaf(decay_of(p.x), v, p.y);
        sum += p.x;
    }
    a.spans[((int64_t)at.b * all + at.range) * a.channels + at.ch] = make_float2(decay_of(sum), v);
}

// ---------------------------------------------------------------- forward
// grid (slabs, ranges, sequences). Bound by memory: 8 x 2048 x 2048 bf16 65 us, where the same loads and stores with nothing
// between them take 62; a value's 33 vector instructions, 6 of them exponentials, roots and reciprocals, are issued in 34.
template <class T, bool GATED, bool WIDE>
__global__ __launch_bounds__(kThreads, 2) void recurrence_fwd_kernel(Args a) {
    constexpr int VC = kVC<T>, TL = 16 / VC, WT = VC * TL, TILE = kWaves * WT;
    static_assert(TILE == kChunk, "a tile begins at a kept state");
    __shared__ float2 spans[2][kWaves][64];
    const Place<T, WIDE> at(a, a.ranges);
    if (at.none) return;
    const Span s = span_of(a, at.b);
    const int64_t begin = at.range * a.range_len;
    const int64_t end = at.range == a.ranges - 1 ? s.len : clamp64(begin + a.range_len, 0, s.len);
    float h = 0.0f;
    const int64_t mine = (int64_t)at.b * a.channels + at.near;
    if (at.range == 0) {
        if (a.first) h = a.ranges > 1 ? a.kept[mine] : a.first[mine];
    } else {
        h = through(a.spans + (int64_t)at.b * a.ranges * a.fine * a.channels + at.near, a.channels, at.range * a.fine, at.wave, at.lane,
                    spans[0]);
    }
    float rate[VC];
#pragma unroll
    for (int j = 0; j < VC; ++j) rate[j] = rate_of(a, at.c0 + j < a.channels ? at.c0 + j : a.channels - 1);
    const int first = at.wave * WT + at.g * TL;  // the thread's first token in a tile
    using IO = Io<T, WIDE>;
    auto io = [&](const Rows& t) { return IO(t, a, s, at.b, first, at.c0, at.mine); };
    const IO xs = io(a.x), gs = io(a.g), is = io(a.i), hs = io(a.h);

    struct Raw {
        u32x4 x[TL], g[TL], i[TL];
    };
    auto fetch = [&](Raw& r, int64_t t0) {
        const auto x = xs.buffer(t0, end, TILE), g = gs.buffer(t0, end, TILE), i = is.buffer(t0, end, TILE);
#pragma unroll
        for (int k = 0; k < TL; ++k) {
            r.x[k] = xs.load(x, k);
            r.g[k] = gs.load(g, k);
            if constexpr (GATED) r.i[k] = is.load(i, k);
        }
    };
    auto tile = [&](Raw& now, Raw& next, int64_t t0, int slot) {
        fetch(next, t0 + TILE);  // nothing past the end
        __builtin_amdgcn_sched_barrier(0);
        if (t0 + TILE > end) {
#pragma unroll
            for (int k = 0; k < TL; ++k) blank<T>(now.x[k], now.g[k], now.i[k], t0 + first + k >= end);
        }
        float dec[TL][VC], in[TL][VC], y[VC], u[VC];
#pragma unroll
        for (int j = 0; j < VC; ++j) {
            y[j] = u[j] = 0.0f;
#pragma unroll
            for (int k = 0; k < TL; ++k) {
                const float e = rate[j] * sigmoid<T>(value<T>(now.g[k], j));
                dec[k][j] = exp2_(-e);
                float w = value<T>(now.x[k], j);
                if constexpr (GATED) w *= sigmoid<T>(value<T>(now.i[k], j));
                in[k][j] = __builtin_amdgcn_sqrtf(room(e, dec[k][j])) * w;
                y[j] += e;
                u[j] = __builtin_fmaf(dec[k][j], u[j], in[k][j]);
            }
        }
        // the wave's spans of one channel
        transpose<VC>(y);
        transpose<VC>(u);
        float sum = 0.0f, got = 0.0f;
#pragma unroll
        for (int i = 0; i < VC; ++i) {
            sum += y[i];
            y[i] = exp2_(-y[i]);
            got = __builtin_fmaf(y[i], got, u[i]);
        }
        spans[slot][at.wave][at.lane] = make_float2(decay_of(sum), got);
        __syncthreads();
        float before = h;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float2 p = spans[slot][w][at.lane];
            if (w == at.wave) before = h;
            h = __builtin_fmaf(p.x, h, p.y);
        }
        const auto kept = __builtin_amdgcn_make_buffer_rsrc(a.states + (s.state + t0 / kChunk) * a.channels, 0,
                                                            a.states && at.wave == 0 ? a.channels * 4 : 0, 0x00020000);
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, before), kept, at.on ? 4 * at.ch : (int)kNowhere, 0, 0);
#pragma unroll
        for (int i = 0; i < VC; ++i) {
            const float x = before;
            before = __builtin_fmaf(y[i], before, u[i]);
            u[i] = x;
        }
        transpose<VC>(u);
        const auto h = hs.buffer(t0, end, TILE);
#pragma unroll
        for (int k = 0; k < TL; ++k) {
#pragma unroll
            for (int j = 0; j < VC; ++j) u[j] = __builtin_fmaf(dec[k][j], u[j], in[k][j]);
            hs.store(h, k, pack<T>(u));
        }
    };
    if (begin < end) {
        Raw one, two;
        fetch(one, begin);
        for (int64_t t0 = begin; t0 < end; t0 += 2 * TILE) {
            tile(one, two, t0, 0);
            if (t0 + TILE < end) tile(two, one, t0 + TILE, 1);
        }
    }
    if (at.wave == 0 && at.on && at.range == a.ranges - 1 && a.last) a.last[mine] = h;
}

// ---------------------------------------------------------------- backward
// The tiles from the last to the first, kChunk tokens each: the state before a tile is the forward's, the cotangent behind
// it is carried. Bound by memory with some 65 vector instructions a value beside it: 1 x 16384 x 2048 bf16 105 us of the call's
// 146. f32 8 x 2048 x 2048 4.4 TB/s, without a gate on the input 4.7.
template <class T, bool GATED, bool WIDE>
__global__ __launch_bounds__(kThreads, 2) void recurrence_bwd_kernel(Args a) {
    constexpr int VC = kVC<T>, TL = 16 / VC, WT = VC * TL, TILE = kWaves * WT;
    static_assert(TILE == kChunk, "a tile begins at a kept state");
    // Of f32 with a gate on the input not all that the first half forms fits the registers next to two tiles of inputs: what comes
    // of a, sg and in alone is formed again. 8 x 2048 x 2048 212 us (11 registers still spilled), with all of it kept and 29
    // spilled 233.
    constexpr bool AGAIN = sizeof(T) == 4 && GATED;
    __shared__ float2 spans[2][kWaves][64];
    __shared__ float backs[2][kWaves][64];
    const Place<T, WIDE> at(a, a.ranges);
    if (at.none) return;
    const Span s = span_of(a, at.b);
    const int64_t begin = at.range * a.range_len;
    const int64_t end = at.range == a.ranges - 1 ? s.len : clamp64(begin + a.range_len, 0, s.len);
    float m = 0.0f;  // the cotangent behind the tile, times its decay
    const int64_t mine = (int64_t)at.b * a.channels + at.near;
    if (at.range == a.ranges - 1) {
        if (a.first) m = a.first[mine];
    } else {  // the last range's span holds what is behind it
        m = through(a.spans + ((int64_t)(at.b + 1) * a.ranges * a.fine - 1) * a.channels + at.near, -(int64_t)a.channels,
                    (a.ranges - 1 - at.range) * a.fine, at.wave, at.lane, spans[0]);
    }
    float rate[VC], dr[VC];
#pragma unroll
    for (int j = 0; j < VC; ++j) rate[j] = rate_of(a, at.c0 + j < a.channels ? at.c0 + j : a.channels - 1), dr[j] = 0.0f;
    const int first = at.wave * WT + at.g * TL;
    using IO = Io<T, WIDE>;
    auto io = [&](const Rows& t) { return IO(t, a, s, at.b, first, at.c0, at.mine); };
    const IO xs = io(a.x), gs = io(a.g), is = io(a.i), es = io(a.h), dxs = io(a.dx), dgs = io(a.dg), dis = io(a.di);

    struct Raw {
        u32x4 x[TL], g[TL], i[TL], e[TL];
        float h;
    };
    auto fetch = [&](Raw& r, int64_t to) {  // nothing before the beginning
        const int64_t t0 = to >= begin ? to : begin, upto = !WIDE || to >= begin ? end : begin;
        const auto x = xs.buffer(t0, upto, TILE), g = gs.buffer(t0, upto, TILE);
        const auto i = is.buffer(t0, upto, TILE), e = es.buffer(t0, upto, TILE);
#pragma unroll
        for (int k = 0; k < TL; ++k) {
            r.g[k] = gs.load(g, k);
            r.e[k] = es.load(e, k);
            r.x[k] = xs.load(x, k);
            if constexpr (GATED) r.i[k] = is.load(i, k);
        }
        r.h = a.states[(s.state + t0 / kChunk) * a.channels + at.near];
    };
    auto tile = [&](Raw& now, Raw& next, int64_t t0, int slot) {
        fetch(next, t0 - TILE);
        __builtin_amdgcn_sched_barrier(0);
        if (t0 + TILE > end) {
#pragma unroll
            for (int k = 0; k < TL; ++k) {
                const bool out = t0 + first + k >= end;
                blank<T>(now.x[k], now.g[k], now.i[k], out);
#pragma unroll
                for (int e = 0; e < 4; ++e) now.e[k][e] = out ? 0u : now.e[k][e];
            }
        }
        // a, the gates, what x enters by (sqrt(q) sigmoid(i)) and what it takes from dlog a (a sigmoid(i) / sqrt(q))
        constexpr int KEPT = AGAIN ? 1 : TL;
        float dec[TL][VC], sg[TL][VC], si[KEPT][VC], in[TL][VC], near[KEPT][VC], y[VC], u[VC], v[VC];
#pragma unroll
        for (int j = 0; j < VC; ++j) {
            y[j] = u[j] = v[j] = 0.0f;
#pragma unroll
            for (int k = 0; k < TL; ++k) {
                sg[k][j] = sigmoid<T>(value<T>(now.g[k], j));
                const float e = rate[j] * sg[k][j];
                dec[k][j] = exp2_(-e);
                y[j] += e;
                const float q = room(e, dec[k][j]);
                // where nothing decays the root's derivative counts as none
                const float inv = q >= 0x1p-126f ? __builtin_amdgcn_rsqf(q) : q * 0.0f;
                in[k][j] = q * inv;
                if constexpr (AGAIN) {
                    in[k][j] *= sigmoid<T>(value<T>(now.i[k], j));
                } else {
                    near[k][j] = dec[k][j] * inv;
                    if constexpr (GATED) {
                        si[k][j] = sigmoid<T>(value<T>(now.i[k], j));
                        in[k][j] *= si[k][j];
                        near[k][j] *= si[k][j];
                    }
                }
                u[j] = __builtin_fmaf(dec[k][j], u[j], in[k][j] * value<T>(now.x[k], j));
            }
#pragma unroll
            for (int k = TL - 1; k >= 0; --k) v[j] = dec[k][j] * (v[j] + value<T>(now.e[k], j));
        }
        transpose<VC>(y);
        transpose<VC>(u);
        transpose<VC>(v);
        float sum = 0.0f, got = 0.0f, back = 0.0f;
#pragma unroll
        for (int i = 0; i < VC; ++i) {
            sum += y[i];
            y[i] = exp2_(-y[i]);
            got = __builtin_fmaf(y[i], got, u[i]);
        }
#pragma unroll
        for (int i = VC - 1; i >= 0; --i) back = __builtin_fmaf(y[i], back, v[i]);
        spans[slot][at.wave][at.lane] = make_float2(decay_of(sum), got);
        backs[slot][at.wave][at.lane] = back;
        __syncthreads();
        float h = now.h, before = 0.0f, behind = 0.0f;
        float2 p[kWaves];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            p[w] = spans[slot][w][at.lane];
            if (w == at.wave) before = h;
            h = __builtin_fmaf(p[w].x, h, p[w].y);
        }
#pragma unroll
        for (int w = kWaves - 1; w >= 0; --w) {
            if (w == at.wave) behind = m;
            m = __builtin_fmaf(p[w].x, m, backs[slot][w][at.lane]);
        }
        // the inputs are taken apart again: both forms would not fit the registers
#pragma unroll
        for (int k = 0; k < TL; ++k) asm volatile("" : "+v"(now.x[k]), "+v"(now.e[k]));
        if constexpr (AGAIN)
#pragma unroll
            for (int k = 0; k < TL; ++k)
#pragma unroll
                for (int j = 0; j < VC; ++j) asm volatile("" : "+v"(sg[k][j]));
#pragma unroll
        for (int i = 0; i < VC; ++i) {
            const float x = before;
            before = __builtin_fmaf(y[i], before, u[i]);
            u[i] = x;
        }
#pragma unroll
        for (int i = VC - 1; i >= 0; --i) {
            const float x = behind;
            behind = __builtin_fmaf(y[i], behind, v[i]);
            v[i] = x;
        }
        transpose<VC>(u);
        transpose<VC>(v);
        const auto bx = dxs.buffer(t0, end, TILE), bg = dgs.buffer(t0, end, TILE), bi = dis.buffer(t0, end, TILE);
        // each token's state before it
        float was[TL][VC];
#pragma unroll
        for (int k = 0; k < TL; ++k)
#pragma unroll
            for (int j = 0; j < VC; ++j) {
                was[k][j] = u[j];
                u[j] = __builtin_fmaf(dec[k][j], u[j], in[k][j] * value<T>(now.x[k], j));
            }
#pragma unroll
        for (int k = TL - 1; k >= 0; --k) {
            float dx[VC], dg[VC], di[VC];
#pragma unroll
            for (int j = 0; j < VC; ++j) {
                const float l = value<T>(now.e[k], j) + v[j], x = value<T>(now.x[k], j);
                v[j] = dec[k][j] * l;
                float open = 1.0f, part;
                if constexpr (AGAIN) {
                    const float q = room(rate[j] * sg[k][j], dec[k][j]);
                    const float inv = q >= 0x1p-126f ? __builtin_amdgcn_rsqf(q) : q * 0.0f;
                    open = in[k][j] * inv;
                    part = dec[k][j] * open * inv;
                } else {
                    part = near[k][j];
                    if constexpr (GATED) open = si[k][j];
                }
                const float d = sg[k][j] * (v[j] * __builtin_fmaf(-part, x, was[k][j]));
                dr[j] -= d;
                dg[j] = -kLn2 * rate[j] * __builtin_fmaf(-sg[k][j], d, d);
                dx[j] = l * in[k][j];
                if constexpr (GATED) di[j] = dx[j] * __builtin_fmaf(-x, open, x);
            }
            dxs.store(bx, k, pack<T>(dx));
            dgs.store(bg, k, pack<T>(dg));
            if constexpr (GATED) dis.store(bi, k, pack<T>(di));
        }
    };
    if (begin < end) {
        int64_t t0 = begin + (end - 1 - begin) / TILE * TILE;
        Raw one, two;
        fetch(one, t0);
        for (; t0 >= begin; t0 -= 2 * TILE) {
            tile(one, two, t0, 0);
            if (t0 - TILE >= begin) tile(two, one, t0 - TILE, 1);
        }
    }
    if (at.wave == 0 && at.on && at.range == 0 && a.last) a.last[mine] = m;
    // the rate's gradient: a lane's groups, then the waves, in order
    transpose<VC>(dr);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VC; ++i) sum += dr[i];
    __syncthreads();
    backs[0][at.wave][at.lane] = sum;
    __syncthreads();
    if (at.wave || !at.on) return;
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += backs[0][w][at.lane];
    a.drate[((int64_t)at.b * a.ranges + at.range) * a.channels + at.ch] = sum;
}

// The rows of the rate's partial gradients added in a fixed order: 64 channels a workgroup, 16 shares of the rows. Some rows:
// 4 us, latency.
constexpr int kShares = 16;
__global__ __launch_bounds__(64 * kShares) void recurrence_rate_kernel(const float* part, float* out, int64_t rows, int32_t channels) {
    __shared__ float sums[kShares][64];
    const int lane = threadIdx.x & 63, share = threadIdx.x >> 6, c = blockIdx.x * 64 + lane, near = c < channels ? c : channels - 1;
    float sum = 0.0f;
    for (int64_t r = share; r < rows; r += 4 * kShares) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = part[(r + i * kShares < rows ? r + i * kShares : r) * channels + near];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += r + i * kShares < rows ? x[i] : 0.0f;
    }
    sums[share][lane] = sum;
    __syncthreads();
    if (share || c >= channels) return;
#pragma unroll
    for (int i = 1; i < kShares; ++i) sum += sums[i][lane];
    out[c] = sum;
}

// ---------------------------------------------------------------- a few tokens
// A thread takes a sequence's V channels from token to token: no joins. grid (channels, sequences). 32 sequences of 4096
// channels, one token: 4 us, the latency of a load and a store. A state is carried from call to call by each token's own decay,
// so that is carry_of's: after 4000 tokens one at a time at rates of 1e-4 the states are off by 1 half step in the mean, with
// the exponential's value, a little low next to one, by 229.
constexpr int kFewThreads = 64, kFew = 8;  // tokens that the backward holds at once
template <class T, int V>
struct Few {
    T x[V];
    __device__ __forceinline__ float operator[](int j) const {
        if constexpr (sizeof(T) == 4) return x[j];
        else return bf16_to_f32(x[j]);
    }
};
template <class T, int V>
__device__ __forceinline__ Few<T, V> few_load(const Rows& t, int64_t base, int64_t token, int c0) {
    Few<T, V> v;
    __builtin_memcpy(&v, reinterpret_cast<const T*>(t.p) + base + token * t.ts + c0, sizeof(v));
    return v;
}
template <class T, int V>
__device__ __forceinline__ void few_store(const Rows& t, int64_t base, int64_t token, int c0, const float (&v)[V]) {
    Few<T, V> o;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if constexpr (sizeof(T) == 4) o.x[j] = v[j];
        else o.x[j] = __builtin_bit_cast(uint16_t, (__bf16)v[j]);
    }
    __builtin_memcpy(reinterpret_cast<T*>(t.p) + base + token * t.ts + c0, &o, sizeof(o));
}
__device__ __forceinline__ int64_t base_of(const Rows& t, const Args& a, const Span& s, int b) {
    return a.starts ? s.base * t.ts : b * t.bs;
}

template <class T, int V, bool GATED>
__global__ __launch_bounds__(kFewThreads) void recurrence_few_fwd_kernel(Args a) {
    int c0 = (blockIdx.x * kFewThreads + threadIdx.x) * V;
    const int b = blockIdx.y;
    if (c0 >= a.channels) return;
    if (c0 > a.channels - V) c0 = a.channels - V;  // the last piece ends with the last channel, over its neighbour
    const Span s = span_of(a, b);
    const int64_t xb = base_of(a.x, a, s, b), gb = base_of(a.g, a, s, b), ib = base_of(a.i, a, s, b), hb = base_of(a.h, a, s, b);
    const int64_t mine = (int64_t)b * a.channels + c0;
    float rate[V], h[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        rate[j] = rate_of(a, c0 + j);
        h[j] = a.first ? a.first[mine + j] : 0.0f;
    }
    constexpr int TL = 4;
    for (int64_t t0 = 0; t0 < s.len; t0 += TL) {
        Few<T, V> x[TL], g[TL], i[TL];
#pragma unroll
        for (int k = 0; k < TL; ++k) {
            const int64_t t = t0 + k < s.len ? t0 + k : s.len - 1;
            x[k] = few_load<T, V>(a.x, xb, t, c0);
            g[k] = few_load<T, V>(a.g, gb, t, c0);
            if constexpr (GATED) i[k] = few_load<T, V>(a.i, ib, t, c0);
        }
        if (a.states && t0 % kChunk == 0)
#pragma unroll
            for (int j = 0; j < V; ++j) a.states[(s.state + t0 / kChunk) * a.channels + c0 + j] = h[j];
        float dec[TL][V], in[TL][V];  // of all the tokens before the first one's state, which waits for nothing else then
#pragma unroll
        for (int k = 0; k < TL; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float e = rate[j] * sigmoid<T>(g[k][j]);
                dec[k][j] = carry_of(e);
                float w = x[k][j];
                if constexpr (GATED) w *= sigmoid<T>(i[k][j]);
                in[k][j] = __builtin_amdgcn_sqrtf(room(e, dec[k][j])) * w;
            }
#pragma unroll
        for (int k = 0; k < TL; ++k) {
            if (t0 + k >= s.len) break;
#pragma unroll
            for (int j = 0; j < V; ++j) h[j] = __builtin_fmaf(dec[k][j], h[j], in[k][j]);
            few_store<T, V>(a.h, hb, t0 + k, c0, h);
        }
    }
    if (a.last)
#pragma unroll
        for (int j = 0; j < V; ++j) a.last[mine + j] = h[j];
}

// kFew tokens at a time from the last, the states before them from the kept one on
template <class T, int V, bool GATED>
__global__ __launch_bounds__(kFewThreads) void recurrence_few_bwd_kernel(Args a) {
    int c0 = (blockIdx.x * kFewThreads + threadIdx.x) * V;
    const int b = blockIdx.y;
    if (c0 >= a.channels) return;
    if (c0 > a.channels - V) c0 = a.channels - V;  // the last piece ends with the last channel, over its neighbour
    const Span s = span_of(a, b);
    const int64_t xb = base_of(a.x, a, s, b), gb = base_of(a.g, a, s, b), ib = base_of(a.i, a, s, b), eb = base_of(a.h, a, s, b);
    const int64_t dxb = base_of(a.dx, a, s, b), dgb = base_of(a.dg, a, s, b), dib = base_of(a.di, a, s, b);
    const int64_t mine = (int64_t)b * a.channels + c0;
    float rate[V], m[V], dr[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        rate[j] = rate_of(a, c0 + j);
        m[j] = a.first ? a.first[mine + j] : 0.0f;
        dr[j] = 0.0f;
    }
    for (int64_t t1 = s.len; t1 > 0; t1 = (t1 - 1) / kFew * kFew) {
        const int64_t t0 = (t1 - 1) / kFew * kFew;
        const int n = (int)(t1 - t0);
        Few<T, V> x[kFew], g[kFew], i[kFew], e[kFew];
        float h[V], was[kFew][V], decays[kFew][V];
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] = a.states[(s.state + t0 / kChunk) * a.channels + c0 + j];
#pragma unroll
        for (int k = 0; k < kFew; ++k) {
            const int64_t t = t0 + (k < n ? k : n - 1);
            x[k] = few_load<T, V>(a.x, xb, t, c0);
            g[k] = few_load<T, V>(a.g, gb, t, c0);
            if constexpr (GATED) i[k] = few_load<T, V>(a.i, ib, t, c0);
            e[k] = few_load<T, V>(a.h, eb, t, c0);
        }
        auto enter = [&](const Few<T, V>& xs, const Few<T, V>& gs, const Few<T, V>& is, int j, float& dec) {
            const float y = rate[j] * sigmoid<T>(gs[j]);
            dec = carry_of(y);
            float w = xs[j];
            if constexpr (GATED) w *= sigmoid<T>(is[j]);
            return __builtin_amdgcn_sqrtf(room(y, dec)) * w;
        };
        for (int64_t t = t0 / kChunk * kChunk; t < t0; ++t) {
            const Few<T, V> xs = few_load<T, V>(a.x, xb, t, c0), gs = few_load<T, V>(a.g, gb, t, c0);
            Few<T, V> is = {};
            if constexpr (GATED) is = few_load<T, V>(a.i, ib, t, c0);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float dec;
                const float in = enter(xs, gs, is, j, dec);
                h[j] = __builtin_fmaf(dec, h[j], in);
            }
        }
#pragma unroll
        for (int k = 0; k < kFew; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                was[k][j] = h[j];
                const float in = enter(x[k], g[k], i[k], j, decays[k][j]);
                h[j] = __builtin_fmaf(decays[k][j], h[j], in);
            }
#pragma unroll
        for (int k = kFew - 1; k >= 0; --k) {
            if (k >= n) continue;
            float dx[V], dg[V], di[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float sg = sigmoid<T>(g[k][j]), y = rate[j] * sg, dec = decays[k][j], q = room(y, dec);
                const float inv = q >= 0x1p-126f ? __builtin_amdgcn_rsqf(q) : q * 0.0f, xv = x[k][j];
                float in = q * inv, near = dec * inv, si = 1.0f;
                if constexpr (GATED) {
                    si = sigmoid<T>(i[k][j]);
                    in *= si;
                    near *= si;
                }
                const float l = e[k][j] + m[j];
                m[j] = dec * l;
                const float d = sg * (m[j] * __builtin_fmaf(-near, xv, was[k][j]));
                dr[j] -= d;
                dg[j] = -kLn2 * rate[j] * __builtin_fmaf(-sg, d, d);
                dx[j] = l * in;
                if constexpr (GATED) di[j] = dx[j] * __builtin_fmaf(-xv, si, xv);
            }
            few_store<T, V>(a.dx, dxb, t0 + k, c0, dx);
            few_store<T, V>(a.dg, dgb, t0 + k, c0, dg);
            if constexpr (GATED) few_store<T, V>(a.di, dib, t0 + k, c0, di);
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (a.last) a.last[mine + j] = m[j];
        a.drate[mine + j] = dr[j];
    }
}

// ---------------------------------------------------------------- host
int refuse(int code, const char* who, const char* why) {
    set_error("%s: %s", who, why);
    return code;
}

int check_shape(const R97qRecurrence* p, const char* who) {
    if (!p) return refuse(R97Q_EINVAL, who, "null shape");
    if (p->batch < 0 || p->len < 0 || p->channels < 1) return refuse(R97Q_EINVAL, who, "a negative batch or length, or no channel");
    if (p->starts && p->tokens < 0) return refuse(R97Q_EINVAL, who, "a negative count of packed tokens");
    if (p->dtype != R97Q_BF16 && p->dtype != R97Q_F32) return refuse(R97Q_EINVAL, who, "the type is bf16 or f32");
    if (p->batch > 65535) return refuse(R97Q_EUNSUPPORTED, who, "at most 65535 sequences");
    // the launches' work items and a row's bytes stay below 2^32 and 2^31
    if (p->channels > (1 << 27)) return refuse(R97Q_EUNSUPPORTED, who, "at most 2^27 channels");
    if (p->len > 0x7FFFFFFF || (p->starts && p->tokens > 0x7FFFFFFF)) return refuse(R97Q_EUNSUPPORTED, who, "tokens within 31 bits");
    return R97Q_OK;
}

int check_rows(const R97qRows* t, const R97qRecurrence* p, bool output, const char* who, const char* name) {
    const int64_t tokens = p->starts ? p->tokens : p->len;
    if (!t || (!t->data && p->batch > 0 && tokens > 0)) {
        set_error("%s: %s is null", who, name);
        return R97Q_EINVAL;
    }
    if (t->token_stride < 0 || (!p->starts && t->batch_stride < 0) ||
        (output && ((tokens > 1 && !t->token_stride) || (!p->starts && p->batch > 1 && tokens > 0 && !t->batch_stride)))) {
        set_error("%s: %s has a negative stride, or is written through a stride of zero", who, name);
        return R97Q_EINVAL;
    }
    if (output && tokens > 1 && t->token_stride > 0 && t->token_stride < p->channels) {
        set_error("%s: %s is written with its tokens less than a row apart", who, name);
        return R97Q_EINVAL;
    }
    if (reinterpret_cast<uintptr_t>(t->data) & (p->dtype == R97Q_F32 ? 3 : 1)) {
        set_error("%s: %s is off its type's alignment", who, name);
        return R97Q_EINVAL;
    }
    return R97Q_OK;
}

// A lone sequence's and a lone token's strides say nothing. The token's is taken as a row: a tile's places past the last token
// are told by their offsets, which have to lie past its row.
Rows rows_of(const R97qRows* t, const R97qRecurrence* p) {
    if (!t) return {};
    return {static_cast<uint8_t*>(t->data), p->batch > 1 ? t->batch_stride : 0,
            (p->starts ? p->tokens : p->len) > 1 ? t->token_stride : p->channels};
}

// whether a launch's workgroups are dealt by XCD
bool lines_shared(const R97qRecurrence* p, const Args& a) {
    const int64_t size = p->dtype == R97Q_F32 ? 4 : 2, slabs = (p->channels + kSlab - 1) / kSlab;
    const bool off = (reinterpret_cast<uintptr_t>(a.x.p) | (uintptr_t)(a.x.ts * size)) & 127;
    return off && slabs >= 4 && slabs * a.ranges * a.fine * a.batch <= (1 << 20);
}

// pieces: a tile's rows lie within 31 bits of its first
bool wide(const Rows& t) { return t.ts <= (1 << 20); }

int64_t all_tokens(const R97qRecurrence* p) { return p->starts ? p->tokens : p->batch * p->len; }

// How a call is cut. Measured, us forward / backward, bf16 with a gate on the input:
// A thread a sequence, against tiles: 32 sequences of 4096 channels, 16 tokens 10 / 21 against 36 / 58, 32 tokens 17 / 46 against
// 36 / 58, 64 tokens 32 forward; 4 of 1024, 16 tokens 9 / 18 in both, 32 tokens 13 / 37 against 9 / 18. So up to 16 tokens, and
// forward up to 64 where the tiles' workgroups fill the card several times over.
// Ranges of at least 128 tokens, as many as make 256 workgroups (a compute unit holds one of most of the second launch's forms; of
// the spans' it holds two or three, which `fine` does not use), against none: 1 x 512 x 1024 15 / 22 against 14 / 22, 4 x 600 x
// 512 17 / 22 against 17 / 29, 1 x 768 x 512 16 / 21 against 19 / 31, 1 x 1024 x 2048 17 / 21 against 25 / 41, 1 x 16384 x 1024
// 53 / 64 against 345 / 584. 8 x 2048 x 2048, 256 workgroups whole, forward 67; two ranges 100. Two ranges of 86 .. 128
// workgroups were not measured against none. Packed sequences go by their mean: a long one among many short ones is not cut.
void cut(const R97qRecurrence* p, bool back, Args& a) {
    const int64_t slabs = (p->channels + kSlab - 1) / kSlab, have = slabs * p->batch;
    const int64_t mean = p->batch ? all_tokens(p) / p->batch : 0, most = p->len > mean ? p->len : mean;
    a.few = most <= 16 || (!back && most <= 64 && have >= 1024);
    int64_t n = have > 0 && mean >= (back ? 512 : 640) ? 256 / have : 1;
    if (n > mean / 128) n = mean / 128;
    if (n < 1) n = 1;
    a.range_len = ((most + n - 1) / n + kChunk - 1) / kChunk * kChunk;
    if (a.range_len < kChunk) a.range_len = kChunk;
    a.ranges = (int32_t)((most + a.range_len - 1) / a.range_len);
    if (a.ranges < 1) a.ranges = 1;
    // the spans' launch has one range's workgroups less: where that leaves half of them out, two spans a range and more
    a.fine = a.ranges > 1 ? (int32_t)(256 / ((a.ranges - 1) * have)) : 1;
    while (a.fine > 1 && a.range_len % (64 * a.fine)) --a.fine;
    if (a.fine < 1) a.fine = 1;
    a.span_len = a.range_len / a.fine;
}

Args args_of(const R97qRecurrence* p, bool back) {
    Args a = {};
    a.starts = p->starts;
    a.tokens = p->tokens;
    a.len = p->len;
    a.batch = p->batch;
    a.channels = p->channels;
    cut(p, back, a);
    return a;
}
int64_t spans_bytes(const Args& a) { return a.ranges > 1 ? (8LL * a.batch * a.ranges * a.fine * a.channels + 255) / 256 * 256 : 0; }
int64_t row_bytes(const Args& a, int64_t rows) { return (4 * rows * a.channels + 255) / 256 * 256; }

// A launch's grid over slabs, `ranges` and sequences. Rows that do not begin with a line of 128 bytes have slabs that share
// lines, and each XCD has its own L2: then an XCD's workgroups are neighbours.
dim3 deal(const Args& a, int ranges) {
    const unsigned slabs = (unsigned)((a.channels + kSlab - 1) / kSlab);
    return a.dealt ? dim3((slabs * (unsigned)ranges * (unsigned)a.batch + 7) / 8 * 8) : dim3(slabs, (unsigned)ranges, (unsigned)a.batch);
}
template <class T, bool GATED, bool WIDE>
int run_fwd(const Args& a, hipStream_t st) {
    if (a.ranges > 1) {
        hipLaunchKernelGGL((recurrence_spans_kernel<T, GATED, WIDE, false>), deal(a, (a.ranges - 1) * a.fine), dim3(kThreads), 0, st, a);
        if (int e = launch_status("recurrence_spans_kernel")) return e;
    }
    hipLaunchKernelGGL((recurrence_fwd_kernel<T, GATED, WIDE>), deal(a, a.ranges), dim3(kThreads), 0, st, a);
    return launch_status("recurrence_fwd_kernel");
}
template <class T, bool GATED, bool WIDE>
int run_bwd(const Args& a, hipStream_t st) {
    if (a.ranges > 1) {
        hipLaunchKernelGGL((recurrence_spans_kernel<T, false, WIDE, true>), deal(a, (a.ranges - 1) * a.fine), dim3(kThreads), 0, st, a);
        if (int e = launch_status("recurrence_spans_kernel")) return e;
    }
    hipLaunchKernelGGL((recurrence_bwd_kernel<T, GATED, WIDE>), deal(a, a.ranges), dim3(kThreads), 0, st, a);
    return launch_status("recurrence_bwd_kernel");
}
template <class T, int V, bool GATED>
int run_few(const Args& a, bool back, hipStream_t st) {
    const dim3 grid((unsigned)((a.channels + V * kFewThreads - 1) / (V * kFewThreads)), (unsigned)a.batch);
    if (back) hipLaunchKernelGGL((recurrence_few_bwd_kernel<T, V, GATED>), grid, dim3(kFewThreads), 0, st, a);
    else hipLaunchKernelGGL((recurrence_few_fwd_kernel<T, V, GATED>), grid, dim3(kFewThreads), 0, st, a);
    return launch_status("recurrence_few_kernel");
}
template <class T>
int pick(const Args& a, bool back, bool wide, hipStream_t st) {
    if (a.few) {
        if (a.i.p) return wide ? run_few<T, 4, true>(a, back, st) : run_few<T, 1, true>(a, back, st);
        return wide ? run_few<T, 4, false>(a, back, st) : run_few<T, 1, false>(a, back, st);
    }
    if (a.i.p) {
        if (wide) return back ? run_bwd<T, true, true>(a, st) : run_fwd<T, true, true>(a, st);
        return back ? run_bwd<T, true, false>(a, st) : run_fwd<T, true, false>(a, st);
    }
    if (wide) return back ? run_bwd<T, false, true>(a, st) : run_fwd<T, false, true>(a, st);
    return back ? run_bwd<T, false, false>(a, st) : run_fwd<T, false, false>(a, st);
}

}  // namespace
}  // namespace scan
}  // namespace r97q

using namespace r97q;
using namespace r97q::scan;

extern "C" {

int64_t r97q_recurrence_state_rows(const R97qRecurrence* shape) {
    clear_error();
    if (check_shape(shape, "r97q_recurrence_state_rows")) return -1;
    return shape->starts ? shape->tokens / kChunk + shape->batch : shape->batch * ((shape->len + kChunk - 1) / kChunk);
}

int64_t r97q_recurrence_fwd_workspace_bytes(const R97qRecurrence* shape) {
    clear_error();
    if (check_shape(shape, "r97q_recurrence_fwd_workspace_bytes")) return -1;
    const Args a = args_of(shape, false);
    return a.ranges > 1 ? spans_bytes(a) + row_bytes(a, a.batch) : 0;
}

int r97q_recurrence_fwd(const R97qRecurrence* shape, const R97qRows* x, const R97qRows* gate, const R97qRows* input_gate,
                        const float* rate, const float* h0, const R97qRows* h, float* last, float* states, void* workspace,
                        int64_t workspace_bytes, R97IqrStream stream) {
    clear_error();
    const char* who = "r97q_recurrence_fwd";
    if (int e = check_shape(shape, who)) return e;
    if (int e = check_rows(x, shape, false, who, "x")) return e;
    if (int e = check_rows(gate, shape, false, who, "gate")) return e;
    if (input_gate)
        if (int e = check_rows(input_gate, shape, false, who, "input_gate")) return e;
    if (int e = check_rows(h, shape, true, who, "h")) return e;
    if (!rate) return refuse(R97Q_EINVAL, who, "null rate");
    if (shape->batch == 0) return R97Q_OK;
    Args a = args_of(shape, false);
    const int64_t need = a.ranges > 1 ? spans_bytes(a) + row_bytes(a, a.batch) : 0;
    if (need > 0 && (!workspace || workspace_bytes < need)) return refuse(R97Q_EWORKSPACE, who, "the workspace is too small");
    if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15)) return refuse(R97Q_EINVAL, who, "the workspace starts on 16 bytes");
    a.x = rows_of(x, shape);
    a.g = rows_of(gate, shape);
    a.i = rows_of(all_tokens(shape) > 0 ? input_gate : nullptr, shape);
    a.h = rows_of(h, shape);
    a.rate = rate;
    a.first = h0;
    a.last = last;
    a.states = states;
    a.spans = static_cast<float2*>(workspace);
    a.kept = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + spans_bytes(a));
    a.dealt = lines_shared(shape, a);
    // The last piece's channels that are its neighbour's too are read twice, by two workgroups at times: not where one of them may
    // have written over them. Odd widths in place go value by value (8 x 2048 x 2047 forward 138 us, else 66).
    const int unit = shape->dtype == R97Q_F32 ? 4 : 8;
    bool over = h0 && h0 == last;
    for (const Rows& in : {a.x, a.g, a.i}) {
        if (!in.p || in.p != a.h.p) continue;
        if (in.ts != a.h.ts || (!shape->starts && in.bs != a.h.bs))
            return refuse(R97Q_EINVAL, who, "h over an input has that input's strides");
        over = true;
    }
    const bool w = a.channels >= unit && (a.channels % unit == 0 || !over) && wide(a.x) && wide(a.g) && wide(a.i) && wide(a.h);
    return shape->dtype == R97Q_F32 ? pick<float>(a, false, w, (hipStream_t)stream) : pick<uint16_t>(a, false, w, (hipStream_t)stream);
}

int64_t r97q_recurrence_bwd_workspace_bytes(const R97qRecurrence* shape) {
    clear_error();
    if (check_shape(shape, "r97q_recurrence_bwd_workspace_bytes")) return -1;
    const Args a = args_of(shape, true);
    const int64_t rows = (int64_t)a.batch * a.ranges;
    return spans_bytes(a) + (rows > 1 ? row_bytes(a, rows) : 0);
}

int r97q_recurrence_bwd(const R97qRecurrence* shape, const R97qRows* x, const R97qRows* gate, const R97qRows* input_gate,
                        const float* rate, const float* states, const R97qRows* d_h, const float* d_last, const R97qRows* dx,
                        const R97qRows* dgate, const R97qRows* dinput_gate, float* drate, float* dh0, void* workspace,
                        int64_t workspace_bytes, R97IqrStream stream) {
    clear_error();
    const char* who = "r97q_recurrence_bwd";
    if (int e = check_shape(shape, who)) return e;
    if (int e = check_rows(x, shape, false, who, "x")) return e;
    if (int e = check_rows(gate, shape, false, who, "gate")) return e;
    if (!input_gate != !dinput_gate) return refuse(R97Q_EINVAL, who, "input_gate and dinput_gate come together");
    if (input_gate) {
        if (int e = check_rows(input_gate, shape, false, who, "input_gate")) return e;
        if (int e = check_rows(dinput_gate, shape, true, who, "dinput_gate")) return e;
    }
    if (int e = check_rows(d_h, shape, false, who, "d_h")) return e;
    if (int e = check_rows(dx, shape, true, who, "dx")) return e;
    if (int e = check_rows(dgate, shape, true, who, "dgate")) return e;
    if (!rate || !drate) return refuse(R97Q_EINVAL, who, "null rate or drate");
    if (!states && shape->batch > 0 && all_tokens(shape) > 0) return refuse(R97Q_EINVAL, who, "null states");
    Args a = args_of(shape, true);
    hipStream_t st = (hipStream_t)stream;
    const int64_t rows = (int64_t)a.batch * a.ranges, need = spans_bytes(a) + (rows > 1 ? row_bytes(a, rows) : 0);
    if (need > 0 && (!workspace || workspace_bytes < need)) return refuse(R97Q_EWORKSPACE, who, "the workspace is too small");
    if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15)) return refuse(R97Q_EINVAL, who, "the workspace starts on 16 bytes");
    // ranges read what others write: d_last and dh0 are two tensors, and so are an input and an output
    const R97qRows *ins[] = {x, gate, input_gate, d_h}, *outs[] = {dx, dgate, dinput_gate};
    bool over = d_last && d_last == dh0;
    for (const R97qRows* out : outs) {
        for (const R97qRows* in : ins) over |= in && out && out->data && in->data == out->data;
        for (const R97qRows* other : outs) over |= out && other && out != other && out->data && other->data == out->data;
    }
    if (over) return refuse(R97Q_EINVAL, who, "an output over an input or another output");
    a.x = rows_of(x, shape);
    a.g = rows_of(gate, shape);
    a.i = rows_of(all_tokens(shape) > 0 ? input_gate : nullptr, shape);
    a.h = rows_of(d_h, shape);
    a.dx = rows_of(dx, shape);
    a.dg = rows_of(dgate, shape);
    a.di = rows_of(dinput_gate, shape);
    a.rate = rate;
    a.first = d_last;
    a.last = dh0;
    a.states = const_cast<float*>(states);
    a.spans = static_cast<float2*>(workspace);
    a.drate = rows > 1 ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + spans_bytes(a)) : drate;
    a.dealt = lines_shared(shape, a);
    const bool w = a.channels >= (shape->dtype == R97Q_F32 ? 4 : 8) && wide(a.x) && wide(a.g) && wide(a.i) && wide(a.h) && wide(a.dx) &&
                   wide(a.dg) && wide(a.di);
    if (rows > 0)
        if (int e = shape->dtype == R97Q_F32 ? pick<float>(a, true, w, st) : pick<uint16_t>(a, true, w, st)) return e;
    if (rows == 1) return R97Q_OK;
    hipLaunchKernelGGL(recurrence_rate_kernel, dim3((unsigned)((a.channels + 63) / 64)), dim3(64 * kShares), 0, st, a.drate, drate, rows,
                       a.channels);
    return launch_status("recurrence_rate_kernel");
}

}  // extern "C"
