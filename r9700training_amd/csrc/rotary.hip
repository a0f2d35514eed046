// rotary.hip -- rotary positions of the query and key heads, forward and adjoint, in one launch.
//
// A pair (u, v) at position p turns by a = p f_i: (u cos a - v sin a, u sin a + v cos a). The angle goes
// through f64 as a number of turns, p f_i / 2 pi less its nearest whole number, so that a position of
// millions keeps its phase; the sine and cosine of what is left and the rotation are f32, and an output
// is rounded once.
//
// Bound by memory: each value is read and written once. A workgroup takes a few tokens, forms their sines
// and cosines once in LDS (rot / 2 a token, against heads * rot / 2 pairs that use them) and then walks the
// tokens' heads in 16-byte pieces, kItems pieces of a thread in flight together. With several axes a token has a position on
// each and a pair an axis: only the table's positions differ. 16384 tokens, 40 heads of 128: 73 us, as
// neighbouring pairs 75 (4.5 TB/s; a 1 GiB copy reaches 4.9), with three axes 77 .. 79. One token: 4.4 us, latency.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/r97q.h"
#include "iqr_device.h"
#include "status.h"

namespace r97q {
namespace {

constexpr int kThreads = 256;
constexpr int kItems = 4;
constexpr int kTable = 4096;  // (sin, cos) pairs of a workgroup's tokens in LDS: 32 KiB

struct RHeads {
    const void* in;
    void* out;
    int64_t its, ihs, ots, ohs;  // strides of a token and a head, in elements
};

struct RArgs {
    RHeads q, k;
    int32_t hq, heads;   // q's heads, and all of them
    int64_t tokens;
    int32_t tpb;         // tokens a workgroup
    int32_t half;        // pairs
    int32_t turn, copy;  // pieces of a head that turn, and that are copied
    const double* freq;
    const void* pos;
    int32_t pos64, inverse;
    float mscale;
    const int32_t* axis;  // each pair's axis, its positions axis_stride apart; null: one position a token
    int64_t axis_stride;
    int32_t axes;
};

// V values, in one load where they are aligned (WIDE)
template <class T, int V, bool WIDE>
struct Piece {
    static constexpr int kBytes = V * (int)sizeof(T);
    float x[V];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (WIDE && sizeof(T) == 2 && V > 1) {
            uint32_t u[V / 2];
            if constexpr (kBytes == 16)
                *reinterpret_cast<uint4*>(u) = *reinterpret_cast<const uint4*>(p);
            else if constexpr (kBytes == 8)
                *reinterpret_cast<uint2*>(u) = *reinterpret_cast<const uint2*>(p);
            else
                u[0] = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                x[2 * i] = __builtin_bit_cast(float, u[i] << 16);
                x[2 * i + 1] = __builtin_bit_cast(float, u[i] & 0xFFFF0000u);
            }
        } else if constexpr (WIDE && kBytes == 16) {
            *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p);
        } else if constexpr (WIDE && kBytes == 8) {
            *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(p);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if constexpr (sizeof(T) == 2)
                    x[i] = bf16_to_f32(p[i]);
                else
                    x[i] = p[i];
            }
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (WIDE && sizeof(T) == 2 && V > 1) {
            using b2 = __attribute__((ext_vector_type(2))) __bf16;
            uint32_t u[V / 2];
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                b2 v = {(__bf16)x[2 * i], (__bf16)x[2 * i + 1]};
                u[i] = __builtin_bit_cast(uint32_t, v);
            }
            if constexpr (kBytes == 16)
                *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(u);
            else if constexpr (kBytes == 8)
                *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(u);
            else
                *reinterpret_cast<uint32_t*>(p) = u[0];
        } else if constexpr (WIDE && kBytes == 16) {
            *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(x);
        } else if constexpr (WIDE && kBytes == 8) {
            *reinterpret_cast<float2*>(p) = *reinterpret_cast<const float2*>(x);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if constexpr (sizeof(T) == 2)
                    p[i] = f32_to_bf16(x[i]);
                else
                    p[i] = x[i];
            }
        }
    }
};

// V: values a piece: 16 bytes, or as many fewer as widths and places allow, down to one (a neighbouring pair: two, one by
// one). 16384 tokens, 10 heads of 96 of which 24 turn in halves of 12: 73 us a value at a time, 23 in 8 bytes.
// NEAR: neighbouring pairs, else the halves' ones.
template <class T, int V, bool NEAR, bool WIDE>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RArgs a) {
    __shared__ float2 table[kTable];  // (cos, sin) * mscale
    const int64_t t0 = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * a.tpb;
    if (t0 >= a.tokens) return;
    const int nt = a.tokens - t0 < a.tpb ? (int)(a.tokens - t0) : a.tpb;
    for (int i = threadIdx.x; i < nt * a.half; i += kThreads) {
        const int64_t t = t0 + i / a.half;
        double p;
        if (!a.axis) {
            p = !a.pos ? (double)t
                : a.pos64 ? (double)static_cast<const int64_t*>(a.pos)[t] : (double)static_cast<const int32_t*>(a.pos)[t];
        } else {
            const int ax = a.axis[i % a.half];
            const bool one = (uint32_t)ax < (uint32_t)a.axes;
            const int64_t at = one ? ax * a.axis_stride + t : 0;
            p = !one ? 0.0 : a.pos64 ? (double)static_cast<const int64_t*>(a.pos)[at] : (double)static_cast<const int32_t*>(a.pos)[at];
        }
        double turns = p * a.freq[i % a.half] * 0.15915494309189534;
        turns -= rint(turns);
        float s, c;
        sincospif(2.0f * (float)turns, &s, &c);
        table[i] = make_float2(c * a.mscale, (a.inverse ? -s : s) * a.mscale);
    }
    __syncthreads();
    const int per = a.turn + a.copy, n = nt * a.heads * per, step = kThreads * (int)gridDim.y;
    for (int i0 = (int)blockIdx.y * kThreads + threadIdx.x; i0 < n; i0 += kItems * step) {
        Piece<T, V, WIDE> u[kItems], v[kItems];
        T* out[kItems];
        int at[kItems];  // the piece's first pair in the table; -1: copied
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
            const int i = i0 + j * step < n ? i0 + j * step : i0;
            const int c = i % per, hh = i / per, head = hh % a.heads, t = hh / a.heads;
            const RHeads& x = head < a.hq ? a.q : a.k;
            const int hx = head < a.hq ? head : head - a.hq;
            const bool turns = c < a.turn;
            const int e = turns ? V * c : 2 * a.half + V * (c - a.turn);
            const T* in = static_cast<const T*>(x.in) + (t0 + t) * x.its + hx * x.ihs + e;
            out[j] = static_cast<T*>(x.out) + (t0 + t) * x.ots + hx * x.ohs + e;
            at[j] = !turns ? -1 : t * a.half + (NEAR ? e / 2 : e);
            u[j].load(in);
            if (!NEAR && turns) v[j].load(in + a.half);
        }
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
            if (i0 + j * step >= n) break;
            if (at[j] >= 0) {
                if constexpr (NEAR) {
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) {
                        const float2 w = table[at[j] + e];
                        const float x = u[j].x[2 * e], y = u[j].x[2 * e + 1];
                        u[j].x[2 * e] = x * w.x - y * w.y;
                        u[j].x[2 * e + 1] = x * w.y + y * w.x;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float2 w = table[at[j] + e];
                        const float x = u[j].x[e], y = v[j].x[e];
                        u[j].x[e] = x * w.x - y * w.y;
                        v[j].x[e] = x * w.y + y * w.x;
                    }
                    v[j].store(out[j] + a.half);
                }
            }
            u[j].store(out[j]);
        }
    }
}

int refuse(int code, const char* who, const char* why) {
    set_error("%s: %s", who, why);
    return code;
}

bool on(const R97qHeads* t, int unit, int size) {  // pieces of `unit` values are aligned
    return (reinterpret_cast<uintptr_t>(t->data) & (unit * size - 1)) == 0 && t->token_stride % unit == 0 && t->head_stride % unit == 0;
}

int check_pair(const R97qHeads* in, const R97qHeads* out, int32_t dtype, int64_t tokens, const char* who) {
    if (!in || !out || ((!in->data || !out->data) && tokens > 0)) return refuse(R97Q_EINVAL, who, "null heads");
    if (in->dtype != dtype || out->dtype != dtype) return refuse(R97Q_EINVAL, who, "q, k and the outputs are all bf16 or all f32");
    if (in->heads < 1 || out->heads != in->heads) return refuse(R97Q_EINVAL, who, "an output has its input's heads, one or more");
    if (in->token_stride < 0 || in->head_stride < 0 || out->token_stride < 0 || out->head_stride < 0 ||
        (tokens > 1 && !out->token_stride) || (out->heads > 1 && !out->head_stride))
        return refuse(R97Q_EINVAL, who, "a negative stride, or an output with a stride of zero");
    return R97Q_OK;
}

template <class T, int V, bool NEAR, bool WIDE>
int launch(RArgs a, int32_t head_dim, bool in_place, hipStream_t st) {
    a.turn = 2 * a.half / (NEAR ? V : 2 * V);
    a.copy = in_place ? 0 : (head_dim - 2 * a.half) / V;
    // pieces of about 8 rounds of a workgroup's threads, and a table that fits; few tokens: their heads over
    // more workgroups, a round each
    const int64_t per = (int64_t)a.heads * (a.turn + a.copy);
    int64_t tpb = 8 * kThreads / (per < 1 ? 1 : per);
    if (tpb > kTable / a.half) tpb = kTable / a.half;
    if (tpb < 1) tpb = 1;
    if (a.tokens < 256) tpb = 1;
    a.tpb = (int32_t)tpb;
    const int64_t blocks = (a.tokens + tpb - 1) / tpb;
    int64_t across = 1;
    if (blocks < 256) across = (per * tpb + kThreads - 1) / kThreads;
    if (across > 256) across = 256;
    // a launch's first dimension holds fewer than 2^32 threads: what is left goes along the third
    constexpr int64_t most = 0xFFFFFFFFLL / kThreads;
    const int64_t deep = (blocks + most - 1) / most, wide = (blocks + deep - 1) / deep;
    hipLaunchKernelGGL((rotary_kernel<T, V, NEAR, WIDE>), dim3((unsigned)wide, (unsigned)(across < 1 ? 1 : across), (unsigned)deep),
                       dim3(kThreads), 0, st, a);
    return launch_status("rotary_kernel");
}

// unit: the aligned values a piece may hold (1: none but single ones)
template <class T, bool NEAR>
int pick(const RArgs& a, int32_t head_dim, int unit, bool in_place, hipStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (unit == 8) return launch<T, 8, NEAR, true>(a, head_dim, in_place, st);
    if (unit == 4) return launch<T, 4, NEAR, true>(a, head_dim, in_place, st);
    if (unit == 2) return launch<T, 2, NEAR, true>(a, head_dim, in_place, st);
    return launch<T, NEAR ? 2 : 1, NEAR, false>(a, head_dim, in_place, st);
}

struct Axes {
    const int32_t* of_pair;
    int32_t count;
    int64_t stride;
};

int turn(const char* who, const R97qHeads* q, const R97qHeads* q_out, const R97qHeads* k, const R97qHeads* k_out, int64_t tokens,
         int32_t head_dim, int32_t rot, int32_t pairs, const double* inv_freq, const void* positions, int32_t positions64,
         const Axes& axes, float mscale, int32_t inverse, hipStream_t st) {
    if (!q || (q->dtype != R97Q_BF16 && q->dtype != R97Q_F32)) return refuse(R97Q_EINVAL, who, "q is bf16 or f32");
    if (tokens < 0 || tokens > 0x7FFFFFFF) return refuse(R97Q_EINVAL, who, "tokens within 31 bits");
    if (head_dim < 1 || rot < 2 || rot % 2 || rot > head_dim) return refuse(R97Q_EINVAL, who, "rot is even, at least 2 and at most head_dim");
    if (rot > 2 * kTable) return refuse(R97Q_EUNSUPPORTED, who, "at most 8192 values turn");
    if (pairs != R97Q_ROTARY_HALF && pairs != R97Q_ROTARY_INTERLEAVED) return refuse(R97Q_EINVAL, who, "pairs are half or interleaved");
    if (!inv_freq) return refuse(R97Q_EINVAL, who, "null frequencies");
    if (int e = check_pair(q, q_out, q->dtype, tokens, who)) return e;
    if (!k != !k_out) return refuse(R97Q_EINVAL, who, "k and k_out come together");
    if (k)
        if (int e = check_pair(k, k_out, q->dtype, tokens, who)) return e;
    const bool near = pairs == R97Q_ROTARY_INTERLEAVED;
    const int64_t heads = (int64_t)q->heads + (k ? k->heads : 0);
    if (heads * head_dim > 0x3FFFFFFF / 4) return refuse(R97Q_EUNSUPPORTED, who, "a token's heads pass 28 bits");
    if (tokens == 0) return R97Q_OK;
    const int size = q->dtype == R97Q_F32 ? 4 : 2;
    int unit = 16 / size;
    auto fits = [&](int u) {
        return on(q, u, size) && on(q_out, u, size) && (!k || (on(k, u, size) && on(k_out, u, size))) &&
               (near ? rot : rot / 2) % u == 0 && head_dim % u == 0;
    };
    while (unit > 1 && !fits(unit)) unit /= 2;
    auto same = [](const R97qHeads* x, const R97qHeads* y) {
        return x->data == y->data && x->token_stride == y->token_stride && x->head_stride == y->head_stride;
    };
    bool in_place = same(q, q_out) && (!k || same(k, k_out));
    // single values past an odd rest are copied one by one only in the halves' form: neighbouring pieces are two wide
    if (near && (head_dim - rot) % 2) return refuse(R97Q_EUNSUPPORTED, who, "neighbouring pairs need an even head_dim");
    RArgs a = {};
    auto heads_of = [](const R97qHeads* x, const R97qHeads* y) {
        return RHeads{x->data, y->data, x->token_stride, x->head_stride, y->token_stride, y->head_stride};
    };
    a.q = heads_of(q, q_out);
    if (k) a.k = heads_of(k, k_out);
    a.hq = q->heads;
    a.heads = (int32_t)heads;
    a.tokens = tokens;
    a.half = rot / 2;
    a.freq = inv_freq;
    a.pos = positions;
    a.pos64 = positions64;
    a.inverse = inverse;
    a.mscale = mscale;
    a.axis = axes.of_pair;
    a.axes = axes.count;
    a.axis_stride = axes.stride;
    if (q->dtype == R97Q_BF16)
        return near ? pick<uint16_t, true>(a, head_dim, unit, in_place, st) : pick<uint16_t, false>(a, head_dim, unit, in_place, st);
    return near ? pick<float, true>(a, head_dim, unit, in_place, st) : pick<float, false>(a, head_dim, unit, in_place, st);
}

}  // namespace
}  // namespace r97q

using namespace r97q;

extern "C" {

int r97q_rotary(const R97qHeads* q, const R97qHeads* q_out, const R97qHeads* k, const R97qHeads* k_out, int64_t tokens,
                int32_t head_dim, int32_t rot, int32_t pairs, const double* inv_freq, const void* positions,
                int32_t positions64, float mscale, int32_t inverse, R97IqrStream stream) {
    clear_error();
    return turn("r97q_rotary", q, q_out, k, k_out, tokens, head_dim, rot, pairs, inv_freq, positions, positions64, {nullptr, 1, 0}, mscale,
                inverse, (hipStream_t)stream);
}

int r97q_rotary_axes(const R97qHeads* q, const R97qHeads* q_out, const R97qHeads* k, const R97qHeads* k_out, int64_t tokens,
                     int32_t head_dim, int32_t rot, int32_t pairs, const double* inv_freq, const int32_t* pair_axis, int32_t axes,
                     const void* positions, int32_t positions64, int64_t axis_stride, float mscale, int32_t inverse, R97IqrStream stream) {
    clear_error();
    const char* who = "r97q_rotary_axes";
    if (axes < 1) return refuse(R97Q_EINVAL, who, "one axis or more");
    if (!pair_axis || (!positions && tokens > 0)) return refuse(R97Q_EINVAL, who, "null pair_axis or positions");
    if (axis_stride < 0) return refuse(R97Q_EINVAL, who, "a negative stride");
    return turn(who, q, q_out, k, k_out, tokens, head_dim, rot, pairs, inv_freq, positions, positions64, {pair_axis, axes, axis_stride},
                mscale, inverse, (hipStream_t)stream);
}

int r97q_rotary_frequencies(int32_t rot, double base, int32_t scaling, double factor, double original, double slow,
                            double fast, double* inv_freq, float* mscale) {
    clear_error();
    if (!inv_freq || rot < 2 || rot % 2 || !(base > 0.0)) {
        set_error("r97q_rotary_frequencies: null output, an odd rot or base <= 0");
        return R97Q_EINVAL;
    }
    if (scaling != R97Q_ROTARY_PLAIN && scaling != R97Q_ROTARY_LINEAR && scaling != R97Q_ROTARY_RAMP) {
        set_error("r97q_rotary_frequencies: scaling is plain, linear or ramp");
        return R97Q_EINVAL;
    }
    if ((scaling != R97Q_ROTARY_PLAIN && !(factor > 0.0)) ||
        (scaling == R97Q_ROTARY_RAMP && (!(original > 0.0) || !(fast > slow)))) {
        set_error("r97q_rotary_frequencies: factor > 0, and for the ramp original > 0 and fast > slow");
        return R97Q_EINVAL;
    }
    const int half = rot / 2;
    for (int i = 0; i < half; ++i) {
        const double f = std::pow(base, -(double)i / half);
        if (scaling == R97Q_ROTARY_PLAIN) {
            inv_freq[i] = f;
        } else if (scaling == R97Q_ROTARY_LINEAR) {
            inv_freq[i] = f / factor;
        } else {
            double keep = (original * f / 6.283185307179586 - slow) / (fast - slow);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
            inv_freq[i] = f * keep + f / factor * (1.0 - keep);
        }
    }
    if (mscale) *mscale = scaling == R97Q_ROTARY_RAMP ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return R97Q_OK;
}

}  // extern "C"
