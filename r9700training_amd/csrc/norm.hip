// norm.hip -- the residual's addition, the RMS norm and the 8-bit group quantiser in one pass, and their
// adjoint.
//
//   h = x + r (rounded to the stream's type),  rs = 1 / sqrt(mean h^2 + eps),  y = h rs (w + wadd),
//   scale = amax / 127 a group,  code = rint(y / scale)
//   adjoint, straight through the rounding: e = g_codes / scale + g_y,
//   dx = rs ((w + wadd) e - h rs^2 mean((w + wadd) e h)) + g_h,  dw = sum over rows of e h rs
//
// Bound by memory: a row is read once into registers (8 consecutive columns a thread and step), its sums
// taken across the threads, and everything written from there. Rows of up to 2048 columns belong to a
// wave, four of them to a workgroup, with no barrier; wider ones, up to 16384 columns, to a workgroup. Groups that are no
// multiple of 8 go a column at a time, up to 8192 of them; what is wider takes the general kernels, which read a row again
// for each stage. 16384 x 2048 bf16 with a residual, groups of 128, takes 41 us (5.8 TB/s; a 1 GiB copy reaches 4.9, one that
// fits the 256 MB cache 6.6), one row of 5120 4.0 us.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "../../include/r97q.h"
#include "group_lanes.h"
#include "iqr_device.h"
#include "status.h"

namespace r97q {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

struct NArgs {
    const void* x;         // forward: x; adjoint: h
    const void* res;
    const void* w;
    int64_t rows, n, group;  // group: 1 .. n
    int64_t ngroups;
    float eps, wadd;
    void* h;
    int8_t* codes;
    float* scale;          // forward: written; adjoint: read
    uint16_t* y;
    float* rstd;           // forward: written; adjoint: read
    const void *gc, *gy, *gh;
    void* dx;
    float* part;           // [blocks][n] partial sums of dw; null: no dw
};

template <class T>
__device__ __forceinline__ float ld(const void* p, int64_t i) {
    if constexpr (sizeof(T) == 2)
        return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
    else
        return static_cast<const float*>(p)[i];
}
template <class T>
__device__ __forceinline__ void put(void* p, int64_t i, float v) {
    if constexpr (sizeof(T) == 2)
        static_cast<uint16_t*>(p)[i] = __builtin_bit_cast(uint16_t, (__bf16)v);
    else
        static_cast<float*>(p)[i] = v;
}
template <class T>
__device__ __forceinline__ float as_stored(float v) {
    if constexpr (sizeof(T) == 2)
        return (float)(__bf16)v;
    else
        return v;
}

// the larger value, or the NaN where one is (fmaxf drops it), in one instruction
__device__ __forceinline__ float larger(float x, float y) { return __builtin_elementwise_maximum(x, y); }

// both values of the pair of lanes H apart
template <int H>
__device__ __forceinline__ void lane_pair(float v, float& lo, float& hi) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    if constexpr (H < 16) {
        lo = v;
        hi = __builtin_bit_cast(float, lanes::other<H>(x));
    } else {
        const auto s = H == 16 ? __builtin_amdgcn_permlane16_swap(x, x, false, false)
                               : __builtin_amdgcn_permlane32_swap(x, x, false, false);
        const uint32_t p = s[0], q = s[1];
        lo = __builtin_bit_cast(float, p);
        hi = __builtin_bit_cast(float, q);
    }
}
template <int H>
__device__ __forceinline__ float lane_sum(float v) {
    float lo, hi;
    lane_pair<H>(v, lo, hi);
    return lo + hi;
}
template <int H>
__device__ __forceinline__ float lane_max(float v) {
    float lo, hi;
    lane_pair<H>(v, lo, hi);
    return larger(lo, hi);
}
__device__ __forceinline__ float wave_sum(float v) {
    return lane_sum<32>(lane_sum<16>(lane_sum<8>(lane_sum<4>(lane_sum<2>(lane_sum<1>(v))))));
}
// the maximum over 2^lg neighbouring lanes, in all of them (lg uniform, 0 .. 6)
__device__ __forceinline__ float lanes_max(float v, int lg) {
    if (lg > 0) v = lane_max<1>(v);
    if (lg > 1) v = lane_max<2>(v);
    if (lg > 2) v = lane_max<4>(v);
    if (lg > 3) v = lane_max<8>(v);
    if (lg > 4) v = lane_max<16>(v);
    if (lg > 5) v = lane_max<32>(v);
    return v;
}
__device__ __forceinline__ float wave_max(float v) { return lanes_max(v, 6); }
// over the workgroup, the waves' values in wave order
__device__ float block_sum(float v, float* red) {
    const int waves = blockDim.x >> 6;
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = red[0];
    for (int i = 1; i < waves; ++i) t += red[i];
    return t;
}
__device__ float block_max(float v, float* red) {
    const int waves = blockDim.x >> 6;
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = red[0];
    for (int i = 1; i < waves; ++i) t = larger(t, red[i]);
    return t;
}

// 1 / sqrt(mean of h^2 + eps) from sum(f), a row's sum of (f h)^2. f32 holds the squares of values of some 1e-19 to 1e18, and
// most rows; where the sum leaves its range, upwards or (eps no larger) downwards, it is taken again of the values times a
// power of two that brings it back. The sum is the same in all the row's threads.
template <class Sum>
__device__ __forceinline__ float rstd_of(Sum&& sum, float n, float eps) {
    const float ss = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, sum(1.0f))));
    const bool small = ss < 0x1p-90f && eps < 0x1p-90f;
    if (ss < INFINITY && !small) return 1.0f / sqrtf(ss / n + eps);
    const float f = small ? 0x1p96f : 0x1p-80f;
    return f / sqrtf(sum(f) / n + eps * f * f);
}

// The quantiser of a group with maximum amax: code = rint(y * up * inv). up keeps 127 / amax finite where the
// group's values are tiny. A NaN or an infinity goes into the scale, and the codes say nothing then.
struct Quant {
    float scale, up, inv;
    __device__ __forceinline__ explicit Quant(float amax) {
        scale = amax == 0.0f ? 1.0f : amax / 127.0f;
        up = amax < 0x1p-96f ? 0x1p96f : 1.0f;
        inv = amax == 0.0f ? 0.0f : 127.0f / (amax * up);
    }
    __device__ __forceinline__ int code(float y) const { return (int)rintf(y * up * inv); }
    // in one word: up is one of two, and inv is not negative
    __device__ __forceinline__ float packed() const { return up == 1.0f ? inv : -inv; }
    static __device__ __forceinline__ int code_of(float y, float p) { return (int)rintf(y * (p < 0.0f ? 0x1p96f : 1.0f) * fabsf(p)); }
};

// The codes' cotangent at y, gc / scale, plus y's own. The two may cancel, so the quotient's rounding is
// carried into the sum. up keeps 1 / scale finite.
struct Cotangent {
    float scale, up, inv;
    __device__ __forceinline__ explicit Cotangent(float s) : scale(s), up(s < 0x1p-96f ? 0x1p96f : 1.0f), inv(1.0f / (s * up)) {}
    __device__ __forceinline__ float sum(float gc, float gy) const {
#pragma clang fp contract(off)  // rest is of the rounded q
        const float q = gc * up * inv, rest = fmaf(-q, scale, gc) * up * inv;
        return (q + gy) + rest;
    }
};

// ---------------------------------------------------------------- any width, group, place
// grid (rows). x may be h_out: a value is overwritten by the wave that was the last to read it. 2 x 17408 in groups of 256: a
// row's three passes one after the other, bound by latency.
template <class T>
__global__ __launch_bounds__(kThreads) void norm_any_kernel(NArgs a) {
    __shared__ float red[kWaves];
    const int64_t base = (int64_t)blockIdx.x * a.n;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto h_of = [&](int64_t j) {
        return a.res ? as_stored<T>(ld<T>(a.x, base + j) + ld<T>(a.res, base + j)) : ld<T>(a.x, base + j);
    };
    auto squares = [&](float f) {
        float ss = 0.0f;
        for (int64_t j = threadIdx.x; j < a.n; j += kThreads) {
            const float h = f * h_of(j);
            ss += h * h;
        }
        return block_sum(ss, red);
    };
    const float rs = rstd_of(squares, (float)a.n, a.eps);
    if (threadIdx.x == 0 && a.rstd) a.rstd[blockIdx.x] = rs;
    auto y_of = [&](int64_t j) { return h_of(j) * rs * (ld<T>(a.w, j) + a.wadd); };
    // one group: the workgroup's; more: a wave takes whole groups
    const bool one = a.ngroups == 1;
    const int first = one ? (int)threadIdx.x : lane, step = one ? kThreads : 64;
    for (int64_t g = one ? 0 : wave; g < a.ngroups; g += one ? 1 : kWaves) {
        const int64_t j0 = g * a.group, j1 = j0 + a.group < a.n ? j0 + a.group : a.n;
        float amax = 0.0f;
        for (int64_t j = j0 + first; j < j1; j += step) amax = larger(amax, fabsf(y_of(j)));
        amax = one ? block_max(amax, red) : wave_max(amax);
        const Quant q(amax);
        if (first == 0 && a.scale) a.scale[blockIdx.x * a.ngroups + g] = q.scale;
        for (int64_t j = j0 + first; j < j1; j += step) {
            const float h = h_of(j), y = h * rs * (ld<T>(a.w, j) + a.wadd);
            if (a.codes) a.codes[base + j] = (int8_t)q.code(y);
            if (a.y) a.y[base + j] = f32_to_bf16(y);
            if (a.res) put<T>(a.h, base + j, h);
        }
    }
}

// a workgroup takes rows blockIdx.x, + gridDim.x, ...
template <class T>
__global__ __launch_bounds__(kThreads) void norm_any_bwd_kernel(NArgs a) {
    __shared__ float red[kWaves];
    float* part = a.part ? a.part + (int64_t)blockIdx.x * a.n : nullptr;
    bool fresh = true;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, fresh = false) {
        const int64_t base = r * a.n;
        const float rs = a.rstd[r];
        auto e_of = [&](int64_t j) {
            const float gy = a.gy ? ld<T>(a.gy, base + j) : 0.0f;
            return a.gc ? Cotangent(a.scale[r * a.ngroups + j / a.group]).sum(ld<T>(a.gc, base + j), gy) : gy;
        };
        float dot = 0.0f;
        for (int64_t j = threadIdx.x; j < a.n; j += kThreads)
            dot += (ld<T>(a.w, j) + a.wadd) * e_of(j) * (ld<T>(a.x, base + j) * rs);
        const float mean = block_sum(dot, red) / (float)a.n;
        for (int64_t j = threadIdx.x; j < a.n; j += kThreads) {
            const float e = e_of(j), x = ld<T>(a.x, base + j) * rs;
            float d = rs * ((ld<T>(a.w, j) + a.wadd) * e - x * mean);
            if (a.gh) d += ld<T>(a.gh, base + j);
            put<T>(a.dx, base + j, d);
            if (part) part[j] = fresh ? e * x : part[j] + e * x;
        }
    }
}

// ---------------------------------------------------------------- rows in registers
// A row belongs to a wave (WIDE false, four to a workgroup) or to the workgroup. A thread holds S pieces of V columns,
// V * (threads a row) apart. V 8: 16 bytes of bf16 a load; a wave's 64 pieces are 512 neighbouring columns and a group of
// 8 .. 512 columns (a power of two) lies in 2^lg neighbouring lanes; other multiples of 8 have their maximum gathered in LDS
// (a maximum is the same in any order). LOOSE: pieces of odd widths and unaligned tensors, 16 bytes at any place and the
// row's last piece value by value: 16384 x 1001 bf16 in groups of 128 20 us and back 29 (4.9 TB/s), where single columns took
// 52 and 98. V 1: groups that are no multiple of 8. lg kWhole: one group, the whole row; kGathered:
// through LDS.
constexpr int kMostWaves = 16;
constexpr int kWhole = -1, kGathered = -2;

// words at any place, in one access
template <int N>
struct __attribute__((packed)) Words {
    uint32_t u[N];
};

// A piece as it lies in memory: it is taken apart after the branches that load it, so that all pieces' loads go out
// together. `left` columns are left of the row from the piece's first on: LOOSE pieces may be its short last one, or (left
// <= 0) past it. What is not there is zero.
template <class T, int V, bool LOOSE>
struct Piece {
    static constexpr int N = V == 1 ? 1 : V * (int)sizeof(T) / 4;
    uint32_t u[N];
    __device__ __forceinline__ void load(const void* from, int64_t i, int left) {
        const T* p = static_cast<const T*>(from) + i;
#pragma unroll
        for (int k = 0; k < N; ++k) u[k] = 0;
        if constexpr (V == 1) {
            if (left > 0) u[0] = sizeof(T) == 2 ? (uint32_t)*reinterpret_cast<const uint16_t*>(p) : *reinterpret_cast<const uint32_t*>(p);
        } else if (left >= V) {
#pragma unroll
            for (int j = 0; j < N / 4; ++j) {
                if constexpr (LOOSE) {
                    const auto w = reinterpret_cast<const Words<4>*>(p)[j];
#pragma unroll
                    for (int k = 0; k < 4; ++k) u[4 * j + k] = w.u[k];
                } else {
                    const uint4 w = reinterpret_cast<const uint4*>(p)[j];
                    u[4 * j] = w.x, u[4 * j + 1] = w.y, u[4 * j + 2] = w.z, u[4 * j + 3] = w.w;
                }
            }
        } else if (LOOSE && left > 0) {
#pragma unroll
            for (int k = 0; k < V - 1; ++k) {
                if (k >= left) break;
                if constexpr (sizeof(T) == 2)
                    u[k / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[k] << (16 * (k % 2));
                else
                    u[k] = reinterpret_cast<const uint32_t*>(p)[k];
            }
        }
    }
    __device__ __forceinline__ float at(int k) const {
        if constexpr (sizeof(T) == 2) {
            if constexpr (V == 1) return __builtin_bit_cast(float, u[0] << 16);
            return __builtin_bit_cast(float, k % 2 ? u[k / 2] & 0xFFFF0000u : u[k / 2] << 16);
        } else {
            return __builtin_bit_cast(float, u[k]);
        }
    }
    static __device__ __forceinline__ void store(void* to, int64_t i, int left, const float (&x)[V]) {
        T* p = static_cast<T*>(to) + i;
        if constexpr (V == 1) {
            if (left > 0) put<T>(to, i, x[0]);
        } else if (left >= V) {
            uint32_t w[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                if constexpr (sizeof(T) == 2) {
                    using b2 = __attribute__((ext_vector_type(2))) __bf16;
                    b2 v = {(__bf16)x[2 * k], (__bf16)x[2 * k + 1]};
                    w[k] = __builtin_bit_cast(uint32_t, v);
                } else {
                    w[k] = __builtin_bit_cast(uint32_t, x[k]);
                }
            }
#pragma unroll
            for (int j = 0; j < N / 4; ++j) {
                if constexpr (LOOSE)
                    reinterpret_cast<Words<4>*>(p)[j] = {{w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]}};
                else
                    reinterpret_cast<uint4*>(p)[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
            }
        } else if (LOOSE && left > 0) {
#pragma unroll
            for (int k = 0; k < V - 1; ++k)
                if (k < left) put<T>(to, i + k, x[k]);
        }
    }
};

template <class T, int S, bool WIDE, int V, bool LOOSE>
__global__ __launch_bounds__(WIDE ? 1024 : 256) void norm_rows_kernel(NArgs a, int lg, uint32_t magic) {
    __shared__ float red[kMostWaves];
    extern __shared__ uint32_t gathered[];  // the groups' maxima, as bits (they are not negative, and a NaN's are the largest); of single columns then their quantisers
    const int wave = threadIdx.x >> 6, t = WIDE ? threadIdx.x : threadIdx.x & 63, per = WIDE ? blockDim.x : 64;
    const int64_t row = WIDE ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    if (row >= a.rows) return;
    const int n = (int)a.n;
    const int64_t base = row * n;
    using P = Piece<T, V, LOOSE>;
    P x[S], w[S];
#pragma unroll
    for (int i = 0; i < S; ++i) x[i].load(a.x, base + V * (t + i * per), n - V * (t + i * per));
    float h[S][V];
    if (a.res) {
        P r[S];
#pragma unroll
        for (int i = 0; i < S; ++i) r[i].load(a.res, base + V * (t + i * per), n - V * (t + i * per));
#pragma unroll
        for (int i = 0; i < S; ++i) w[i].load(a.w, V * (t + i * per), n - V * (t + i * per));
#pragma unroll
        for (int i = 0; i < S; ++i) {
#pragma unroll
            for (int k = 0; k < V; ++k) h[i][k] = as_stored<T>(x[i].at(k) + r[i].at(k));
            P::store(a.h, base + V * (t + i * per), n - V * (t + i * per), h[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < S; ++i) {
            w[i].load(a.w, V * (t + i * per), n - V * (t + i * per));
#pragma unroll
            for (int k = 0; k < V; ++k) h[i][k] = x[i].at(k);
        }
    }
    auto squares = [&](float f) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) ss += (f * h[i][k]) * (f * h[i][k]);
        return WIDE ? block_sum(ss, red) : wave_sum(ss);
    };
    const float rs = rstd_of(squares, (float)n, a.eps);
    if (t == 0 && a.rstd) a.rstd[row] = rs;
    float top[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int c = V * (t + i * per);
        top[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            h[i][k] = h[i][k] * rs * (w[i].at(k) + a.wadd);
            top[i] = larger(top[i], fabsf(h[i][k]));
        }
        if (a.y) Piece<uint16_t, V, LOOSE>::store(a.y, base + c, n - c, h[i]);
    }
    if (!a.codes) return;
    const int group = (int)a.group;
    if constexpr (V == 1) {
        float q[S];  // the columns' quantisers
        const int ngroups = (int)a.ngroups;
        for (int i = t; i < ngroups; i += per) gathered[i] = 0;
        __syncthreads();
        // a wave's 64 columns lie in at most two groups where those are wider, and the wave takes their maxima first; of
        // narrower ones a lane its own
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int c = t + i * per, g = (int)__umulhi((uint32_t)c, magic);
            if (group > 64) {
                const int g0 = __builtin_amdgcn_readfirstlane(g);
                const float m0 = wave_max(g == g0 ? top[i] : 0.0f), m1 = wave_max(g == g0 ? 0.0f : top[i]);
                if ((t & 63) == 0 && c < n) {
                    atomicMax(&gathered[g0], __builtin_bit_cast(uint32_t, m0));
                    if (g0 + 1 < ngroups) atomicMax(&gathered[g0 + 1], __builtin_bit_cast(uint32_t, m1));
                }
            } else if (c < n) {
                atomicMax(&gathered[g], __builtin_bit_cast(uint32_t, top[i]));
            }
        }
        __syncthreads();
        for (int i = t; i < ngroups; i += per) {
            const Quant g(__builtin_bit_cast(float, gathered[i]));
            a.scale[row * ngroups + i] = g.scale;
            gathered[i] = __builtin_bit_cast(uint32_t, g.packed());
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int c = t + i * per;
            q[i] = __builtin_bit_cast(float, gathered[__umulhi((uint32_t)(c < n ? c : 0), magic)]);
        }
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int c = t + i * per;
            if (c < n) a.codes[base + c] = (int8_t)Quant::code_of(h[i][0], q[i]);
        }
        return;
    }
    if (lg == kWhole) {
#pragma unroll
        for (int i = 1; i < S; ++i) top[0] = larger(top[0], top[i]);
        top[0] = WIDE ? block_max(top[0], red) : wave_max(top[0]);
#pragma unroll
        for (int i = 1; i < S; ++i) top[i] = top[0];
    } else if (WIDE && lg == kGathered) {
        for (int i = t; i < (int)a.ngroups; i += per) gathered[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int c = V * (t + i * per);
            if (c < n) atomicMax(&gathered[__umulhi((uint32_t)c, magic)], __builtin_bit_cast(uint32_t, top[i]));
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int c = V * (t + i * per);
            if (c < n) top[i] = __builtin_bit_cast(float, gathered[__umulhi((uint32_t)c, magic)]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < S; ++i) top[i] = lanes_max(top[i], lg);
    }
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int c = V * (t + i * per);
        if (c >= n) continue;
        const Quant q(top[i]);
        uint32_t b[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < V; ++k) b[(k >> 2) & 1] |= (uint32_t)(q.code(h[i][k]) & 255) << (8 * (k & 3));
        if constexpr (!LOOSE) {
            *reinterpret_cast<uint2*>(a.codes + base + c) = make_uint2(b[0], b[1]);
        } else if (n - c >= V) {
            *reinterpret_cast<Words<2>*>(a.codes + base + c) = {{b[0], b[1]}};
        } else {
#pragma unroll
            for (int k = 0; k < V - 1; ++k)
                if (k < n - c) a.codes[base + c + k] = (int8_t)(b[k >> 2] >> (8 * (k & 3)));
        }
        const int g = lg == kWhole ? 0 : lg == kGathered ? (int)__umulhi((uint32_t)c, magic) : c >> (lg + 3);
        if (c == g * group) a.scale[row * a.ngroups + g] = q.scale;
    }
}

// The adjoint: a wave or workgroup walks rows and keeps its columns' sums of dw in registers. 4096 x 5120 f32, three
// cotangents or fewer: 82 us for 420 MB (5.1 TB/s).
template <class T, int S, bool WIDE, int V, bool LOOSE>
__global__ __launch_bounds__(WIDE ? 1024 : 256) void norm_rows_bwd_kernel(NArgs a, int lg, uint32_t magic) {
    __shared__ float red[kMostWaves];
    __shared__ float sums[WIDE ? 1 : 4 * 64 * V * S];
    const int wave = threadIdx.x >> 6, t = WIDE ? threadIdx.x : threadIdx.x & 63, per = WIDE ? blockDim.x : 64;
    const int n = (int)a.n;
    const int64_t first = WIDE ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave, step = WIDE ? gridDim.x : (int64_t)gridDim.x * 4;
    float dw[S][V] = {};
    for (int64_t row = first; row < a.rows; row += step) {
        const int64_t base = row * n;
        const float rs = a.rstd[row];
        using P = Piece<T, V, LOOSE>;
        P xs[S], ys[S], cs[S], hs[S], w[S];
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int c = V * (t + i * per);
            xs[i].load(a.x, base + c, n - c);
            ys[i].load(a.gy, base + c, a.gy ? n - c : 0);
            cs[i].load(a.gc, base + c, a.gc ? n - c : 0);
            hs[i].load(a.gh, base + c, a.gh ? n - c : 0);
            w[i].load(a.w, c, n - c);
        }
        float x[S][V], e[S][V];
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int c = V * (t + i * per);
#pragma unroll
            for (int k = 0; k < V; ++k) e[i][k] = ys[i].at(k);
            if (a.gc && c < n) {
                const Cotangent q(a.scale[row * a.ngroups + (lg == kWhole ? 0 : lg >= 0 ? c >> (lg + 3) : (int)__umulhi((uint32_t)c, magic))]);
#pragma unroll
                for (int k = 0; k < V; ++k) e[i][k] = q.sum(cs[i].at(k), e[i][k]);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                x[i][k] = xs[i].at(k) * rs;
                dw[i][k] += e[i][k] * x[i][k];
                e[i][k] *= w[i].at(k) + a.wadd;
                dot += e[i][k] * x[i][k];
            }
        }
        const float mean = (WIDE ? block_sum(dot, red) : wave_sum(dot)) / (float)n;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int c = V * (t + i * per);
            float d[V];
#pragma unroll
            for (int k = 0; k < V; ++k) d[k] = hs[i].at(k) + rs * (e[i][k] - x[i][k] * mean);
            P::store(a.dx, base + c, n - c, d);
        }
    }
    if (!a.part) return;
    float* part = a.part + (int64_t)blockIdx.x * n;
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int c = V * (t + i * per);
            Piece<float, V, LOOSE>::store(part, c, n - c, dw[i]);
        }
    } else {
        constexpr int W = 64 * V * S;
#pragma unroll
        for (int i = 0; i < S; ++i) Piece<float, V, false>::store(sums, wave * W + i * 64 * V + V * t, V, dw[i]);
        __syncthreads();
        for (int c = threadIdx.x; c < n; c += 256) part[c] = (sums[c] + sums[W + c]) + (sums[2 * W + c] + sums[3 * W + c]);
    }
}

// ---------------------------------------------------------------- dw from the workgroups' partial sums
// 32 columns a workgroup, of `cols` of a row's n; each of its 32 half waves adds every 32nd of the partial rows, their sums are
// added in order. 512 partial rows of 5120 columns: 4.7 us, latency.
__global__ __launch_bounds__(1024) void norm_dw_kernel(const float* __restrict__ part, int64_t parts, int64_t n, int64_t cols,
                                                       float* __restrict__ dw, int32_t add) {
    __shared__ float sum[32][32];
    const int col = threadIdx.x & 31, half = threadIdx.x >> 5;
    const int64_t j = (int64_t)blockIdx.x * 32 + col;
    float s = 0.0f;
    if (j < cols) {
#pragma unroll 8
        for (int64_t p = half; p < parts; p += 32) s += part[p * n + j];
    }
    sum[half][col] = s;
    __syncthreads();
    if (half == 0 && j < cols) {
        float t = sum[0][col];
#pragma unroll
        for (int i = 1; i < 32; ++i) t += sum[i][col];
        dw[j] = add ? dw[j] + t : t;
    }
}

// how the rows are taken: pieces a thread (0: the general kernels) of `columns` each, threads of a workgroup, and how
// the groups' maxima are found (gathers: in LDS, by a workgroup a row)
struct Rows {
    int pieces, columns, threads, lg;
    bool wide, loose;
};
Rows rows_plan(int64_t n, int64_t group, bool gathers, std::initializer_list<const void*> tensors) {
    Rows r = {};
    if (n <= 16384 && (group >= n || group % 8 == 0)) {
        r.loose = n % 8 != 0;
        for (const void* p : tensors) r.loose = r.loose || !lanes::aligned16(p);
        r.lg = group >= n ? kWhole : lanes::group_log(group) >= 0 ? lanes::group_log(group) - 3 : kGathered;
        r.columns = 8;
        r.wide = n > 2048 || (gathers && r.lg == kGathered);
        r.pieces = r.wide ? 2 : (int)((n + 511) / 512);
        r.threads = r.wide ? 64 * (int)((n + 1023) / 1024) : 256;
    } else if (n <= 8192 && group > 1) {
        r.lg = kGathered;
        r.columns = 1;
        r.wide = true;
        r.pieces = n <= 2048 ? 4 : 8;
        r.threads = 64 * (int)((n + 64 * r.pieces - 1) / (64 * r.pieces));
    }
    return r;
}
// a column's group is its product with this, over 2^32: exact for columns and groups below 2^14. (One group: not used.)
uint32_t group_magic(int64_t group) { return group > 1 && group < (1 << 14) ? (uint32_t)((1ULL << 32) / (uint64_t)group + 1) : 0; }
// f(a kernel's pieces, whether the row is a workgroup's, a piece's columns, whether pieces lie anywhere)
template <class F>
void with_rows(const Rows& r, F&& f) {
    using std::integral_constant;
    const integral_constant<int, 8> eight;
    const integral_constant<int, 1> one;
    auto of_eight = [&](auto loose) {
        if (r.wide) return f(integral_constant<int, 2>{}, std::true_type{}, eight, loose);
        if (r.pieces == 1) return f(one, std::false_type{}, eight, loose);
        if (r.pieces == 2) return f(integral_constant<int, 2>{}, std::false_type{}, eight, loose);
        if (r.pieces == 3) return f(integral_constant<int, 3>{}, std::false_type{}, eight, loose);
        return f(integral_constant<int, 4>{}, std::false_type{}, eight, loose);
    };
    if (r.columns == 1) return r.pieces == 4 ? f(integral_constant<int, 4>{}, std::true_type{}, one, std::false_type{}) : f(eight, std::true_type{}, one, std::false_type{});
    return r.loose ? of_eight(std::true_type{}) : of_eight(std::false_type{});
}

// workgroups of `threads` in a launch: its threads stay below 2^32
constexpr int64_t most_groups(int threads) { return 0xFFFFFFFFLL / threads; }
// f(the arguments of some rows) until all have had theirs, at most `most` of them at a time, a multiple of 16: later rows then
// lie on 16 bytes where the first does
template <class F>
void rows_in_turn(NArgs a, int64_t most, int size, F&& f) {
    const int64_t rows = a.rows;
    auto past = [](auto*& p, int64_t bytes) {
        if (p) p = (std::remove_reference_t<decltype(p)>)(reinterpret_cast<uintptr_t>(p) + bytes);
    };
    most -= most % 16;
    for (int64_t done = 0;;) {
        a.rows = rows - done < most ? rows - done : most;
        f(a);
        done += a.rows;
        if (done == rows) return;
        const int64_t values = a.rows * a.n;
        past(a.x, values * size);
        past(a.res, values * size);
        past(a.h, values * size);
        past(a.codes, values);
        past(a.y, 2 * values);
        past(a.scale, 4 * a.rows * a.ngroups);
        past(a.rstd, 4 * a.rows);
    }
}

int64_t bwd_parts(int64_t rows) { return rows < 512 ? rows : 512; }

int refuse(const char* who, int code, const char* why) {
    set_error("%s: %s", who, why);
    return code;
}

int check(const char* who, const void* x, const void* w, int32_t dtype, int64_t rows, int64_t n) {
    if (dtype != R97Q_BF16 && dtype != R97Q_F32) return refuse(who, R97Q_EINVAL, "the stream is bf16 or f32");
    if (rows < 0 || n < 1) return refuse(who, R97Q_EINVAL, "rows >= 0 and n >= 1");
    if (rows > 0x7FFFFFFF || n > 0x7FFFFFFF) return refuse(who, R97Q_EUNSUPPORTED, "rows and n within 31 bits");
    if ((!x && rows > 0) || !w) return refuse(who, R97Q_EINVAL, "null activation or gain");
    return R97Q_OK;
}

}  // namespace
}  // namespace r97q

using namespace r97q;

extern "C" {

int r97q_add_rmsnorm_i8g(const void* x, const void* residual, const void* w, int32_t dtype, int64_t rows, int64_t n,
                         int64_t group, float eps, float wadd, void* h_out, int8_t* codes, float* scale,
                         uint16_t* y_out, float* rstd, R97IqrStream stream) {
    clear_error();
    const char* who = "r97q_add_rmsnorm_i8g";
    if (int e = check(who, x, w, dtype, rows, n)) return e;
    if (!codes != !scale) return refuse(who, R97Q_EINVAL, "codes and scale come together");
    if (rows > 0 && residual && !h_out) return refuse(who, R97Q_EINVAL, "a residual needs h_out");
    if (!residual && h_out) return refuse(who, R97Q_EINVAL, "without a residual h is x: h_out is null");
    if (rows == 0) return R97Q_OK;
    if (!codes && !y_out && !residual && !rstd) return refuse(who, R97Q_EINVAL, "no output");
    NArgs a = {};
    a.x = x;
    a.res = residual;
    a.w = w;
    a.rows = rows;
    a.n = n;
    a.group = group <= 0 || group > n ? n : group;
    a.ngroups = (n + a.group - 1) / a.group;
    a.eps = eps;
    a.wadd = wadd;
    a.h = h_out;
    a.codes = codes;
    a.scale = scale;
    a.y = y_out;
    a.rstd = rstd;
    const Rows r = rows_plan(n, a.group, codes, {x, residual, w, h_out, codes, y_out});
    const int size = dtype == R97Q_BF16 ? 2 : 4;
    if (r.pieces) {
        with_rows(r, [&](auto pieces, auto wide, auto columns, auto loose) {
            const uint32_t magic = group_magic(a.group);
            const unsigned lds = r.lg == kGathered ? (unsigned)(4 * a.ngroups) : 0;
            const int each = wide ? 1 : 4;  // rows a workgroup
            rows_in_turn(a, each * most_groups(r.threads), size, [&](const NArgs& b) {
                const dim3 grid((unsigned)((b.rows + each - 1) / each)), threads(r.threads);
                if (dtype == R97Q_BF16)
                    hipLaunchKernelGGL((norm_rows_kernel<uint16_t, pieces, wide, columns, loose>), grid, threads, lds, (hipStream_t)stream, b, r.lg, magic);
                else
                    hipLaunchKernelGGL((norm_rows_kernel<float, pieces, wide, columns, loose>), grid, threads, lds, (hipStream_t)stream, b, r.lg, magic);
            });
        });
        return launch_status("norm_rows_kernel");
    }
    rows_in_turn(a, most_groups(kThreads), size, [&](const NArgs& b) {
        if (dtype == R97Q_BF16)
            hipLaunchKernelGGL(norm_any_kernel<uint16_t>, dim3((unsigned)b.rows), dim3(kThreads), 0, (hipStream_t)stream, b);
        else
            hipLaunchKernelGGL(norm_any_kernel<float>, dim3((unsigned)b.rows), dim3(kThreads), 0, (hipStream_t)stream, b);
    });
    return launch_status("norm_any_kernel");
}

int64_t r97q_add_rmsnorm_i8g_bwd_workspace_bytes(int64_t rows, int64_t n) {
    if (rows < 0 || n < 1 || rows > 0x7FFFFFFF || n > 0x7FFFFFFF) return -1;
    return 4 * bwd_parts(rows) * n;
}

int r97q_add_rmsnorm_i8g_bwd(const void* h, const void* w, int32_t dtype, int64_t rows, int64_t n, int64_t group,
                             float wadd, const float* rstd, const float* scale, const void* g_codes,
                             const void* g_y, const void* g_h, void* dx, float* dw, int32_t dw_accumulate,
                             void* workspace, int64_t workspace_bytes, R97IqrStream stream) {
    clear_error();
    const char* who = "r97q_add_rmsnorm_i8g_bwd";
    if (int e = check(who, h, w, dtype, rows, n)) return e;
    if (rows > 0 && (!rstd || !dx)) return refuse(who, R97Q_EINVAL, "null rstd or dx");
    if (rows > 0 && g_codes && !scale) return refuse(who, R97Q_EINVAL, "the codes' cotangent needs the forward's scale");
    if (dw && rows > 0 && (!workspace || workspace_bytes < r97q_add_rmsnorm_i8g_bwd_workspace_bytes(rows, n)))
        return refuse(who, R97Q_EWORKSPACE, "the workspace is too small");
    hipStream_t st = (hipStream_t)stream;
    NArgs a = {};
    a.x = h;
    a.w = w;
    a.rows = rows;
    a.n = n;
    a.group = group <= 0 || group > n ? n : group;
    a.ngroups = (n + a.group - 1) / a.group;
    a.wadd = wadd;
    a.rstd = const_cast<float*>(rstd);
    a.scale = const_cast<float*>(scale);
    a.gc = g_codes;
    a.gy = g_y;
    a.gh = g_h;
    a.dx = dx;
    a.part = dw ? static_cast<float*>(workspace) : nullptr;
    int64_t parts = bwd_parts(rows);
    const Rows r = rows_plan(n, a.group, false, {h, w, g_codes, g_y, g_h, dx, a.part});
    if (rows > 0 && r.pieces) {
        // four rows at a time a workgroup where a row is a wave's
        int64_t most = r.wide ? rows : (rows + 3) / 4;
        if (most > most_groups(r.threads)) most = most_groups(r.threads);
        if (parts > most) parts = most;
        with_rows(r, [&](auto pieces, auto wide, auto columns, auto loose) {
            const dim3 grid((unsigned)(dw ? parts : most)), threads(r.threads);
            const uint32_t magic = group_magic(a.group);
            if (dtype == R97Q_BF16)
                hipLaunchKernelGGL((norm_rows_bwd_kernel<uint16_t, pieces, wide, columns, loose>), grid, threads, 0, st, a, r.lg, magic);
            else
                hipLaunchKernelGGL((norm_rows_bwd_kernel<float, pieces, wide, columns, loose>), grid, threads, 0, st, a, r.lg, magic);
        });
        if (int e = launch_status("norm_rows_bwd_kernel")) return e;
    } else if (rows > 0) {
        const dim3 grid((unsigned)(dw ? parts : rows < most_groups(kThreads) ? rows : most_groups(kThreads)));
        if (dtype == R97Q_BF16)
            hipLaunchKernelGGL(norm_any_bwd_kernel<uint16_t>, grid, dim3(kThreads), 0, st, a);
        else
            hipLaunchKernelGGL(norm_any_bwd_kernel<float>, grid, dim3(kThreads), 0, st, a);
        if (int e = launch_status("norm_any_bwd_kernel")) return e;
    }
    if (!dw) return R97Q_OK;
    for (int64_t c = 0, most = 32 * most_groups(1024); c < n; c += most) {
        const int64_t cols = n - c < most ? n - c : most;
        hipLaunchKernelGGL(norm_dw_kernel, dim3((unsigned)((cols + 31) / 32)), dim3(1024), 0, st, a.part + c, parts, n, cols, dw + c, dw_accumulate);
    }
    return launch_status("norm_dw_kernel");
}

}  // extern "C"
