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
// wave, four of them to a workgroup, with no barrier; wider ones to a workgroup. Rows past 8192 columns, odd
// widths, groups that do not fall on lanes and unaligned tensors take the general kernels, which read a
// row again for each stage.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/r97q.h"
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
        static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
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

__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
// over the workgroup, the waves' values in wave order
__device__ float block_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = red[0];
    for (int i = 1; i < kWaves; ++i) t += red[i];
    return t;
}
__device__ float block_max(float v, float* red) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = red[0];
    for (int i = 1; i < kWaves; ++i) t = fmaxf(t, red[i]);
    return t;
}

// The quantiser of a group with maximum amax: code = rint(y * up * inv). up keeps 127 / amax finite where the
// group's values are tiny.
struct Quant {
    float scale, up, inv;
    __device__ __forceinline__ explicit Quant(float amax) {
        scale = amax > 0.0f ? amax / 127.0f : 1.0f;
        up = amax < 0x1p-96f ? 0x1p96f : 1.0f;
        inv = amax > 0.0f ? 127.0f / (amax * up) : 0.0f;
    }
    __device__ __forceinline__ int code(float y) const { return (int)rintf(y * up * inv); }
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
// grid (rows). x may be h_out: a value is overwritten by the wave that was the last to read it.
template <class T>
__global__ __launch_bounds__(kThreads) void norm_any_kernel(NArgs a) {
    __shared__ float red[kWaves];
    const int64_t base = (int64_t)blockIdx.x * a.n;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto h_of = [&](int64_t j) {
        return a.res ? as_stored<T>(ld<T>(a.x, base + j) + ld<T>(a.res, base + j)) : ld<T>(a.x, base + j);
    };
    float ss = 0.0f;
    for (int64_t j = threadIdx.x; j < a.n; j += kThreads) {
        const float h = h_of(j);
        ss += h * h;
    }
    const float rs = 1.0f / sqrtf(block_sum(ss, red) / (float)a.n + a.eps);
    if (threadIdx.x == 0 && a.rstd) a.rstd[blockIdx.x] = rs;
    auto y_of = [&](int64_t j) { return h_of(j) * rs * (ld<T>(a.w, j) + a.wadd); };
    // one group: the workgroup's; more: a wave takes whole groups
    const bool one = a.ngroups == 1;
    const int first = one ? (int)threadIdx.x : lane, step = one ? kThreads : 64;
    for (int64_t g = one ? 0 : wave; g < a.ngroups; g += one ? 1 : kWaves) {
        const int64_t j0 = g * a.group, j1 = j0 + a.group < a.n ? j0 + a.group : a.n;
        float amax = 0.0f;
        for (int64_t j = j0 + first; j < j1; j += step) amax = fmaxf(amax, fabsf(y_of(j)));
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

// ---------------------------------------------------------------- dw from the workgroups' partial sums
// 64 columns a workgroup; each of its 16 waves adds every 16th of the partial rows, the waves' sums are
// added in order.
__global__ __launch_bounds__(1024) void norm_dw_kernel(const float* __restrict__ part, int64_t parts, int64_t n,
                                                       float* __restrict__ dw, int32_t add) {
    __shared__ float sum[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t j = (int64_t)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (j < n) {
#pragma unroll 8
        for (int64_t p = wave; p < parts; p += 16) s += part[p * n + j];
    }
    sum[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && j < n) {
        float t = sum[0][lane];
#pragma unroll
        for (int i = 1; i < 16; ++i) t += sum[i][lane];
        dw[j] = add ? dw[j] + t : t;
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
    if (dtype == R97Q_BF16)
        hipLaunchKernelGGL(norm_any_kernel<uint16_t>, dim3((unsigned)rows), dim3(kThreads), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(norm_any_kernel<float>, dim3((unsigned)rows), dim3(kThreads), 0, (hipStream_t)stream, a);
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
    const int64_t parts = bwd_parts(rows);
    if (rows > 0) {
        const dim3 grid((unsigned)(dw ? parts : rows));
        if (dtype == R97Q_BF16)
            hipLaunchKernelGGL(norm_any_bwd_kernel<uint16_t>, grid, dim3(kThreads), 0, st, a);
        else
            hipLaunchKernelGGL(norm_any_bwd_kernel<float>, grid, dim3(kThreads), 0, st, a);
        if (int e = launch_status("norm_any_bwd_kernel")) return e;
    }
    if (!dw) return R97Q_OK;
    hipLaunchKernelGGL(norm_dw_kernel, dim3((unsigned)((n + 63) / 64)), dim3(1024), 0, st, a.part, parts, n, dw, dw_accumulate);
    return launch_status("norm_dw_kernel");
}

}  // extern "C"
