// paged.hip -- new tokens' keys and values into a paged cache.
//
// Token i of a sequence's n new ones takes position m - n + i of its m: slot (position mod page size) of the page that the
// sequence's row of the table names. Bound by memory, each value read and written once; a workgroup walks a sequence's tokens
// in pieces of 8 values, kItems of a thread's loads out together. A token without a place (before the sequence, past the
// table, a page outside the pool) is left out: m is the length as it is given, not what the table has room for, so the
// tokens of a sequence that has outgrown its table write over none that the cache holds. 16384 tokens of 8 heads of 128 into
// pages of 64 or 16: 25 us, 5.3 TB/s (a 1 GiB copy reaches 5.0; part of these tensors stays in the cache); 2048 10 us, one
// each of 16 sequences 9, the call's latency.
#include "attn.h"
#include "status.h"

namespace r97q {
namespace attn {
namespace {

constexpr int kThreads = 256, kItems = 4;

template <bool F32>
__global__ __launch_bounds__(kThreads) void paged_write_kernel(Args a, Heads k, Heads v) {
    const Seq s = sequence(a, blockIdx.y);
    const int per = a.d / 8, all = 2 * a.hk * per;  // pieces of a head, and of a token's keys and values
    const int64_t n = (int64_t)s.lq * all, step = (int64_t)gridDim.x * kThreads;
    const int32_t* table = a.table + s.b * a.table_stride;
    const int64_t off = (int64_t)uniform(a.kv_lens[s.b]) - s.lq;
    const uint8_t *kb = q_at(k, a, s, 0), *vb = q_at(v, a, s, 0);
    for (int64_t i0 = (int64_t)blockIdx.x * kThreads + threadIdx.x; i0 < n; i0 += kItems * step) {
        u32x4 w[kItems];
        uint8_t* to[kItems];
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
            const int64_t i = i0 + j * step < n ? i0 + j * step : i0;
            const int tok = n < 1LL << 31 ? (int)((uint32_t)i / (uint32_t)all) : (int)(i / all);
            const int rest = (int)(i - (int64_t)tok * all), head = rest / per, e = 8 * (rest - head * per);
            const bool keys = head < a.hk;
            const int h = keys ? head : head - a.hk;
            const int64_t at = tok * (keys ? k.ts : v.ts) + h * (keys ? k.hs : v.hs) + e;
            if constexpr (F32) {
                const float4* x = reinterpret_cast<const float4*>((keys ? kb : vb) + 4 * at);
                const float4 lo = x[0], hi = x[1];
                w[j] = (u32x4){pack_bf16(lo.x, lo.y), pack_bf16(lo.z, lo.w), pack_bf16(hi.x, hi.y), pack_bf16(hi.z, hi.w)};
            } else {
                w[j] = *reinterpret_cast<const u32x4*>((keys ? kb : vb) + 2 * at);
            }
            const int64_t pos = tok + off;
            const bool in = pos >= 0 && pos >> a.page_shift < a.max_pages && i0 + j * step < n;
            const int page = in ? table[pos >> a.page_shift] : -1;
            to[j] = (uint32_t)page < (uint32_t)a.pages
                        ? (keys ? a.k.data : a.v.data) + 2 * (page * (keys ? a.k.bs : a.v.bs) + h * (keys ? a.k.hs : a.v.hs) + e +
                                                              (pos & ((1 << a.page_shift) - 1)) * (keys ? a.k.ts : a.v.ts))
                        : nullptr;
        }
#pragma unroll
        for (int j = 0; j < kItems; ++j)
            if (to[j]) *reinterpret_cast<u32x4*>(to[j]) = w[j];
    }
}

}  // namespace

int launch_write(const Args& a, const Heads& k, const Heads& v, hipStream_t st) {
    // a round of the longest sequence's pieces, some 4096 workgroups in all at most; the kernel's loop takes what is left
    const int64_t pieces = (int64_t)a.lq * 2 * a.hk * (a.d / 8);
    int64_t blocks = (pieces + kThreads * kItems - 1) / (kThreads * kItems);
    if (pieces < 64 * kThreads * kItems) blocks = (pieces + kThreads - 1) / kThreads;  // few: a piece a thread
    const int64_t most = a.batch < 4096 ? 4096 / a.batch : 1;
    if (blocks > most) blocks = most;
    const dim3 grid((unsigned)(blocks < 1 ? 1 : blocks), (unsigned)a.batch);
    if (k.f32)
        hipLaunchKernelGGL(paged_write_kernel<true>, grid, dim3(kThreads), 0, st, a, k, v);
    else
        hipLaunchKernelGGL(paged_write_kernel<false>, grid, dim3(kThreads), 0, st, a, k, v);
    return launch_status("paged_write_kernel");
}

}  // namespace attn
}  // namespace r97q
