// attn_fwd.hip -- attention's forward: O = softmax(scale Q K^T + mask) V and each row's log-sum-exp.
//
// One pass over the keys with a running maximum and sum (in f32), per row:
//   m' = max(m, max_j s_j),  l' = l e^(m - m') + sum_j e^(s_j - m'),  O' = O e^(m - m') + sum_j e^(s_j - m') v_j
// and O / l, m + ln l at the end. The probabilities are rounded to bf16 for the second product (the
// matrix cores' input type; relative 2^-9 at most, as the output's own rounding), their sum is of the
// unrounded values in f32.
#include "attn.h"
#include "status.h"

namespace r97q {
namespace attn {
namespace {

// The running maximum is taken of the raw products, so the scale has to be positive: a negative one flips
// the queries' signs instead, and with a scale of zero the queries are zeros. In base 2 for the exponentials.
__device__ __forceinline__ float score_scale(const Args& a) { return a.scale == 0.0f ? kLog2e : fabsf(a.scale) * kLog2e; }
template <int D>
__device__ __forceinline__ void turn_sign(const Args& a, bf16x8 (&q)[D / 16]) {
    if (a.scale > 0.0f) return;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u, keep = a.scale < 0.0f ? ~0u : 0u;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
        u32x4 w = __builtin_bit_cast(u32x4, q[c]);
        q[c] = as_bf16x8((w & keep) ^ flip);
    }
}

// ---------------------------------------------------------------- tiles of 128 rows
// A workgroup's 4 waves take 32 rows each of one key head's rows and walk the keys together, KT at a
// time, from LDS.
template <int D, int KT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attn_fwd_kernel(Args a) {
    using T = Tile<D>;
    __shared__ __attribute__((aligned(16))) uint8_t kt[2][KT * T::RB];
    __shared__ __attribute__((aligned(16))) uint8_t vt[2][KT * T::RB];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, h = lane >> 5;
    const int hk = blockIdx.y;
    const Seq s = sequence(a, blockIdx.z);
    const int64_t rows = s.lq * a.g;
    const float sl = score_scale(a);
    const uint8_t* kb = kv_at(a.k, a, s, hk);
    const uint8_t* vb = kv_at(a.v, a, s, hk);
    for (int64_t tile = gridDim.x - 1 - blockIdx.x; tile * 128 < rows; tile += gridDim.x) {
        const int64_t r0 = tile * 128 + 32 * wave;
        const int64_t r = r0 + col, rr = r < rows ? r : rows - 1;
        const int64_t tok = rr / a.g;
        const int head = hk * a.g + (int)(rr % a.g);
        bf16x8 q[D / 16];
        load_row<D>(q_at(a.q, a, s, head) + 2 * tok * a.q.ts, r < rows, a.d, lane, q);
        turn_sign<D>(a, q);
        int64_t lo, hi, wlo, whi;
        const int64_t end = tile * 128 + 127 < rows ? tile * 128 + 127 : rows - 1;
        key_range(a, s, tile * 128 / a.g, end / a.g, lo, hi);
        lo = lo / KT * KT;
        // the wave's own rows: what its first and last token see
        const int64_t t0 = (r0 < rows ? r0 : rows - 1) / a.g, t1 = (r0 + 31 < rows ? r0 + 31 : rows - 1) / a.g;
        key_range(a, s, t0, t1, wlo, whi);
        const int64_t all_lo = a.window ? t1 + s.off - a.window + 1 : 0;                     // every row sees from here
        const int64_t all_hi = a.causal ? clamp64(t0 + s.off + 1, 0, s.lk) : s.lk;            // to here
        f32x16 o[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] = (f32x16){};
        float m = -INFINITY, l = 0.0f;
        if (lo < hi) {
            Stage<D, KT, 256> ks, vs;
            ks.load(kb, 2 * a.k.ts, lo, s.lk - 1, a.d, tid);
            vs.load(vb, 2 * a.v.ts, lo, s.lk - 1, a.d, tid);
            ks.store(kt[0], tid);
            vs.store(vt[0], tid);
            __syncthreads();
            int buf = 0;
            for (int64_t j0 = lo; j0 < hi; j0 += KT, buf ^= 1) {
                const bool more = j0 + KT < hi;
                if (more) {
                    ks.load(kb, 2 * a.k.ts, j0 + KT, s.lk - 1, a.d, tid);
                    vs.load(vb, 2 * a.v.ts, j0 + KT, s.lk - 1, a.d, tid);
                }
                if (j0 < whi && j0 + KT > wlo) {
                    f32x16 x[KT / 32];
#pragma unroll
                    for (int i = 0; i < KT / 32; ++i) {
                        x[i] = (f32x16){};
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) x[i] = mfma(T::rows(kt[buf], 32 * i, c, lane), q[c], x[i]);
                    }
                    if (j0 < all_lo || j0 + KT > all_hi) {
                        // positions relative to the tile fit 32 bits once clamped
                        const int top = (int)clamp64((a.causal ? tok + s.off : s.lk - 1) - j0, -1, KT);
                        const int cap = (int)clamp64(s.lk - 1 - j0, -1, KT);
                        const int last = top < cap ? top : cap;
                        const int first = a.window ? (int)clamp64(tok + s.off - a.window + 1 - j0, 0, KT) : 0;
#pragma unroll
                        for (int i = 0; i < KT / 32; ++i)
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const int j = 32 * i + 8 * (e >> 2) + 4 * h + (e & 3);
                                x[i][e] = j <= last && j >= first ? x[i][e] : -INFINITY;
                            }
                    }
                    float top = x[0][0];
#pragma unroll
                    for (int i = 0; i < KT / 32; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) top = fmaxf(top, x[i][e]);
                    top = pair_max(top) * sl;
                    const float m1 = fmaxf(m, top);
                    const float base = m1 == -INFINITY ? 0.0f : m1;
                    const float turn = __builtin_amdgcn_exp2f(m - base);
                    m = m1;
                    float sum = 0.0f;
                    bf16x8 p[KT / 16];
#pragma unroll
                    for (int i = 0; i < KT / 32; ++i) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            x[i][e] = __builtin_amdgcn_exp2f(x[i][e] * sl - base);
                            sum += x[i][e];
                        }
                        bf16x8 two[2];
                        pack_tile(x[i], two);
                        p[2 * i] = two[0];
                        p[2 * i + 1] = two[1];
                    }
                    l = l * turn + sum;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[i][e] *= turn;
#pragma unroll
                    for (int c = 0; c < KT / 16; ++c)
#pragma unroll
                        for (int i = 0; i < D / 32; ++i) o[i] = mfma(T::cols(vt[buf], 16 * c, i, lane), p[c], o[i]);
                }
                if (more) {
                    ks.store(kt[buf ^ 1], tid);
                    vs.store(vt[buf ^ 1], tid);
                }
                __syncthreads();
            }
        }
        l = pair_sum(l);
        if (r < rows) {
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            uint8_t* out = q_at(a.o, a, s, head) + (a.o.f32 ? 4 : 2) * tok * a.o.ts;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d0 = 32 * i + 8 * e + 4 * h;
                    if (d0 < a.d)
                        store4(out, a.o.f32, d0, o[i][4 * e] * inv, o[i][4 * e + 1] * inv, o[i][4 * e + 2] * inv, o[i][4 * e + 3] * inv);
                }
            if (a.lse && h == 0) a.lse[stat_at(a, s, head, tok)] = l > 0.0f ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
        }
        __syncthreads();
    }
}

}  // namespace

int launch_fwd(const Args& a, hipStream_t st) {
    const int64_t tiles = (a.lq * a.g + 127) / 128;
    const dim3 grid((unsigned)(tiles < 65535 ? tiles : 65535), a.hk, a.batch);
    if (a.d <= 64)
        hipLaunchKernelGGL((attn_fwd_kernel<64, 64>), grid, dim3(256), 0, st, a);
    else if (a.d <= 128)
        hipLaunchKernelGGL((attn_fwd_kernel<128, 64>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((attn_fwd_kernel<256, 32>), grid, dim3(256), 0, st, a);
    return launch_status("attn_fwd_kernel");
}

}  // namespace attn
}  // namespace r97q
