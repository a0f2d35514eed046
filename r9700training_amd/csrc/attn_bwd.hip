// attn_bwd.hip -- attention's backward pass, the probabilities recomputed from the log-sum-exp L:
//   P = exp(scale Q K^T - L)    D_i = sum_d dO_id O_id    dS = P o (dO V^T - D)
//   dV = P^T dO    dQ = scale dS K    dK = scale dS^T Q,  dK and dV summed over the heads that share a key head.
//
// Two launches: attn_dq_kernel walks the keys for tiles of rows (and writes D), attn_dkdv_kernel walks the
// rows for tiles of keys. Both recompute P and dO V^T: seven products where one launch would need five,
// but every sum has one owner and a fixed order, so repeated calls give the same bits, and no f32 gradient
// passes through memory. P and dS are rounded to bf16 for their products (relative 2^-9 at most, each
// term of a sum on its own), everything else is f32.
#include "attn.h"
#include "status.h"

namespace r97q {
namespace attn {
namespace {

// ---------------------------------------------------------------- dQ (and D): 128 rows a workgroup
template <int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attn_dq_kernel(Args a) {
    using T = Tile<D>;
    constexpr int KT = 32;
    __shared__ __attribute__((aligned(16))) uint8_t kt[2][KT * T::RB];
    __shared__ __attribute__((aligned(16))) uint8_t vt[2][KT * T::RB];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, h = lane >> 5;
    const int hk = blockIdx.y;
    const Seq s = sequence(a, blockIdx.z);
    const int64_t rows = s.lq * a.g;
    const float sl = a.scale * kLog2e;
    const uint8_t* kb = kv_at(a.k, a, s, hk);
    const uint8_t* vb = kv_at(a.v, a, s, hk);
    for (int64_t tile = gridDim.x - 1 - blockIdx.x; tile * 128 < rows; tile += gridDim.x) {
        const int64_t r0 = tile * 128 + 32 * wave;
        const int64_t r = r0 + col, rr = r < rows ? r : rows - 1;
        const int64_t tok = rr / a.g;
        const int head = hk * a.g + (int)(rr % a.g);
        bf16x8 q[D / 16], go[D / 16];
        load_row<D>(q_at(a.q, a, s, head) + 2 * tok * a.q.ts, r < rows, a.d, lane, q);
        load_row<D>(q_at(a.d_o, a, s, head) + 2 * tok * a.d_o.ts, r < rows, a.d, lane, go);
        const uint8_t* op = q_at(a.o, a, s, head) + (a.o.f32 ? 4 : 2) * tok * a.o.ts;
        float delta = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            const int e = 16 * c + 8 * h;
            if (e < a.d) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = a.o.f32 ? reinterpret_cast<const float*>(op)[e + j]
                                            : bf16_to_f32(reinterpret_cast<const uint16_t*>(op)[e + j]);
                    delta += x * (float)go[c][j];
                }
            }
        }
        delta = pair_sum(delta);
        const int64_t at = stat_at(a, s, head, tok);
        if (r < rows && h == 0) a.delta[at] = delta;
        const float lse = a.lse[at];
        const float base = lse == -INFINITY ? 0.0f : lse * kLog2e;
        int64_t lo, hi, wlo, whi;
        const int64_t end = tile * 128 + 127 < rows ? tile * 128 + 127 : rows - 1;
        key_range(a, s, tile * 128 / a.g, end / a.g, lo, hi);
        lo = lo / KT * KT;
        const int64_t t0 = (r0 < rows ? r0 : rows - 1) / a.g, t1 = (r0 + 31 < rows ? r0 + 31 : rows - 1) / a.g;
        key_range(a, s, t0, t1, wlo, whi);
        const int64_t all_lo = a.window ? t1 + s.off - a.window + 1 : 0;
        const int64_t all_hi = a.causal ? clamp64(t0 + s.off + 1, 0, s.lk) : s.lk;
        f32x16 dq[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dq[i] = (f32x16){};
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
                    f32x16 x = {}, y = {};
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) x = mfma(T::rows(kt[buf], 0, c, lane), q[c], x);
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) y = mfma(T::rows(vt[buf], 0, c, lane), go[c], y);
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = __builtin_amdgcn_exp2f(x[e] * sl - base) * (y[e] - delta);
                    if (j0 < all_lo || j0 + KT > all_hi) {
                        const int top = (int)clamp64((a.causal ? tok + s.off : s.lk - 1) - j0, -1, KT);
                        const int cap = (int)clamp64(s.lk - 1 - j0, -1, KT);
                        const int last = top < cap ? top : cap;
                        const int first = a.window ? (int)clamp64(tok + s.off - a.window + 1 - j0, 0, KT) : 0;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int j = 8 * (e >> 2) + 4 * h + (e & 3);
                            x[e] = j <= last && j >= first ? x[e] : 0.0f;
                        }
                    }
                    bf16x8 ds[2];
                    pack_tile(x, ds);
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int i = 0; i < D / 32; ++i) dq[i] = mfma(T::cols(kt[buf], 16 * c, i, lane), ds[c], dq[i]);
                }
                if (more) {
                    ks.store(kt[buf ^ 1], tid);
                    vs.store(vt[buf ^ 1], tid);
                }
                __syncthreads();
            }
        }
        if (r < rows) {
            uint8_t* out = q_at(a.dq, a, s, head) + (a.dq.f32 ? 4 : 2) * tok * a.dq.ts;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d0 = 32 * i + 8 * e + 4 * h;
                    if (d0 < a.d)
                        store4(out, a.dq.f32, d0, dq[i][4 * e] * a.scale, dq[i][4 * e + 1] * a.scale,
                               dq[i][4 * e + 2] * a.scale, dq[i][4 * e + 3] * a.scale);
                }
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- dK, dV: 128 keys a workgroup
// A wave holds 32 keys and their gradients; the workgroup walks the rows that see its keys, 32 at a time.
template <int D>
__global__ __launch_bounds__(256, 1) void attn_dkdv_kernel(Args a) {
    using T = Tile<D>;
    constexpr int RT = 32, N = RT * T::CH / 256;
    __shared__ __attribute__((aligned(16))) uint8_t qt[2][RT * T::RB];
    __shared__ __attribute__((aligned(16))) uint8_t ot[2][RT * T::RB];
    __shared__ __attribute__((aligned(16))) float stat[2][2][RT];  // log-sum-exp (base 2), delta
    __shared__ __attribute__((aligned(16))) int see[2][2][RT];     // first and last key a row sees, from the tile's first
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, h = lane >> 5;
    const int hk = blockIdx.y;
    const Seq s = sequence(a, blockIdx.z);
    const int64_t cover = a.kv_starts ? s.lk : a.lk;  // the dense form's keys past a sequence's length get zeros
    const float sl = a.scale * kLog2e;
    for (int64_t j0 = (int64_t)blockIdx.x * 128; j0 < cover; j0 += (int64_t)gridDim.x * 128) {
        const int64_t j = j0 + 32 * wave + col;
        bf16x8 k[D / 16], v[D / 16];
        const int64_t jj = j < s.lk ? j : 0;
        load_row<D>(kv_at(a.k, a, s, hk) + 2 * jj * a.k.ts, j < s.lk, a.d, lane, k);
        load_row<D>(kv_at(a.v, a, s, hk) + 2 * jj * a.v.ts, j < s.lk, a.d, lane, v);
        // the tokens that see any of the keys j0 .. j1
        const int64_t j1 = j0 + 127 < s.lk ? j0 + 127 : s.lk - 1;
        int64_t t0 = 0, t1 = s.lq;
        if (a.causal) t0 = clamp64(j0 - s.off, 0, s.lq);
        if (a.window) t1 = clamp64(j1 + a.window - s.off, 0, s.lq);
        if (j0 >= s.lk) t1 = t0;
        const int64_t rlo = t0 * a.g, rhi = t1 * a.g;
        f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dk[i] = dv[i] = (f32x16){};
        u32x4 qx[N], ox[N];
        float st = 0.0f;
        int sf = 0, sz = 0;
        // rows [r0, r0 + 32) into registers; rows past the end repeat the last one and see nothing
        auto load = [&](int64_t r0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int p = tid + 256 * i, ch = p % T::CH;
                const int64_t want = r0 + p / T::CH, r = want < rhi ? want : rhi - 1, tok = r / a.g;
                const int head = hk * a.g + (int)(r % a.g), e = 8 * ch < a.d ? 16 * ch : 0;
                qx[i] = *reinterpret_cast<const u32x4*>(q_at(a.q, a, s, head) + 2 * tok * a.q.ts + e);
                ox[i] = *reinterpret_cast<const u32x4*>(q_at(a.d_o, a, s, head) + 2 * tok * a.d_o.ts + e);
            }
            if (tid < 2 * RT) {
                const int64_t want = r0 + (tid & (RT - 1)), r = want < rhi ? want : rhi - 1, tok = r / a.g;
                const int64_t at = stat_at(a, s, hk * a.g + (int)(r % a.g), tok);
                const float x = tid < RT ? a.lse[at] * kLog2e : a.delta[at];
                st = x == -INFINITY ? 0.0f : x;
                const int64_t cap = s.lk - 1, top = a.causal && tok + s.off < cap ? tok + s.off : cap;
                sz = want < rhi ? (int)clamp64(top - j0, -1, 128) : -1;
                sf = a.window ? (int)clamp64(tok + s.off - a.window + 1 - j0, 0, 128) : 0;
            }
        };
        auto put = [&](int buf) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int p = tid + 256 * i;
                *reinterpret_cast<u32x4*>(qt[buf] + T::at(p / T::CH, p % T::CH)) = qx[i];
                *reinterpret_cast<u32x4*>(ot[buf] + T::at(p / T::CH, p % T::CH)) = ox[i];
            }
            if (tid < 2 * RT) {
                stat[buf][tid / RT][tid & (RT - 1)] = st;
                see[buf][tid / RT][tid & (RT - 1)] = tid < RT ? sf : sz;
            }
        };
        if (rlo < rhi) {
            load(rlo);
            put(0);
            __syncthreads();
            int buf = 0;
            for (int64_t r0 = rlo; r0 < rhi; r0 += RT, buf ^= 1) {
                const bool more = r0 + RT < rhi;
                if (more) load(r0 + RT);
                f32x16 x = {}, y = {};
#pragma unroll
                for (int c = 0; c < D / 16; ++c) x = mfma(T::rows(qt[buf], 0, c, lane), k[c], x);
#pragma unroll
                for (int c = 0; c < D / 16; ++c) y = mfma(T::rows(ot[buf], 0, c, lane), v[c], y);
                const int me = 32 * wave + col;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int at = 8 * q + 4 * h;
                    const float4 ls = *reinterpret_cast<const float4*>(&stat[buf][0][at]);
                    const float4 dl = *reinterpret_cast<const float4*>(&stat[buf][1][at]);
                    const int4 f = *reinterpret_cast<const int4*>(&see[buf][0][at]);
                    const int4 z = *reinterpret_cast<const int4*>(&see[buf][1][at]);
                    const float lv[4] = {ls.x, ls.y, ls.z, ls.w}, dv4[4] = {dl.x, dl.y, dl.z, dl.w};
                    const int fv[4] = {f.x, f.y, f.z, f.w}, zv[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool on = me >= fv[e] && me <= zv[e];
                        const float p = on ? __builtin_amdgcn_exp2f(x[4 * q + e] * sl - lv[e]) : 0.0f;
                        x[4 * q + e] = p;
                        y[4 * q + e] = on ? p * (y[4 * q + e] - dv4[e]) : 0.0f;
                    }
                }
                bf16x8 p[2], ds[2];
                pack_tile(x, p);
                pack_tile(y, ds);
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        dv[i] = mfma(T::cols(ot[buf], 16 * c, i, lane), p[c], dv[i]);
                        dk[i] = mfma(T::cols(qt[buf], 16 * c, i, lane), ds[c], dk[i]);
                    }
                if (more) put(buf ^ 1);
                __syncthreads();
            }
        }
        if (j < cover) {
            uint8_t* ok = kv_at(a.dk, a, s, hk) + (a.dk.f32 ? 4 : 2) * j * a.dk.ts;
            uint8_t* ov = kv_at(a.dv, a, s, hk) + (a.dv.f32 ? 4 : 2) * j * a.dv.ts;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d0 = 32 * i + 8 * e + 4 * h;
                    if (d0 < a.d) {
                        store4(ok, a.dk.f32, d0, dk[i][4 * e] * a.scale, dk[i][4 * e + 1] * a.scale,
                               dk[i][4 * e + 2] * a.scale, dk[i][4 * e + 3] * a.scale);
                        store4(ov, a.dv.f32, d0, dv[i][4 * e], dv[i][4 * e + 1], dv[i][4 * e + 2], dv[i][4 * e + 3]);
                    }
                }
        }
        __syncthreads();
    }
}

template <int D>
int launch(const Args& a, hipStream_t st) {
    const int64_t tiles = (a.lq * a.g + 127) / 128, keys = (a.lk + 127) / 128;
    if (tiles > 0) {
        hipLaunchKernelGGL(attn_dq_kernel<D>, dim3((unsigned)(tiles < 65535 ? tiles : 65535), a.hk, a.batch), dim3(256), 0, st, a);
        if (int e = launch_status("attn_dq_kernel")) return e;
    }
    if (keys > 0) {
        hipLaunchKernelGGL(attn_dkdv_kernel<D>, dim3((unsigned)(keys < 65535 ? keys : 65535), a.hk, a.batch), dim3(256), 0, st, a);
        return launch_status("attn_dkdv_kernel");
    }
    return R97Q_OK;
}

}  // namespace

int launch_bwd(const Args& a, hipStream_t st) {
    return a.d <= 64 ? launch<64>(a, st) : a.d <= 128 ? launch<128>(a, st) : launch<256>(a, st);
}

}  // namespace attn
}  // namespace r97q
