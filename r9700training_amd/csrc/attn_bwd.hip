// attn_bwd.hip -- attention's backward pass, the probabilities recomputed from the log-sum-exp L:
//   P = exp(scale Q K^T - L)    D_i = sum_d dO_id O_id    dS = P o (dO V^T - D)
//   dV = P^T dO    dQ = scale dS K    dK = scale dS^T Q,  dK and dV summed over the heads that share a key head.
//
// Two launches: attn_dq_kernel walks the keys for tiles of rows (and writes D), attn_dkdv_kernel walks the
// rows for tiles of keys. Both recompute P and dO V^T: seven products where one launch would need five,
// but every sum has one owner and a fixed order, so repeated calls give the same bits, and no f32 gradient
// passes through memory. P and dS are rounded to bf16 for their products (half a step of 2^-8 relative, each
// term of a sum on its own), everything else is f32.
//
// Bound by the matrix cores. The vector work of a tile lies beside products that do not need it: the
// exponentials beside dO V^T, dS beside dV.
#include "attn.h"
#include "status.h"

namespace r97q {
namespace attn {
namespace {

// ---------------------------------------------------------------- dQ (and D): 32 NW rows a workgroup
template <int D, int KT, int NW, int PER>
__global__ __launch_bounds__(64 * NW, PER) void attn_dq_kernel(Args a) {
    using T = Tile<D>;
    constexpr int TB = KT * T::RB;
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * TB];  // keys' two slots, then the values'
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, h = lane >> 5;
    const int nb = a.batch * a.hk, bh = blockIdx.x % nb, hk = bh % a.hk, tiles = gridDim.x / nb;
    const Seq s = sequence(a, bh / a.hk);
    const int rows = s.lq * a.g;
    const float sl = a.scale * kLog2e;
    const uint8_t* kb = kv_at(a.k, a, s, hk);
    const uint8_t* vb = kv_at(a.v, a, s, hk);
    const int64_t kts = 2 * a.k.ts, vts = 2 * a.v.ts;
    const Loader<D, KT, 64 * NW> kl(kts, a.d, tid), vl(vts, a.d, tid);
    const uint32_t mine = lds_at(lds) + 1024 * wave;
    for (int64_t tile = tiles - 1 - (int)(blockIdx.x / nb); tile * 32 * NW < rows; tile += tiles) {
        const int w0 = (int)tile * 32 * NW, r0 = w0 + 32 * wave, r = r0 + col;
        const int rr = r < rows ? r : rows - 1, tok = rr / a.g, head = hk * a.g + (rr - tok * a.g);
        const int wend = w0 + 32 * NW - 1 < rows ? w0 + 32 * NW - 1 : rows - 1;
        const Keys all = keys_of(a, s, w0 / a.g, wend / a.g);
        const int rend = r0 + 31 < rows ? r0 + 31 : rows - 1;
        const Keys own = keys_of(a, s, (r0 < rows ? r0 : rows - 1) / a.g, rend / a.g);
        const int lo = all.lo / KT * KT, hi = all.hi;
        Rows kr(kb, kts, lo, hi, a.d), vr(vb, vts, lo, hi, a.d);
        if (lo < hi) {
            kl.load(kr, mine);
            vl.load(vr, mine + 2 * TB);
        }
        int d = fresh(a.d);
        bf16x8 q[D / 16], go[D / 16];
        load_row<D>(q_at(a.q, a, s, head) + 2 * (tok * a.q.ts), r < rows, d, lane, q);
        load_row<D>(q_at(a.d_o, a, s, head) + 2 * (tok * a.d_o.ts), r < rows, d, lane, go);
        const uint8_t* op = q_at(a.o, a, s, head) + (a.o.f32 ? 4 : 2) * (tok * a.o.ts);
        float delta = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            const int e = 16 * c + 8 * h;
            if (e < d) {
                if (a.o.f32) {
                    const float4 x = *reinterpret_cast<const float4*>(op + 4 * e), y = *reinterpret_cast<const float4*>(op + 4 * e + 16);
                    delta += x.x * (float)go[c][0] + x.y * (float)go[c][1] + x.z * (float)go[c][2] + x.w * (float)go[c][3];
                    delta += y.x * (float)go[c][4] + y.y * (float)go[c][5] + y.z * (float)go[c][6] + y.w * (float)go[c][7];
                } else {
                    const bf16x8 x = as_bf16x8(*reinterpret_cast<const u32x4*>(op + 2 * e));
#pragma unroll
                    for (int j = 0; j < 8; ++j) delta += (float)x[j] * (float)go[c][j];
                }
            }
        }
        delta = pair_sum(delta);
        const int64_t at = stat_at(a, s, head, tok);
        const float lse = a.lse[at], base = lse == -INFINITY ? 0.0f : lse * kLog2e;
        if (r < rows && h == 0) a.base[at] = make_float2(base, delta);
        const int first = a.window ? (int)clamp64((int64_t)tok + s.off - a.window + 1, 0, s.lk) : 0;
        const int last = a.causal && tok + s.off < s.lk - 1 ? tok + s.off : s.lk - 1;
        f32x16 dq[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dq[i] = (f32x16){};
        int slot = 0;
        for (int j0 = lo; j0 < hi; j0 += KT, slot ^= 1) {
            landed();
            __syncthreads();
            if (j0 + KT < hi) {
                kr.step(KT * kts, 2 * a.d);
                vr.step(KT * vts, 2 * a.d);
                kl.load(kr, mine + (slot ^ 1) * TB);
                vl.load(vr, mine + (2 + (slot ^ 1)) * TB);
            }
            if (j0 >= own.hi || j0 + KT <= own.lo || r0 >= rows) continue;
            const uint8_t *kt = lds + slot * TB, *vt = lds + (2 + slot) * TB;
            f32x16 x[KT / 32], y[KT / 32];
#pragma unroll
            for (int i = 0; i < KT / 32; ++i) x[i] = y[i] = (f32x16){};
#pragma unroll
            for (int c = 0; c < D / 16; ++c)
#pragma unroll
                for (int i = 0; i < KT / 32; ++i) x[i] = mfma(T::rows(kt, 32 * i, c, lane), q[c], x[i]);
#pragma unroll
            for (int c = 0; c < D / 16; ++c)
#pragma unroll
                for (int i = 0; i < KT / 32; ++i) y[i] = mfma(T::rows(vt, 32 * i, c, lane), go[c], y[i]);
#pragma unroll
            for (int i = 0; i < KT / 32; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) x[i][e] = __builtin_amdgcn_exp2f(x[i][e] * sl - base) * (y[i][e] - delta);
            if (j0 < own.all_lo || j0 + KT > own.all_hi) {
                const uint32_t many = last < first ? 0u : (uint32_t)(last - first) + 1u, from = (uint32_t)(j0 + 4 * h - first);
#pragma unroll
                for (int i = 0; i < KT / 32; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const uint32_t j = from + (uint32_t)(32 * i + 8 * (e >> 2) + (e & 3));
                        x[i][e] = j < many ? x[i][e] : 0.0f;
                    }
            }
#pragma unroll
            for (int i = 0; i < KT / 32; ++i) {
                bf16x8 ds[2];
                pack_tile(x[i], ds);
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int n = 0; n < D / 32; ++n) dq[n] = mfma(T::cols(kt, 32 * i + 16 * c, n, lane), ds[c], dq[n]);
            }
        }
        d = fresh(a.d);
        const int hs = fresh_lane(h);
        uint8_t* out = q_at(a.dq, a, s, head) + (a.dq.f32 ? 4 : 2) * (tok * a.dq.ts);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) store_block(out, a.dq.f32, r < rows, 32 * i, d, hs, dq[i], a.scale);
        __syncthreads();
    }
}

// ---------------------------------------------------------------- dK, dV: 32 NW keys a workgroup
// A wave holds 32 keys and their gradients; the workgroup walks the heads and the tokens that see its keys,
// RT tokens of a head at a time. KEPT: the keys stay in registers; at 256 columns the gradients take 256 of a
// lane's 512 and the keys stay in LDS instead.
template <int D, int RT, int NW, bool KEPT>
__global__ __launch_bounds__(64 * NW, 1) void attn_dkdv_kernel(Args a) {
    using T = Tile<D>;
    constexpr int TB = RT * T::RB;
    constexpr int KB = KEPT ? 0 : 32 * NW * T::RB;
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * TB + KB];         // queries' two slots, then dO's, then the keys
    __shared__ __attribute__((aligned(16))) float2 stat[2][RT];               // (log-sum-exp in base 2, D) a row
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, h = lane >> 5;
    const int nb = a.batch * a.hk, bh = blockIdx.x % nb, hk = bh % a.hk, tiles = gridDim.x / nb;
    const Seq s = sequence(a, bh / a.hk);
    const int cover = a.kv_starts ? s.lk : a.lk;  // the dense form's keys past a sequence's length get zeros
    const float sl = a.scale * kLog2e;
    const int64_t qts = 2 * a.q.ts, ots = 2 * a.d_o.ts;
    const Loader<D, RT, 64 * NW> ql(qts, a.d, tid), ol(ots, a.d, tid);
    const uint32_t mine = lds_at(lds) + 1024 * wave, smine = lds_at(stat) + 256 * wave;
    for (int64_t tile = (int)(blockIdx.x / nb); tile * 32 * NW < cover; tile += tiles) {
        const int w0 = (int)tile * 32 * NW, k0 = w0 + 32 * wave, key = k0 + col;
        bf16x8 k[KEPT ? D / 16 : 1], v[D / 16];
        const int kk = key < s.lk ? key : 0;
        uint8_t* held = lds + 4 * TB;
        if constexpr (KEPT) {
            load_row<D>(kv_at(a.k, a, s, hk) + 2 * (kk * a.k.ts), key < s.lk, fresh(a.d), lane, k);
        } else {
            const Loader<D, 32, 64 * NW> kl(2 * a.k.ts, a.d, tid);
            Rows kr(kv_at(a.k, a, s, hk), 2 * a.k.ts, w0, s.lk, a.d);
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                kl.load(kr, lds_at(held) + i * 32 * T::RB + 1024 * wave);
                kr.step(64 * a.k.ts, 2 * a.d);
            }
        }
        load_row<D>(kv_at(a.v, a, s, hk) + 2 * (kk * a.v.ts), key < s.lk, fresh(a.d), lane, v);
        // the tokens [t0, t1) that see any of the workgroup's keys
        const int wend = w0 + 32 * NW - 1 < s.lk ? w0 + 32 * NW - 1 : s.lk - 1;
        int t0 = 0, t1 = s.lq;
        if (a.causal) t0 = (int)clamp64((int64_t)w0 - s.off, 0, s.lq);
        if (a.window) t1 = (int)clamp64((int64_t)wend + a.window - s.off, t0, s.lq);
        if (w0 >= s.lk) t1 = t0;
        f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dk[i] = dv[i] = (f32x16){};
        auto load = [&](int hd, int t, int slot) {
            const Rows qr(q_at(a.q, a, s, hk * a.g + hd), qts, t, t1, a.d), orr(q_at(a.d_o, a, s, hk * a.g + hd), ots, t, t1, a.d);
            ql.load(qr, mine + slot * TB);
            ol.load(orr, mine + (2 + slot) * TB);
            if (64 * wave < 2 * RT) {
                const Rows sr(reinterpret_cast<const uint8_t*>(a.base + stat_at(a, s, hk * a.g + hd, 0)), 8, t, t1, 4);
                load_words(sr.buffer(), 4 * tid, smine + slot * (8 * RT));
            }
        };
        if (t0 < t1) {
            load(0, t0, 0);
            int hd = 0, t = t0, slot = 0;
            while (hd < a.g) {
                int hn = hd, tn = t + RT;  // the next tile
                if (tn >= t1) tn = t0, ++hn;
                landed();
                __syncthreads();
                if (hn < a.g) load(hn, tn, slot ^ 1);
                const int tl = t + RT - 1 < t1 ? t + RT - 1 : t1 - 1;
                // none of the wave's keys is seen: tokens before them, or past their window
                const bool none = k0 >= s.lk || (a.causal && tl + s.off < k0) ||
                                  (a.window && (int64_t)t + s.off - a.window >= k0 + 31);
                if (!none) {
                    const bool whole = t + RT <= t1 && (!a.causal || ((int64_t)t + s.off >= k0 + 31 && (!a.window || (int64_t)tl + s.off - a.window < k0)));
                    const uint8_t *qt = lds + slot * TB, *ot = lds + (2 + slot) * TB;
#pragma unroll
                    for (int i = 0; i < RT / 32; ++i) {
                        f32x16 x = {}, y = {};
#pragma unroll
                        for (int c = 0; c < D / 16; ++c)
                            x = mfma(T::rows(qt, 32 * i, c, lane), KEPT ? k[KEPT ? c : 0] : T::rows(held, 32 * wave, c, lane), x);
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) y = mfma(T::rows(ot, 32 * i, c, lane), v[c], y);
                        float dl[16];
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float4 w = *reinterpret_cast<const float4*>(&stat[slot][32 * i + 8 * (e >> 2) + 4 * h + (e & 3)]);
                            x[e] = __builtin_amdgcn_exp2f(x[e] * sl - w.x);
                            x[e + 1] = __builtin_amdgcn_exp2f(x[e + 1] * sl - w.z);
                            dl[e] = w.y;
                            dl[e + 1] = w.w;
                        }
                        if (!whole) {  // the rows, from the tile's first, that see the lane's key
                            const int top = a.causal ? (int)clamp64((int64_t)key - s.off - t, 0, RT) : 0;
                            const int cap = t1 - t < RT ? t1 - t : RT;
                            const int end = a.window ? (int)clamp64((int64_t)key - s.off - t + a.window, 0, cap) : cap;
                            const uint32_t many = end < top ? 0u : (uint32_t)(end - top), from = (uint32_t)(32 * i + 4 * h - top);
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const uint32_t row = from + (uint32_t)(8 * (e >> 2) + (e & 3));
                                x[e] = row < many ? x[e] : 0.0f;
                            }
                        }
                        bf16x8 p[2], ds[2];
                        pack_tile(x, p);
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int d = 0; d < D / 32; ++d) dv[d] = mfma(T::cols(ot, 32 * i + 16 * c, d, lane), p[c], dv[d]);
#pragma unroll
                        for (int e = 0; e < 16; ++e) y[e] = x[e] * (y[e] - dl[e]);
                        pack_tile(y, ds);
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int d = 0; d < D / 32; ++d) dk[d] = mfma(T::cols(qt, 32 * i + 16 * c, d, lane), ds[c], dk[d]);
                    }
                }
                hd = hn;
                t = tn;
                slot ^= 1;
            }
        }
        if constexpr (!KEPT) landed();
        const bool seen = key < s.lk;
        const int dd = fresh(a.d), hs = fresh_lane(h);
        uint8_t* ok = kv_at(a.dk, a, s, hk) + (a.dk.f32 ? 4 : 2) * (key * a.dk.ts);
        uint8_t* ov = kv_at(a.dv, a, s, hk) + (a.dv.f32 ? 4 : 2) * (key * a.dv.ts);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            if (!seen) dk[i] = dv[i] = (f32x16){};
            store_block(ok, a.dk.f32, key < cover, 32 * i, dd, hs, dk[i], a.scale);
            store_block(ov, a.dv.f32, key < cover, 32 * i, dd, hs, dv[i], 1.0f);
        }
        __syncthreads();
    }
}

template <int D, int KT, int PER, int RT, bool KEPT>
int launch(const Args& a, hipStream_t st) {
    const int64_t nb = (int64_t)a.batch * a.hk, most = 0x7FFFFFFF / nb;
    int64_t tiles = ((int64_t)a.lq * a.g + 127) / 128, keys = (a.lk + 127) / 128;
    if (tiles > most) tiles = most;
    if (keys > most) keys = most;
    if (tiles > 0) {
        hipLaunchKernelGGL((attn_dq_kernel<D, KT, 4, PER>), dim3((unsigned)(tiles * nb)), dim3(256), 0, st, a);
        if (int e = launch_status("attn_dq_kernel")) return e;
    }
    if (keys > 0) {
        hipLaunchKernelGGL((attn_dkdv_kernel<D, RT, 4, KEPT>), dim3((unsigned)(keys * nb)), dim3(256), 0, st, a);
        return launch_status("attn_dkdv_kernel");
    }
    return R97Q_OK;
}

}  // namespace

int launch_bwd(const Args& a, hipStream_t st) {
    return a.d <= 64 ? launch<64, 64, 2, 64, true>(a, st) : a.d <= 128 ? launch<128, 32, 2, 32, true>(a, st) : launch<256, 32, 1, 32, false>(a, st);
}

}  // namespace attn
}  // namespace r97q
