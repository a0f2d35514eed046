// attn_dkdv.hip -- attention's backward pass, second launch: dK and dV (the formulas and the first launch are in
// attn_dq.hip). Built once for heads of up to 128 columns and once, R97Q_WIDE, for heads of 256.
#include "attn.h"
#include "status.h"

namespace r97q {
namespace attn {
namespace {

// ---------------------------------------------------------------- dK, dV: 32 NW keys a workgroup
// A wave holds 32 keys and their gradients; the workgroup walks the heads and the tokens that see its keys,
// RT tokens of a head at a time. KEPT: the keys stay in registers; at 256 columns the gradients take 256 of a
// lane's 512 and the keys stay in LDS instead.
template <int D, int RT, int NW, bool KEPT>
__global__ __launch_bounds__(64 * NW, 1) void attn_dkdv_kernel(Args a) {
    using T = Tile<D>;
    using F = Frags<D>;
    constexpr int TB = RT * T::RB, n = D / 16, KB = KEPT ? 0 : 32 * NW * T::RB;
    // queries' two slots, then dO's, then the keys
    __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * TB + KB];
    __shared__ __attribute__((aligned(16))) float stat[2][2][64];  // log-sum-exp in base 2, and D, of a tile's rows
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, h = lane >> 5;
    const int nb = a.batch * a.hk, bh = blockIdx.x % nb, hk = bh % a.hk, tiles = gridDim.x / nb;
    const Seq s = sequence(a, bh / a.hk);
    const int cover = a.kv_starts ? s.lk : a.lk;  // the dense form's keys past a sequence's length get zeros
    const float sl = back_scale(a), out_of_sight = sl > 0.0f ? -INFINITY : INFINITY;
    const int64_t qts = 2 * a.q.ts, ots = 2 * a.d_o.ts;
    const Loader<D, RT, 64 * NW> ql(qts, a.d, tid), ol(ots, a.d, tid);
    const uint32_t at = lds_at(lds), mine = at + 1024 * wave, rat = at + F::row0(lane), cat = at + F::col0(lane);
    const uint32_t hat = rat + 4 * TB + 32 * wave * T::RB;  // the wave's keys, where they are not kept
    for (int64_t tile = (int)(blockIdx.x / nb); tile * 32 * NW < cover; tile += tiles) {
        const int w0 = (int)tile * 32 * NW, k0 = w0 + 32 * wave, key = k0 + col;
        bf16x8 k[KEPT ? D / 16 : 1], v[D / 16];
        const int kk = key < s.lk ? key : 0;
        if constexpr (KEPT) {
            load_row<D>(kv_at(a.k, a, s, hk) + 2 * (kk * a.k.ts), key < s.lk, fresh(a.d), lane, k);
        } else {
            const Loader<D, 32, 64 * NW> kl(2 * a.k.ts, a.d, tid);
            Rows kr(kv_at(a.k, a, s, hk), 2 * a.k.ts, w0, s.lk, a.d);
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                kl.load(kr, mine + 4 * TB + i * 32 * T::RB);
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
        if (t0 < t1) {
            // where the next tile of tokens lies: a head's, from t0, then the next head's
            const int64_t qhs = 2 * a.q.hs, ohs = 2 * a.d_o.hs;
            const uint8_t *qb = q_at(a.q, a, s, hk * a.g), *ob = q_at(a.d_o, a, s, hk * a.g);
            const uint8_t* sb = reinterpret_cast<const uint8_t*>((wave & 1 ? a.delta : a.base) + stat_at(a, s, hk * a.g, 0));
            const int64_t shs = 4 * (a.q_starts ? a.q_tokens : a.lq);
            Rows qr(qb, qts, t0, t1, a.d), orr(ob, ots, t0, t1, a.d), sr(sb, 4, t0, t1, 2);
            auto load_stat = [&](int slot) {  // wave 0 the one, wave 1 the other
                if (wave < 2) load_words(sr.buffer(), 4 * lane, lds_at(stat) + 512 * slot + 256 * wave);
            };
            ql.load(qr, mine);
            ol.load(orr, mine + 2 * TB);
            load_stat(0);
            const int per = (t1 - t0 + RT - 1) / RT, count = per * a.g;
            int t = t0, left = per;
            for (int step = 0, slot = 0; step < count; ++step, slot ^= 1) {
                if (--left == 0) {
                    qb += qhs, ob += ohs, sb += shs;
                    left = per;
                    qr = Rows(qb, qts, t0, t1, a.d);
                    orr = Rows(ob, ots, t0, t1, a.d);
                    sr = Rows(sb, 4, t0, t1, 2);
                    if (step + 1 == count) qr.left = orr.left = sr.left = 0;  // nothing follows: zeros
                } else {
                    qr.step(RT * qts, 2 * a.d);
                    orr.step(RT * ots, 2 * a.d);
                    sr.step(4 * RT, 4);
                }
                landed();
                __syncthreads();
                load_stat(slot ^ 1);
                const int tl = t + RT - 1 < t1 ? t + RT - 1 : t1 - 1;
                // every row of the tile sees every key of the wave
                const bool whole = t + RT <= t1 && (!a.causal || ((int64_t)t + s.off >= k0 + 31 &&
                                                                  (!a.window || (int64_t)tl + s.off - a.window < k0)));
                constexpr int total = 4 * n * (RT / 32);
                const uint32_t qat = rat + slot * TB, qct = cat + slot * TB, sat = lds_at(stat) + 512 * slot + 16 * h;
                typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
                f32x16 x = {}, y = {};
                u32x4 p[2], ds[2];
                f32x4 ls[4], dl[4];
                bf16x8 f[kAhead], kf[kAhead];
                // operand of product i: of 32 rows, Q and dO as they lie, then the columns of dO and Q
                auto frag = [&](auto i) {
                    constexpr int sub = i / (4 * n), ph = i % (4 * n) / n, c = i % n;
                    if constexpr (ph == 0) return F::template rows<32 * sub, c>(qat);
                    else if constexpr (ph == 1) return F::template rows<32 * sub + 2 * RT, c>(qat);
                    else return F::template cols<32 * sub + 16 * (c / (D / 32)) + (ph == 2 ? 2 * RT : 0), c % (D / 32)>(qct);
                };
                steps<kAhead>([&](auto i) {
                    f[i] = frag(i);
                    if constexpr (!KEPT) kf[i] = F::template rows<0, i>(hat);
                });
                steps<total>([&](auto i) {
                    constexpr int sub = i / (4 * n), ph = i % (4 * n) / n, c = i % n;
                    if constexpr (ph == 1 && c == 0) {
                        if (!whole) {  // the rows, from the tile's first, that see the lane's key
                            const int top = a.causal ? (int)clamp64((int64_t)key - s.off - t, 0, RT) : 0;
                            const int cap = t1 - t < RT ? t1 - t : RT;
                            const int end = a.window ? (int)clamp64((int64_t)key - s.off - t + a.window, 0, cap) : cap;
                            const uint32_t many = end < top ? 0u : (uint32_t)(end - top), from = (uint32_t)(32 * sub + 4 * h - top);
#pragma unroll
                            for (int e = 0; e < 16; ++e) x[e] = from + (uint32_t)(8 * (e >> 2) + (e & 3)) < many ? x[e] : out_of_sight;
                        }
                    }
                    pin();
                    const bf16x8 now = f[i % kAhead];
                    if constexpr (i + kAhead < total) f[i % kAhead] = frag(std::integral_constant<int, i + kAhead>{});
                    if constexpr (i == 1) ql.load(qr, mine + (slot ^ 1) * TB);
                    if constexpr (i == 2) ol.load(orr, mine + (2 + (slot ^ 1)) * TB);
                    // the vector work of a product's results starts two products after its last
                    constexpr int w = c - 2, m = n - 2;
                    if constexpr (ph == 0) {
                        bf16x8 kc;
                        if constexpr (KEPT) {
                            kc = k[c];
                        } else {
                            kc = kf[c % kAhead];
                            if constexpr (c + kAhead < n) kf[c % kAhead] = F::template rows<0, c + kAhead>(hat);
                        }
                        if constexpr (c == 0) x = (f32x16){};
                        x = mfma(now, kc, x);
                        if constexpr (c >= n - 4) ls[c - (n - 4)] = *(lds_f32x4*)(uintptr_t)(sat + 128 * sub + 32 * (c - (n - 4)));
                    } else if constexpr (ph == 1) {
                        if constexpr (c == 0) y = (f32x16){};
                        y = mfma(now, v[c], y);
                        if constexpr (w >= 0) {
#pragma unroll
                            for (int e = 2 * (8 * w / m); e < 2 * (8 * (w + 1) / m); e += 2) {
                                x[e] = __builtin_amdgcn_exp2f(x[e] * sl - ls[e >> 2][e & 3]);
                                x[e + 1] = __builtin_amdgcn_exp2f(x[e + 1] * sl - ls[e >> 2][(e & 3) + 1]);
                                pack_two(x, e, p);
                            }
                        }
                        if constexpr (c >= n - 4) dl[c - (n - 4)] = *(lds_f32x4*)(uintptr_t)(sat + 256 + 128 * sub + 32 * (c - (n - 4)));
                    } else if constexpr (ph == 2) {
                        dv[c % (D / 32)] = mfma(now, as_bf16x8(p[c / (D / 32)]), dv[c % (D / 32)]);
                        if constexpr (w >= 0) {
#pragma unroll
                            for (int e = 2 * (8 * w / m); e < 2 * (8 * (w + 1) / m); e += 2) {
                                y[e] = x[e] * (y[e] - dl[e >> 2][e & 3]);
                                y[e + 1] = x[e + 1] * (y[e + 1] - dl[e >> 2][(e & 3) + 1]);
                                pack_two(y, e, ds);
                            }
                        }
                    } else {
                        dk[c % (D / 32)] = mfma(now, as_bf16x8(ds[c / (D / 32)]), dk[c % (D / 32)]);
                        if constexpr (!KEPT && sub + 1 < RT / 32 && c >= n - kAhead)
                            kf[c - (n - kAhead)] = F::template rows<0, c - (n - kAhead)>(hat);
                    }
                });
                pin();
                t = left == per ? t0 : t + RT;
            }
        }
        landed();
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

template <int D, int RT, bool KEPT>
int run(const Args& a, hipStream_t st) {
    const int64_t nb = (int64_t)a.batch * a.hk, most = 0x7FFFFFFF / nb;
    int64_t keys = ((int64_t)a.lk + 127) / 128;
    if (keys > most) keys = most;
    if (keys == 0) return R97Q_OK;
    hipLaunchKernelGGL((attn_dkdv_kernel<D, RT, 4, KEPT>), dim3((unsigned)(keys * nb)), dim3(256), 0, st, a);
    return launch_status("attn_dkdv_kernel");
}

}  // namespace

#if R97Q_WIDE
int launch_dkdv_wide(const Args& a, hipStream_t st) { return run<256, 32, false>(a, st); }
#else
int launch_dkdv(const Args& a, hipStream_t st) { return a.d <= 64 ? run<64, 64, true>(a, st) : run<128, 64, true>(a, st); }
#endif

}  // namespace attn
}  // namespace r97q
