// attn_dkdv.hip -- attention's backward pass: dK and dV (the formulas and the other launches are in attn_dq.hip). Built once
// for heads of up to 128 columns and once, R97Q_WIDE, for heads of 256.
#include "attn.h"
#include "status.h"

namespace r97q {
namespace attn {
namespace {

// ---------------------------------------------------------------- dK, dV: 32 NW keys a workgroup
// A wave holds 32 keys and their gradients; the workgroup walks the heads and the tokens that see its keys,
// RT tokens of a head at a time. KEPT: the keys stay in registers; at 256 columns the gradients take 256 of a
// lane's 512 and the keys stay in LDS instead. SLOTS: tiles of Q and dO in LDS; with three, the
// next tile has landed a step early and its first operands are read before the step's barrier. STORE: dS^T is written out for
// dQ's launch.
//
// Bound by the products and what one wave issues beside them. At 128 columns and more the gradients, values and keys leave room
// for one wave a SIMD: a step of 64 tokens at 128 columns is 64 products of 32 cycles among some 470 other instructions (200
// vector, 112 LDS), 1.55 us at 2.4 GHz. 8 x 2048 tokens causal, 16 over 4 heads, counted over the launch: of 64 175 us (785 TFLOP/s
// of the four products; matrix cores busy 38%, vector instructions at 4 cycles each 26%, a wave waits 24%), of 128 276 .. 298 us
// (920 .. 1000; 48%, 19%, 27%), of 256 555 .. 605 us (910 .. 990; 51%, 14%, 24%), at 2.0 GHz; no LDS bank conflicts.
template <int D, int RT, int NW, bool KEPT, int PER, int SLOTS, bool STORE>
__global__ __launch_bounds__(64 * NW, PER) void attn_dkdv_kernel(Args a) {
    using T = Tile<D>;
    using F = Frags<D>;
    constexpr int TB = RT * T::RB, n = D / 16, KB = KEPT ? 0 : 32 * NW * T::RB;
    constexpr bool ACC = PER == 1;
    constexpr int OB = SLOTS * TB, HB = 2 * SLOTS * TB;  // queries' slots, then dO's, then the keys
    __shared__ __attribute__((aligned(1024))) uint8_t lds[HB + KB];
    __shared__ __attribute__((aligned(16))) float stat[SLOTS][2][64];  // log-sum-exp in base 2, and D, of a tile's rows
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, h = lane >> 5;
    const int nb = a.batch * a.hk;
    const Place place(nb, (nb + 7) / 8);  // the heads' queries are too many to keep: by work alone
    const int bh = place.bh, hk = bh % a.hk, part = place.part;
    const int tiles = gridDim.x / (nb * a.k_splits), split = part % a.k_splits;
    const Seq s = sequence(a, bh / a.hk);
    const int cover = a.kv_starts ? s.lk : a.lk;  // the dense form's keys past a sequence's length get zeros
    const float sl = back_scale(a), out_of_sight = sl > 0.0f ? -INFINITY : INFINITY;
    const int64_t qts = 2 * a.q.ts, ots = 2 * a.d_o.ts;
    const uint32_t at = lds_at(lds), mine = at + 1024 * wave, rat = at + F::row0(lane), cat = at + F::col0(lane);
    const uint32_t hat = rat + HB + 32 * wave * T::RB;  // the wave's keys, where they are not kept
    for (int64_t tile = part / a.k_splits; tile * 32 * NW < cover; tile += tiles) {
        const int w0 = (int)tile * 32 * NW, k0 = w0 + 32 * wave, key = k0 + col;
        const int t_ = fresh_lane(tid);  // not held over the results' stores
        const Loader<D, RT, 64 * NW> ql(qts, a.d, t_), ol(ots, a.d, t_);
        bf16x8 k[KEPT ? D / 16 : 1], v[D / 16];
        const int kk = key < s.lk ? key : 0;
        if constexpr (KEPT) {
            load_row<D>(kv_at(a.k, a, s, hk) + 2 * (kk * a.k.ts), key < s.lk, fresh(a.d), lane, k);
        } else {
            const Loader<D, 32, 64 * NW> kl(2 * a.k.ts, a.d, tid);
            Rows kr(kv_at(a.k, a, s, hk), 2 * a.k.ts, w0, s.lk, a.d);
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                kl.load(kr, mine + HB + i * 32 * T::RB);
                kr.step(32);
            }
        }
        // the values of keys before every query's window may hold anything, and their gradients are zero
        const int seen0 = a.window ? (int)clamp64((int64_t)s.off - a.window + 1, 0, s.lk) : 0;
        load_row<D>(kv_at(a.v, a, s, hk) + 2 * (kk * a.v.ts), key >= seen0 && key < s.lk, fresh(a.d), lane, v);
        settle(v);
        if constexpr (KEPT) settle(k);
        // the tokens [t0, t1) that see any of the workgroup's keys, from a tile's first
        static_assert(NW == 4, "tokens_of() is for 128 keys");
        int t0, t1;
        tokens_of(a, s, w0, RT, t0, t1);
        f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dk[i] = dv[i] = (f32x16){};
        if (t0 < t1) {
            // where the next tile of tokens lies: a head's, from t0, then the next head's
            const int64_t qhs = 2 * a.q.hs, ohs = 2 * a.d_o.hs;
            const uint8_t *qb = q_at(a.q, a, s, hk * a.g), *ob = q_at(a.d_o, a, s, hk * a.g);
            const uint8_t* sb = reinterpret_cast<const uint8_t*>((wave & 1 ? a.delta : a.base) + stat_at(a, s, hk * a.g, 0));
            const int64_t shs = 4 * (a.q_starts ? a.q_tokens : a.lq);
            // the steps [first, end) of a head's tiles of tokens, head after head
            const int per = (t1 - t0 + RT - 1) / RT, count = per * a.g;
            const int first = (int)((int64_t)count * split / a.k_splits), end = (int)((int64_t)count * (split + 1) / a.k_splits);
            const int hd = first / per;
            const int t = t0 + (first - hd * per) * RT;
            int left = per - (first - hd * per);
            qb += hd * qhs, ob += hd * ohs, sb += hd * shs;
            Rows qr(qb, qts, t, t1, a.d), orr(ob, ots, t, t1, a.d), sr(sb, 4, t, t1, 2);
            int to_load = end - first;
            uint16_t* kept = nullptr;  // this key's row of dS^T
            int64_t ds_head = 0;
            if constexpr (STORE) {
                kept = ds_at(a, s, hk * a.g + hd, key < cover ? key : 0);
                ds_head = (a.kv_starts ? a.kv_tokens : (int64_t)a.lk) * a.pitch;
            }
            auto load_stat = [&](int slot) {  // wave 0 the one, wave 1 the other
                if (wave < 2) load_words(sr.template buffer<RT>(), 4 * lane, lds_at(stat) + 512 * slot + 256 * wave);
            };
            auto load_q = [&](int slot) { ql.load(qr, mine + slot * TB); };
            auto load_o = [&](int slot) { ol.load(orr, mine + OB + slot * TB); };
            auto next = [&]() {
                qr.step(RT), orr.step(RT), sr.step(RT);
                if (--left == 0) {
                    qb += qhs, ob += ohs, sb += shs;
                    left = per;
                    qr = Rows(qb, qts, t0, t1, a.d);
                    orr = Rows(ob, ots, t0, t1, a.d);
                    sr = Rows(sb, 4, t0, t1, 2);
                }
                if (--to_load <= 0) qr.left = orr.left = sr.left = 0;  // nothing follows: zeros
            };
#pragma unroll
            for (int i = 0; i < SLOTS - 1; ++i) {
                load_stat(i);
                load_q(i);
                load_o(i);
                next();
            }
            // A tile of tokens from t on is whole, every row seeing every key of the wave, for t in [whole0, whole1].
            const int whole0 = a.causal ? (int)clamp64((int64_t)k0 + 31 - s.off, 0, 0x7FFFFFFF) : 0;
            const int whole1 = (a.window ? (int)clamp64((int64_t)k0 + a.window - s.off, -1, t1) : t1) - RT;
            bf16x8 f[kAhead], kf[kAhead];
            uint32_t held = hat;
            auto first_frags = [&](uint32_t at0) {
                steps<kAhead>([&](auto i) {
                    f[i] = F::template rows<0, i>(at0);
                    if constexpr (!KEPT) kf[i] = F::template rows<0, i>(held);
                });
            };
            if constexpr (SLOTS > 2) {
                landed();
                __syncthreads();
                first_frags(rat);
            }
            for (int step = first, slot = 0, fill = SLOTS - 1, at_t = t; step < end; ++step) {
                // all but the last step's stores, which went out after its loads (a wave past the keys has none)
                if (STORE && step > first && k0 < cover)
                    landed<2 * (RT / 32)>();
                else
                    landed();
                __syncthreads();
                load_stat(fill);
                held = (uint32_t)fresh_lane((int)hat);  // its addresses are made here, not held through the loop
                const int t = at_t, slot1 = slot + 1 == SLOTS ? 0 : slot + 1;
                const bool whole = t >= whole0 && t <= whole1;
                constexpr int total = 4 * n * (RT / 32);
                const uint32_t qat = rat + slot * TB, oat = qat + OB, qct = cat + slot * TB, oct = qct + OB, sat = lds_at(stat) + 512 * slot + 16 * h;
                typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
                f32x16 x = {}, y = {};
                u32x4 p[2], ds[2];
                f32x4 ls[4];
                const uint32_t qat1 = rat + slot1 * TB;
                // operand of product i: of 32 rows, Q and dO as they lie, then the columns of dO and Q; then the next step's
                auto frag = [&](auto i) {
                    constexpr int sub = i / (4 * n), ph = i % (4 * n) / n, c = i % n;
                    if constexpr (i >= total) return F::template rows<0, i - total>(qat1);
                    else if constexpr (ph == 0) return F::template rows<32 * sub, c>(qat);
                    else if constexpr (ph == 1) return F::template rows<32 * sub, c>(oat);
                    else return F::template cols<32 * sub + 16 * (c / (D / 32)), c % (D / 32)>(ph == 2 ? oct : qct);
                };
                if constexpr (SLOTS == 2) first_frags(qat);
                steps<total>([&](auto i) {
                    constexpr int sub = i / (4 * n), ph = i % (4 * n) / n, c = i % n;
                    if constexpr (ph == 1 && c == 0) {
                        if (!whole) {
                            asm volatile("");  // a branch: most tiles need no mask
                            // the rows, from the tile's first, that see the lane's key
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
                    if constexpr (SLOTS > 2 || i + kAhead < total) f[i % kAhead] = frag(std::integral_constant<int, i + kAhead>{});
                    if constexpr (i == 1) load_q(fill);
                    if constexpr (i == 2) load_o(fill);
                    if constexpr (ph == 0) {
                        bf16x8 kc;
                        if constexpr (KEPT) {
                            kc = k[c];
                        } else {
                            kc = kf[c % kAhead];
                            if constexpr (c + kAhead < n) kf[c % kAhead] = F::template rows<0, c + kAhead>(held);
                        }
                        if constexpr (c == 0) x = (f32x16){};
                        x = mfma(now, kc, x);
                        if constexpr (c >= n - 4) {
                            constexpr int r = c - (n - 4);
                            ls[r] = *(lds_f32x4*)(uintptr_t)(sat + 128 * sub + 32 * r);
                            const f32x4 dl = *(lds_f32x4*)(uintptr_t)(sat + 256 + 128 * sub + 32 * r);
#pragma unroll
                            for (int e = 0; e < 4; ++e) y[4 * r + e] = dl[e];  // dO V^T - D: the sum starts from -D
                        }
                    } else if constexpr (ph == 1) {
                        y = mfma(now, v[c], y);
                    } else if constexpr (ph == 2) {
                        add_product<ACC>(now, as_bf16x8(p[c / (D / 32)]), dv[c % (D / 32)]);
                    } else {
                        add_product<ACC>(now, as_bf16x8(ds[c / (D / 32)]), dk[c % (D / 32)]);
                        if constexpr (!KEPT && (SLOTS > 2 || sub + 1 < RT / 32) && c >= n - kAhead)
                            kf[c - (n - kAhead)] = F::template rows<0, c - (n - kAhead)>(held);
                    }
                    if constexpr (STORE && ph == 3 && c == n - 1) {
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            if (key < cover) *reinterpret_cast<u32x4*>(kept + t + 32 * sub + 16 * u + 8 * h) = rows_of(ds[u]);
                    }
                    // Vector work, spread over the products that do not need it: the exponentials from two products after
                    // x's last one to the second half's use, dS likewise after y's.
                    constexpr int st = i % (4 * n), len = n - 3 + D / 32;
#pragma unroll
                    for (int e = pair_from(st, n + 2, len); e < pair_from(st + 1, n + 2, len); e += 2) {
                        x[e] = __builtin_amdgcn_exp2f(x[e] * sl - ls[e >> 2][e & 3]);
                        x[e + 1] = __builtin_amdgcn_exp2f(x[e + 1] * sl - ls[e >> 2][(e & 3) + 1]);
                        pack_two(x, e, p);
                    }
#pragma unroll
                    for (int e = pair_from(st, 2 * n + 2, len); e < pair_from(st + 1, 2 * n + 2, len); e += 2) {
                        y[e] *= x[e];
                        y[e + 1] *= x[e + 1];
                        pack_two(y, e, ds);
                    }
                });
                pin();
                next();
                if constexpr (STORE) {
                    if (t + RT >= t1) kept += ds_head;
                }
                at_t = t + RT < t1 ? t + RT : t0;
                slot = slot1;
                fill = fill + 1 == SLOTS ? 0 : fill + 1;
            }
        }
        landed();
        settled<ACC>();
        const bool seen = key < s.lk;
        const int dd = fresh(a.d), hs = fresh_lane(h);
        if (a.k_splits > 1) {
            const int64_t at = (split * a.kv_slots + kv_slot(a, s, hk, key)) * dd;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                settle_sum<ACC>(dk[i]);
                if (!seen) dk[i] = (f32x16){};
                store_block(reinterpret_cast<uint8_t*>(a.dk_part + at), true, key < cover, 32 * i, dd, hs, dk[i], 1.0f);
                settle_sum<ACC>(dv[i]);
                if (!seen) dv[i] = (f32x16){};
                store_block(reinterpret_cast<uint8_t*>(a.dv_part + at), true, key < cover, 32 * i, dd, hs, dv[i], 1.0f);
            }
            __syncthreads();
            continue;
        }
        uint8_t* ok = kv_at(a.dk, a, s, hk) + (a.dk.f32 ? 4 : 2) * (key * a.dk.ts);
        uint8_t* ov = kv_at(a.dv, a, s, hk) + (a.dv.f32 ? 4 : 2) * (key * a.dv.ts);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            settle_sum<ACC>(dk[i]);
            if (!seen) dk[i] = (f32x16){};
            store_block(ok, a.dk.f32, key < cover, 32 * i, dd, hs, dk[i], a.scale);
            settle_sum<ACC>(dv[i]);
            if (!seen) dv[i] = (f32x16){};
            store_block(ov, a.dv.f32, key < cover, 32 * i, dd, hs, dv[i], 1.0f);
        }
        __syncthreads();
    }
}

template <int D, int RT, bool KEPT, int PER, int SLOTS>
int run(const Args& a, hipStream_t st) {
    const int64_t nb = (int64_t)a.batch * a.hk * a.k_splits, most = most_groups(256) / nb;
    int64_t keys = ((int64_t)a.lk + 127) / 128;
    if (keys > most) keys = most;
    if (keys == 0) return R97Q_OK;
    if constexpr (D > 64) {  // narrower heads' dS is not kept
        if (a.ds) {
            hipLaunchKernelGGL((attn_dkdv_kernel<D, RT, 4, KEPT, PER, SLOTS, true>), dim3((unsigned)(keys * nb)), dim3(256), 0, st, a);
            return launch_status("attn_dkdv_kernel");
        }
    }
    hipLaunchKernelGGL((attn_dkdv_kernel<D, RT, 4, KEPT, PER, SLOTS, false>), dim3((unsigned)(keys * nb)), dim3(256), 0, st, a);
    return launch_status("attn_dkdv_kernel");
}

}  // namespace

#if R97Q_WIDE
int launch_dkdv_wide(const Args& a, hipStream_t st) { return run<256, 32, false, 1, 2>(a, st); }
#else
int launch_dkdv(const Args& a, hipStream_t st) { return a.d <= 64 ? run<64, 64, true, 2, 3>(a, st) : run<128, 64, true, 1, 3>(a, st); }
#endif

}  // namespace attn
}  // namespace r97q
