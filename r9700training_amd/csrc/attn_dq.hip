// attn_dq.hip -- attention's backward pass: dQ, D and the sums of partial results. The probabilities are recomputed from the
// log-sum-exp L:
//   P = exp(scale Q K^T - L)    D_i = sum_d dO_id O_id    dS = P o (dO V^T - D)
//   dV = P^T dO    dQ = scale dS K    dK = scale dS^T Q,  dK and dV summed over the heads that share a key head.
//
// One launch walks the keys for tiles of rows, another the rows for tiles of keys, so every sum has one owner and a fixed
// order, and repeated calls give the same bits. Two ways:
//   recomputed  attn_dq_kernel (dQ, and D for the other), then attn_dkdv_kernel: both form P and dO V^T, seven products
//   kept        attn_base_kernel (D), attn_dkdv_kernel, which writes dS^T out as it goes, attn_dq_kept_kernel: five
// Which, and in how many cuts, is decided beside the entry. P and dS are rounded to bf16 for their products (off by at most
// 2^-8 relative, each term of a sum on its own), everything else is f32.
#include "attn.h"
#include "status.h"

namespace r97q {
namespace attn {
namespace {

// ---------------------------------------------------------------- dQ (and D): 32 NW rows a workgroup
// The waves walk the keys together, 32 at a time. Step j of a wave: dO V_j^T beside the exponentials of the scores j,
// the scores j + 1 beside dS_j, then dQ += dS_j K_j. At its top the values up to j + 1 and the keys up to j + 2 have
// landed, and the slots of the values j - 1 and the keys j - 1 are free for the next loads. Every product's LDS operand
// is read kAhead products before it, the first ones of step j + 1 in step j.
// Bound like the forward: 8 x 2048 tokens causal, 16 over 4 heads of 64 127 us (810 TFLOP/s of the three products; the matrix cores
// busy 38% of the cycles, vector instructions 42%), of 128 240 us (860; 42% and 29%, a wave waits 38% of its time). Tiles of 32
// keys: a wave holds its queries, dO and sums, 2 D registers a lane, and has no room for more scores.
template <int D, int NW, int PER>
__global__ __launch_bounds__(64 * NW, PER) void attn_dq_kernel(Args a) {
    using T = Tile<D>;
    using F = Frags<D>;
    constexpr int KT = 32, TB = KT * T::RB, n = D / 16;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[7 * TB];  // keys' four slots, then the values' three
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, h = lane >> 5;
    const int nb = a.batch * a.hk;
    const Place place(nb, a.together);
    const int bh = place.bh, hk = bh % a.hk, part = place.part;
    const int tiles = gridDim.x / (nb * a.q_splits), split = part % a.q_splits;
    const Seq s = sequence(a, bh / a.hk);
    const int rows = s.lq * a.g;
    const float sl = back_scale(a), out_of_sight = sl > 0.0f ? -INFINITY : INFINITY;
    const uint8_t* kb = kv_at(a.k, a, s, hk);
    const uint8_t* vb = kv_at(a.v, a, s, hk);
    const int64_t kts = 2 * a.k.ts, vts = 2 * a.v.ts;
    const uint32_t at = lds_at(lds), mine = at + 1024 * wave, rat = at + F::row0(lane), cat = at + F::col0(lane);
    for (int64_t tile = tiles - 1 - part / a.q_splits; tile * 32 * NW < rows; tile += tiles) {
        const int t_ = fresh_lane(tid);  // not held over the results' stores
        const Loader<D, KT, 64 * NW> kl(kts, a.d, t_), vl(vts, a.d, t_);
        const int w0 = (int)tile * 32 * NW, r0 = w0 + 32 * wave, r = r0 + col;
        const int rr = r < rows ? r : rows - 1, tok = rr / a.g, head = hk * a.g + (rr - tok * a.g);
        const int wend = w0 + 32 * NW - 1 < rows ? w0 + 32 * NW - 1 : rows - 1;
        const Keys all = keys_of(a, s, w0 / a.g, wend / a.g);
        const int rend = r0 + 31 < rows ? r0 + 31 : rows - 1;
        const Keys own = keys_of(a, s, (r0 < rows ? r0 : rows - 1) / a.g, rend / a.g);
        int lo = all.lo, hi = all.hi;
        if (a.q_splits > 1 && lo < hi) {  // this range's tiles
            const int nt = (hi - lo + KT - 1) / KT, from = (int)((int64_t)nt * split / a.q_splits), to = (int)((int64_t)nt * (split + 1) / a.q_splits);
            hi = to * KT < hi - lo ? lo + to * KT : hi;
            lo += from * KT;
        }
        Rows kr(kb, kts, lo, hi, a.d), vr(vb, vts, lo, hi, a.d);
        if (lo < hi) {
            kl.load(kr, mine);
            kr.step(KT);
        }
        int d = fresh(a.d);
        bf16x8 q[n], go[n];
        load_row<D>(q_at(a.q, a, s, head) + 2 * (tok * a.q.ts), r < rows, d, lane, q);
        settle(q);
        load_row<D>(q_at(a.d_o, a, s, head) + 2 * (tok * a.d_o.ts), r < rows, d, lane, go);
        settle(go);
        const uint8_t* op = q_at(a.o, a, s, head) + (a.o.f32 ? 4 : 2) * (tok * a.o.ts);
        float delta = 0.0f;
#pragma unroll
        for (int c = 0; c < n; ++c) {
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
        const int64_t st = stat_at(a, s, head, tok);
        const float lse = a.lse[st], base = lse == -INFINITY ? 0.0f : lse * kLog2e;
        if (r < rows && h == 0 && split == 0) {
            a.base[st] = base;
            a.delta[st] = -delta;
        }
        const int first = a.window ? (int)clamp64((int64_t)tok + s.off - a.window + 1, 0, s.lk) : 0;
        const int last = a.causal && tok + s.off < s.lk - 1 ? tok + s.off : s.lk - 1;
        const uint32_t many = last < first ? 0u : (uint32_t)(last - first) + 1u;
        f32x16 dq[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dq[i] = (f32x16){};
        if (lo < hi) {
            const int nt = (hi - lo + KT - 1) / KT;
            auto load_k = [&](uint32_t to) {
                kl.load(kr, mine + to);
                kr.step(KT);
            };
            auto load_v = [&](uint32_t to) {
                vl.load(vr, mine + 4 * TB + to);
                vr.step(KT);
            };
            load_k(TB);
            load_v(0);
            load_k(2 * TB);
            load_v(TB);
            landed();
            __syncthreads();
            f32x16 x0 = {}, x1 = {};
            auto product = [&](f32x16& x, uint32_t from) {
                bf16x8 f[kAhead];
                steps<kAhead>([&](auto i) { f[i] = F::template rows<0, i>(from); });
                steps<n>([&](auto i) {
                    const bf16x8 now = f[i % kAhead];
                    if constexpr (i + kAhead < n) f[i % kAhead] = F::template rows<0, i + kAhead>(from);
                    x = mfma(now, q[i], i == 0 ? (f32x16){} : x);
                });
            };
            product(x0, rat);
            bf16x8 f[kAhead];
            steps<kAhead>([&](auto i) { f[i] = F::template rows<0, i>(rat + 4 * TB); });
            uint32_t k0 = 0, k1 = TB, k2 = 2 * TB, k3 = 3 * TB, v0 = 0, v1 = TB, v2 = 2 * TB;  // slots of tiles j, j + 1, ..
            auto step = [&](f32x16& x, f32x16& next, int j) {
                landed();
                __syncthreads();
                const int j0 = lo + j * KT;
                if (j0 < own.all_lo || j0 + KT > own.all_hi) {
                    asm volatile("");  // a branch: most tiles need no mask
                    const uint32_t from = (uint32_t)(j0 + 4 * h - first);
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = from + (uint32_t)(8 * (e >> 2) + (e & 3)) < many ? x[e] : out_of_sight;
                }
                f32x16 y = {};
                u32x4 ds[2];
                const uint32_t vat = rat + 4 * TB + v0, kat = rat + k1, dat = cat + k0, next_vat = rat + 4 * TB + v1;
                // operand of product i: V rows, next K rows, K columns, the next step's V rows
                auto frag = [&](auto i) {
                    if constexpr (i < n) return F::template rows<0, i>(vat);
                    else if constexpr (i >= 3 * n) return F::template rows<0, i - 3 * n>(next_vat);
                    else if constexpr (i < 2 * n) return F::template rows<0, i - n>(kat);
                    else return F::template cols<16 * ((i - 2 * n) / (D / 32)), (i - 2 * n) % (D / 32)>(dat);
                };
                steps<3 * n>([&](auto i) {
                    pin();
                    const bf16x8 now = f[i % kAhead];
                    f[i % kAhead] = frag(std::integral_constant<int, i + kAhead>{});
                    if constexpr (i == 0) load_k(k3);
                    if constexpr (i == 1) load_v(v2);
                    if constexpr (i < n) {
                        y = mfma(now, go[i], y);
                    } else if constexpr (i < 2 * n) {
                        next = mfma(now, q[i - n], i == n ? (f32x16){} : next);
                    } else {
                        constexpr int c = (i - 2 * n) / (D / 32), m = (i - 2 * n) % (D / 32);
                        dq[m] = mfma(now, as_bf16x8(ds[c]), dq[m]);
                    }
                    // vector work, spread: the exponentials, and from two products after y's last one dS
#pragma unroll
                    for (int e = pair_from(i, 0, n); e < pair_from(i + 1, 0, n); ++e) x[e] = __builtin_amdgcn_exp2f(x[e] * sl - base);
#pragma unroll
                    for (int e = pair_from(i, n + 2, n - 3 + D / 32); e < pair_from(i + 1, n + 2, n - 3 + D / 32); e += 2) {
                        x[e] *= y[e] - delta;
                        x[e + 1] *= y[e + 1] - delta;
                        pack_two(x, e, ds);
                    }
                });
                pin();
                const uint32_t k = k0, v = v0;
                k0 = k1, k1 = k2, k2 = k3, k3 = k;
                v0 = v1, v1 = v2, v2 = v;
            };
            for (int j = 0; j < nt; j += 2) {
                step(x0, x1, j);
                if (j + 1 < nt) step(x1, x0, j + 1);
            }
            landed();
        }
        d = fresh(a.d);
        const int hs = fresh_lane(h);
        if (a.q_splits > 1) {
            uint8_t* out = reinterpret_cast<uint8_t*>(a.dq_part + (split * a.slots + st) * d);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) store_block(out, true, r < rows, 32 * i, d, hs, dq[i], 1.0f);
            __syncthreads();
            continue;
        }
        uint8_t* out = q_at(a.dq, a, s, head) + (a.dq.f32 ? 4 : 2) * (tok * a.dq.ts);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) store_block(out, a.dq.f32, r < rows, 32 * i, d, hs, dq[i], a.scale);
        __syncthreads();
    }
}

// ---------------------------------------------------------------- D alone
// D and the log-sum-exp in base 2 for dK's and dV's launch, where that one goes first. grid (batch * q heads, tokens):
// d / 8 threads a row, rounded up to a power of two, kBaseRows rows each, so that their loads go out together. Bound by
// memory: 8 x 2048 tokens, 16 heads of 256 46 us (5.8 TB/s; 72 a row at a time).
constexpr int kBaseRows = 4;
template <bool F32>
__global__ __launch_bounds__(256) void attn_base_kernel(Args a, int lanes) {
    const int head = blockIdx.x % a.hq, rows = 256 / lanes, c = 8 * (threadIdx.x % lanes), cc = c < a.d ? c : 0;
    const Seq s = sequence(a, blockIdx.x / a.hq);
    const uint8_t *ob = q_at(a.o, a, s, head), *gb = q_at(a.d_o, a, s, head);
    const int each = rows * kBaseRows;
    for (int64_t t0 = (int64_t)blockIdx.y * each; t0 < s.lq; t0 += (int64_t)gridDim.y * each) {
        const int64_t t1 = t0 + threadIdx.x / lanes;
        u32x4 g[kBaseRows], o[kBaseRows][F32 ? 2 : 1];
        float lse[kBaseRows];
#pragma unroll
        for (int i = 0; i < kBaseRows; ++i) {
            const int64_t t = t1 + i * rows < s.lq ? t1 + i * rows : s.lq - 1;
            g[i] = *reinterpret_cast<const u32x4*>(gb + 2 * (t * a.d_o.ts + cc));
            const uint8_t* row = ob + (F32 ? 4 : 2) * (t * a.o.ts + cc);
            o[i][0] = *reinterpret_cast<const u32x4*>(row);
            if constexpr (F32) o[i][1] = *reinterpret_cast<const u32x4*>(row + 16);
            lse[i] = a.lse[stat_at(a, s, head, (int)t)];
        }
#pragma unroll
        for (int i = 0; i < kBaseRows; ++i) {
            const bf16x8 x = as_bf16x8(g[i]);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (F32)
                    sum += __builtin_bit_cast(float, (uint32_t)o[i][j / 4][j % 4]) * (float)x[j];
                else
                    sum += (float)as_bf16x8(o[i][0])[j] * (float)x[j];
            }
            if (c >= a.d) sum = 0.0f;
            for (int k = lanes / 2; k > 0; k >>= 1) sum += __shfl_xor(sum, k);
            const int64_t t = t1 + i * rows;
            if (t < s.lq && c == 0) {
                const int64_t at = stat_at(a, s, head, (int)t);
                a.base[at] = lse[i] == -INFINITY ? 0.0f : lse[i] * kLog2e;
                a.delta[at] = -sum;
            }
        }
    }
}

// ---------------------------------------------------------------- dQ from the kept dS
// dQ^T = scale K^T dS^T for 128 tokens of a query head: 32 of them a wave. The keys and dS^T's rows of the same keys go
// through two slots of LDS, both read transposed. dS^T is written for blocks of 128 keys and RT tokens where any
// of them sees any; a wave passes over the others. No mask: an unseen pair's dS is zero.
// Twice its floor, and what holds it is not known: 8 x 2048 tokens causal, 16 over 4 heads of 256 207 us (660 TFLOP/s and 2.7
// TB/s of dS^T; the matrix cores are busy 30% of the cycles, a wave waits 60% of its time); 4 x 2048, heads of 128 75 us (460 and
// 3.6).
template <int D, int KT, int PER, int RT>
__global__ __launch_bounds__(256, PER) void attn_dq_kept_kernel(Args a) {
    using F = Frags<D>;
    using S = Frags<128>;  // rows of 128 tokens
    constexpr int TB = KT * 2 * D, SB = KT * 256, SLOT = TB + SB, n = (KT / 16) * (D / 32);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * SLOT];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, h = lane >> 5;
    // the query heads of a key head one beside the other
    const int nb = a.batch * a.hk;
    const Place place(nb, a.together);
    const int bh = place.bh, hk = bh % a.hk, parts = gridDim.x / nb, tiles = parts / a.g, head = hk * a.g + place.part % a.g;
    const Seq s = sequence(a, bh / a.hk);
    const uint8_t* kb = kv_at(a.k, a, s, hk);
    const int64_t kts = 2 * a.k.ts;
    const uint32_t at = lds_at(lds), mine = at + 1024 * wave, kat = at + F::col0(lane), sat = (at + TB + S::col0(lane)) ^ (64 * wave);
    for (int64_t tile = tiles - 1 - place.part / a.g; tile * 128 < s.lq; tile += tiles) {
        const int t_ = fresh_lane(tid);
        const Loader<D, KT, 256> kl(kts, a.d, t_);
        const Loader<128, KT, 256> sl(2 * a.pitch, 128, t_);
        const int w0 = (int)tile * 128, r0 = w0 + 32 * wave, wend = w0 + 127 < s.lq ? w0 + 127 : s.lq - 1;
        const Keys all = keys_of(a, s, w0, wend);
        const int lo = all.lo / 128 * 128, hi = all.hi;
        Rows kr(kb, kts, lo, hi, a.d), sr(reinterpret_cast<const uint8_t*>(ds_at(a, s, head, 0) + w0), 2 * a.pitch, lo, hi, 128);
        f32x16 dq[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dq[i] = (f32x16){};
        auto load = [&](int slot) {
            kl.load(kr, mine + slot * SLOT);
            sl.load(sr, mine + slot * SLOT + TB);
            kr.step(KT);
            sr.step(KT);
        };
        if (lo < hi) load(0);
        bool seen = false;
        auto step = [&](int j0, auto slot_) {
            constexpr int slot = slot_;
            landed();
            __syncthreads();
            load(1 - slot);
            if (j0 < all.lo) {  // keys before the first that is seen, in its block: they may hold anything, also in dS^T
                const int none = all.lo - j0 < KT ? all.lo - j0 : KT;
                for (int i = 16 * tid; i < none * 2 * D; i += 16 * 256) *reinterpret_cast<u32x4*>(lds + slot * SLOT + i) = (u32x4){};
                for (int i = 16 * tid; i < none * 256; i += 16 * 256) *reinterpret_cast<u32x4*>(lds + slot * SLOT + TB + i) = (u32x4){};
                __syncthreads();
            }
            if ((j0 & 127) == 0) {
                int t0, t1;
                tokens_of(a, s, j0, RT, t0, t1);
                seen = t0 < t1 && r0 + 32 > t0 && r0 < (t1 + RT - 1) / RT * RT && r0 < s.lq;
            }
            if (!seen) return;
            bf16x8 f[kAhead], g[KT / 16];
            auto frag = [&](auto i) { return F::template cols<16 * (i / (D / 32)) + slot * (SLOT / (2 * D)), i % (D / 32)>(kat); };
            steps<KT / 16>([&](auto i) { g[i] = S::template cols<16 * i + slot * (SLOT / 256), 0>(sat); });
            steps<kAhead>([&](auto i) { f[i] = frag(i); });
            steps<n>([&](auto i) {
                pin();
                const bf16x8 now = f[i % kAhead];
                if constexpr (i + kAhead < n) f[i % kAhead] = frag(std::integral_constant<int, i + kAhead>{});
                dq[i % (D / 32)] = mfma(now, g[i / (D / 32)], dq[i % (D / 32)]);
            });
            pin();
        };
        for (int j0 = lo; j0 < hi; j0 += 2 * KT) {
            step(j0, std::integral_constant<int, 0>{});
            if (j0 + KT < hi) step(j0 + KT, std::integral_constant<int, 1>{});
        }
        landed();
        const int t = r0 + col, d = fresh(a.d), hs = fresh_lane(h);
        uint8_t* out = q_at(a.dq, a, s, head) + (a.dq.f32 ? 4 : 2) * ((int64_t)t * a.dq.ts);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) store_block(out, a.dq.f32, t < s.lq, 32 * i, d, hs, dq[i], a.scale);
        __syncthreads();
    }
}

// ---------------------------------------------------------------- partial sums added
// grid (batch * heads, tokens, tensors): a row's partial sums in order, times the tensor's factor, to the output. A thread
// takes four columns of kSumRows rows, and four parts at once, so that their loads go out together. dK's and dV's three parts
// of some 3400 tokens, 4 heads of 128: 13 us for 55 MB (4.2 TB/s).
constexpr int kSumRows = 2;
struct Sum {
    Heads out[2];
    const float* part[2];
    float factor[2];
    int32_t splits;
    bool keys;  // rows of dK and dV, else of dQ
};
__global__ __launch_bounds__(256) void attn_sum_kernel(Args a, Sum u) {
    const bool keys = u.keys;
    const int heads = keys ? a.hk : a.hq, head = blockIdx.x % heads, which = blockIdx.z;
    const Heads out = u.out[which];
    const float* part = u.part[which];
    const float f = u.factor[which];
    const Seq s = sequence(a, blockIdx.x / heads);
    const int per = a.d / 4, rows = 256 / per, r = threadIdx.x / per, c = 4 * (threadIdx.x % per);
    const int cover = !keys ? s.lq : a.kv_starts ? s.lk : a.lk;
    const int64_t slots = keys ? a.kv_slots : a.slots;
    if (r >= rows) return;
    const int each = rows * kSumRows;
    for (int64_t t0 = (int64_t)blockIdx.y * each + r; t0 < cover; t0 += (int64_t)gridDim.y * each) {
        int64_t at[kSumRows];
        float4 v[kSumRows];
#pragma unroll
        for (int j = 0; j < kSumRows; ++j) {
            const int t = (int)(t0 + j * rows < cover ? t0 + j * rows : t0);
            at[j] = (keys ? kv_slot(a, s, head, t) : stat_at(a, s, head, t)) * a.d + c;
            v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        for (int i = 0; i < u.splits; i += 4) {
            float4 w[kSumRows][4];
#pragma unroll
            for (int j = 0; j < kSumRows; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) w[j][k] = *reinterpret_cast<const float4*>(part + (i + k < u.splits ? i + k : i) * slots * a.d + at[j]);
#pragma unroll
            for (int j = 0; j < kSumRows; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (i + k < u.splits) v[j].x += w[j][k].x, v[j].y += w[j][k].y, v[j].z += w[j][k].z, v[j].w += w[j][k].w;
        }
#pragma unroll
        for (int j = 0; j < kSumRows; ++j) {
            const int64_t t = t0 + j * rows;
            if (t >= cover) continue;
            uint8_t* row = (keys ? kv_at(out, a, s, head) : q_at(out, a, s, head)) + (out.f32 ? 4 : 2) * (t * out.ts);
            if (out.f32)
                *reinterpret_cast<float4*>(row + 4 * c) = make_float4(v[j].x * f, v[j].y * f, v[j].z * f, v[j].w * f);
            else
                *reinterpret_cast<uint2*>(row + 2 * c) = make_uint2(pack_bf16(v[j].x * f, v[j].y * f), pack_bf16(v[j].z * f, v[j].w * f));
        }
    }
}

template <int D, int PER>
int run(const Args& a, hipStream_t st) {
    const int64_t nb = (int64_t)a.batch * a.hk * a.q_splits, most = most_groups(256) / nb;
    int64_t tiles = ((int64_t)a.lq * a.g + 127) / 128;
    if (tiles > most) tiles = most;
    if (tiles == 0) return R97Q_OK;
    hipLaunchKernelGGL((attn_dq_kernel<D, 4, PER>), dim3((unsigned)(tiles * nb)), dim3(256), 0, st, a);
    return launch_status("attn_dq_kernel");
}

}  // namespace

int launch_sums(const Args& a, bool keys, hipStream_t st) {
    const int64_t tokens = keys ? a.lk : a.lq, each = 256 / (a.d / 4) * kSumRows, blocks = (tokens + each - 1) / each;
    if (blocks == 0) return R97Q_OK;
    Sum u = {{keys ? a.dk : a.dq, a.dv}, {keys ? a.dk_part : a.dq_part, a.dv_part}, {a.scale, 1.0f}, keys ? a.k_splits : a.q_splits, keys};
    hipLaunchKernelGGL(attn_sum_kernel, dim3((unsigned)(a.batch * (keys ? a.hk : a.hq)), (unsigned)(blocks < 65535 ? blocks : 65535), keys ? 2 : 1),
                       dim3(256), 0, st, a, u);
    return launch_status("attn_sum_kernel");
}

int launch_base(const Args& a, hipStream_t st) {
    const int lanes = a.d <= 64 ? 8 : a.d <= 128 ? 16 : 32, each = 256 / lanes * kBaseRows;
    const int64_t blocks = ((int64_t)a.lq + each - 1) / each;
    if (blocks == 0) return R97Q_OK;
    const dim3 grid((unsigned)(a.batch * a.hq), (unsigned)(blocks < 65535 ? blocks : 65535));
    if (a.o.f32)
        hipLaunchKernelGGL(attn_base_kernel<true>, grid, dim3(256), 0, st, a, lanes);
    else
        hipLaunchKernelGGL(attn_base_kernel<false>, grid, dim3(256), 0, st, a, lanes);
    return launch_status("attn_base_kernel");
}

template <int D, int KT, int PER, int RT>
int run_kept(const Args& a, hipStream_t st) {
    const int64_t nb = (int64_t)a.batch * a.hq, most = most_groups(256) / nb;
    int64_t tiles = ((int64_t)a.lq + 127) / 128;
    if (tiles > most) tiles = most;
    if (tiles == 0) return R97Q_OK;
    hipLaunchKernelGGL((attn_dq_kept_kernel<D, KT, PER, RT>), dim3((unsigned)(tiles * nb)), dim3(256), 0, st, a);
    return launch_status("attn_dq_kept_kernel");
}
int launch_dq_kept(const Args& a, hipStream_t st) {
    return a.d <= 128 ? run_kept<128, 64, 2, 64>(a, st) : run_kept<256, 32, 2, 32>(a, st);
}

int launch_dq(const Args& a, hipStream_t st) { return a.d <= 64 ? run<64, 2>(a, st) : a.d <= 128 ? run<128, 2>(a, st) : run<256, 1>(a, st); }

}  // namespace attn
}  // namespace r97q
