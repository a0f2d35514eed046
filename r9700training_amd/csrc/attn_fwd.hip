// attn_fwd.hip -- attention's forward: O = softmax(scale Q K^T + mask) V and each row's log-sum-exp.
//
// One pass over the keys with a running maximum and sum (in f32), per row:
//   m' = max(m, max_j s_j),  l' = l e^(m - m') + sum_j e^(s_j - m'),  O' = O e^(m - m') + sum_j e^(s_j - m') v_j
// and O / l, m + ln l at the end. m need not be the maximum, only near it: it moves when some row's maximum has
// passed it by more than a factor of 2^8, so most tiles rescale nothing (f32 has the room, and a bf16
// probability the same relative precision at any size). The probabilities are rounded to bf16 for the second
// product (the matrix cores' input type; off by at most 2^-8 relative), their sum is of the unrounded values in f32.
#include "attn.h"
#include "status.h"

namespace r97q {
namespace attn {
namespace {

constexpr float kLoose = 8.0f;  // how far, in powers of two, a maximum may pass m before m moves

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

// the natural log-sum-exp of a sum l relative to 2^m; nothing summed: minus infinity
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2; }

// 32 rows' running state: a lane's query is column lane % 32, shared with lane ^ 32
template <int D>
struct Running {
    f32x16 o[D / 32];
    float m, l;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] = (f32x16){};
        m = -INFINITY;
        l = 0.0f;
    }
    // m moves where a maximum passed it (top: this tile's, times the scale)
    __device__ __forceinline__ void rise(float top) {
        if (__builtin_amdgcn_ballot_w64(top > m + kLoose) == 0) return;
        const float m1 = fmaxf(m, top);
        const float turn = __builtin_amdgcn_exp2f(m - (m1 == -INFINITY ? 0.0f : m1));
        m = m1;
        l *= turn;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] *= turn;
    }
};

// S^T tiles of KT keys against 32 rows
template <int D, int KT>
__device__ __forceinline__ void scores(const uint8_t* kt, const bf16x8 (&q)[D / 16], int lane, f32x16 (&x)[KT / 32]) {
#pragma unroll
    for (int i = 0; i < KT / 32; ++i) x[i] = (f32x16){};
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int i = 0; i < KT / 32; ++i) x[i] = mfma(Tile<D>::rows(kt, 32 * i, c, lane), q[c], x[i]);
}
// keys outside [first, last], counted from the tile's first, to minus infinity (one comparison a key: the
// distance from the first, unsigned, against how many there are)
template <int KT>
__device__ __forceinline__ void mask(f32x16 (&x)[KT / 32], int first, int last, int h) {
    const uint32_t many = last < first ? 0u : (uint32_t)(last - first) + 1u;
#pragma unroll
    for (int i = 0; i < KT / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const uint32_t j = (uint32_t)(4 * h - first) + (uint32_t)(32 * i + 8 * (e >> 2) + (e & 3));
            x[i][e] = j < many ? x[i][e] : -INFINITY;
        }
}
template <int KT>
__device__ __forceinline__ float tile_max(const f32x16 (&x)[KT / 32]) {
    float t[KT / 32];
#pragma unroll
    for (int i = 0; i < KT / 32; ++i) {
        t[i] = x[i][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) t[i] = fmaxf(t[i], x[i][e]);
    }
#pragma unroll
    for (int i = 1; i < KT / 32; ++i) t[0] = fmaxf(t[0], t[i]);
    return pair_max(t[0]);
}
// probabilities of a tile's scores, their sum into r.l, and their product with the values into r.o
template <int D, int KT>
__device__ __forceinline__ void absorb(const uint8_t* vt, f32x16 (&x)[KT / 32], float sl, int lane, Running<D>& r) {
    const float base = r.m == -INFINITY ? 0.0f : r.m;
    bf16x8 p[KT / 16];
    float sum[KT / 32];
#pragma unroll
    for (int i = 0; i < KT / 32; ++i) {
        sum[i] = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            x[i][e] = __builtin_amdgcn_exp2f(x[i][e] * sl - base);
            sum[i] += x[i][e];
        }
        bf16x8 two[2];
        pack_tile(x[i], two);
        p[2 * i] = two[0];
        p[2 * i + 1] = two[1];
#pragma unroll
        for (int c = 2 * i; c < 2 * i + 2; ++c)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) r.o[d] = mfma(Tile<D>::cols(vt, 16 * c, d, lane), p[c], r.o[d]);
    }
#pragma unroll
    for (int i = 0; i < KT / 32; ++i) r.l += sum[i];
}

// a row's place
struct Row {
    int tok, head;
    bool on;
    __device__ __forceinline__ Row(const Args& a, int hk, int r, int rows) {
        const int rr = r < rows ? r : rows - 1;
        tok = rr / a.g;
        head = hk * a.g + (rr - tok * a.g);
        on = r < rows;
    }
};

template <int D>
__device__ __forceinline__ void finish(const Args& a, const Seq& s, const Row& row, int h, int split, const Running<D>& r, float l) {
    const int d = fresh(a.d);
    h = fresh_lane(h);
    if (a.splits > 1) {
        const int64_t at = split * a.slots + stat_at(a, s, row.head, row.tok);
        uint8_t* out = reinterpret_cast<uint8_t*>(a.part + at * d);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) store_block(out, true, row.on, 32 * i, d, h, r.o[i], 1.0f);
        if (row.on && h == 0) a.stats[at] = make_float2(r.m, l);
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint8_t* out = q_at(a.o, a, s, row.head) + (a.o.f32 ? 4 : 2) * (row.tok * a.o.ts);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) store_block(out, a.o.f32, row.on, 32 * i, d, h, r.o[i], inv);
    if (row.on && a.lse && h == 0)
        a.lse[stat_at(a, s, row.head, row.tok)] = log_sum(r.m, l);
}

// ---------------------------------------------------------------- tiles of 32 NW rows
// A workgroup's NW waves take 32 rows each of one key head's rows and walk the keys together, KT at a time, from
// LDS. Step j of a wave: the products of the scores j + 1, then those of P_j V_j; beside them, spread evenly, the
// maximum of the scores j and their exponentials, each half a k step ahead of its use. At the step's top the keys
// of tile j + 1 and the values of tile j have landed, and both of tile j - 1's slots are free for the loads of tiles
// j + 2 and j + 1. Every LDS operand is read kAhead products before its use.
//
// Bound by products and vector instructions that two waves a SIMD overlap in part: a step at 128 columns is 32 products of 32
// cycles among some 190 vector, 48 LDS and 50 scalar instructions. Counted over 8 x 2048 tokens causal, 32 over 8 heads of
// 128: the matrix cores are busy 48% of the cycles, vector instructions at 4 cycles each make 35%, a wave waits (for loads,
// LDS, the barrier) 23% of its time, no LDS bank conflicts, 1.9 GHz. 64 keys a tile (32 at 256 columns, where a wave's sums
// and queries fill its registers and one wave a SIMD remains: 33% and 20%): 302 .. 312 us, 880 .. 910 TFLOP/s; 16 over 4 heads
// of 256 350 .. 390 us, 705 .. 785; of 64 94 .. 100 us, 690 .. 730 (32% and 45%, 11 vector instructions a product). Two waves
// that share 32 rows and halve their keys were 6 .. 10% faster on grids of under 256 workgroups only, and are not built.
template <int D, int KT, int NW, int PER>
__global__ __launch_bounds__(64 * NW, PER) void attn_fwd_kernel(Args a) {
    using T = Tile<D>;
    using F = Frags<D>;
    constexpr int TB = KT * T::RB, SUBS = KT / 32, n = D / 16;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * TB];  // keys' two slots, then the values'
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, h = lane >> 5;
    const int nb = a.batch * a.hk;
    const Place place(nb, a.together);
    const int bh = place.bh, hk = bh % a.hk, part = place.part;
    const int tiles = gridDim.x / (nb * a.splits), split = part % a.splits;
    const Seq s = sequence(a, bh / a.hk);
    const int rows = s.lq * a.g;
    const float sl = score_scale(a);
    const uint8_t* kb = kv_at(a.k, a, s, hk);
    const uint8_t* vb = kv_at(a.v, a, s, hk);
    const int64_t kts = 2 * a.k.ts, vts = 2 * a.v.ts;
    const Loader<D, KT, 64 * NW> kl(kts, a.d, tid), vl(vts, a.d, tid);
    const uint32_t at = lds_at(lds), mine = at + 1024 * wave, rat = at + F::row0(lane), cat = at + 2 * TB + F::col0(lane);
    // the last tiles first: under a causal mask they have the most keys
    for (int64_t tile = tiles - 1 - part / a.splits; tile * 32 * NW < rows; tile += tiles) {
        const int w0 = (int)tile * 32 * NW, r0 = w0 + 32 * wave;
        const Row row(a, hk, r0 + col, rows);
        const int wend = w0 + 32 * NW - 1 < rows ? w0 + 32 * NW - 1 : rows - 1;
        const Keys all = keys_of(a, s, w0 / a.g, wend / a.g);
        const int rend = r0 + 31 < rows ? r0 + 31 : rows - 1;
        Keys own = keys_of(a, s, (r0 < rows ? r0 : rows - 1) / a.g, rend / a.g);
        if (r0 >= rows) own.hi = own.lo;
        int lo = all.lo, hi = all.hi;  // from the first key that is seen: what lies before it may hold anything
        if (a.splits > 1) {
            lo = (int)clamp64((int64_t)lo + (int64_t)split * a.chunk, lo, hi);
            if (split < a.splits - 1 && hi - lo > a.chunk) hi = lo + a.chunk;  // the last range takes what is left
        }
        Rows kr(kb, kts, lo, hi, a.d), vr(vb, vts, lo, hi, a.d);
        auto load_k = [&](int slot) {
            kl.load(kr, mine + slot * TB);
            kr.step(KT);
        };
        auto load_v = [&](int slot) {
            vl.load(vr, mine + (2 + slot) * TB);
            vr.step(KT);
        };
        if (lo < hi) {
            load_k(0);
            load_k(1);
            load_v(0);
        }
        bf16x8 q[n];
        load_row<D>(q_at(a.q, a, s, row.head) + 2 * (row.tok * a.q.ts), row.on, fresh(a.d), lane, q);
        turn_sign<D>(a, q);
        settle(q);
        // the keys this lane's row sees, first and last
        const int first = a.window ? (int)clamp64((int64_t)row.tok + s.off - a.window + 1, 0, s.lk) : 0;
        const int last = a.causal && row.tok + s.off < s.lk - 1 ? row.tok + s.off : s.lk - 1;
        Running<D> run;
        run.clear();
        if (lo < hi) {
            const int end = own.hi < hi ? own.hi : hi;
            // tiles this wave looks at: [n0, n1) of nt
            const int nt = (hi - lo + KT - 1) / KT, n0 = own.lo > lo ? (own.lo - lo) / KT : 0, n1 = end > lo ? (end - lo + KT - 1) / KT : 0;
            landed();
            __syncthreads();
            f32x16 x0[SUBS], x1[SUBS];
            constexpr int NA = SUBS * n, NB = 2 * SUBS * (D / 32);
            auto only_scores = [&](f32x16 (&x)[SUBS], uint32_t from) {
                bf16x8 f[kAhead];
                steps<kAhead>([&](auto i) { f[i] = F::template rows<32 * (i % SUBS), i / SUBS>(from); });
                steps<NA>([&](auto i) {
                    const bf16x8 now = f[i % kAhead];
                    if constexpr (i + kAhead < NA) f[i % kAhead] = F::template rows<32 * ((i + kAhead) % SUBS), (i + kAhead) / SUBS>(from);
                    x[i % SUBS] = mfma(now, q[i / SUBS], i < SUBS ? (f32x16){} : x[i % SUBS]);
                });
            };
            only_scores(x0, rat);
            auto step = [&](f32x16 (&x)[SUBS], f32x16 (&xn)[SUBS], int j, auto slot_) {
                constexpr int slot = slot_;
                if (j > 0) {  // the first tiles' loads are the ones above
                    landed();
                    __syncthreads();
                    load_k(slot);
                    load_v(1 - slot);
                } else {
                    __syncthreads();
                    load_k(slot);
                    load_v(1 - slot);
                }
                if (j >= n0 && j < n1) {
                    const int j0 = lo + j * KT;
                    if (j0 < own.all_lo || j0 + KT > own.all_hi) mask<KT>(x, first - j0, last - j0, h);
                    bf16x8 f[kAhead];
                    // operand of product i: the next keys' rows, the values' columns
                    auto frag = [&](auto i) {
                        if constexpr (i < NA) return F::template rows<(1 - slot) * KT + 32 * (i % SUBS), i / SUBS>(rat);
                        else return F::template cols<slot * KT + 16 * ((i - NA) / (D / 32)), (i - NA) % (D / 32)>(cat);
                    };
                    steps<kAhead>([&](auto i) { f[i] = frag(i); });
                    constexpr int MX = NA / 2, EL = NA + (KT / 16 - 1) * (D / 32) - MX, pairs = KT / 4;
                    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f}, base = 0.0f;
                    u32x4 p[KT / 16];
                    steps<NA + NB>([&](auto i) {
                        if constexpr (i == MX) {
                            run.rise(pair_max(fmaxf(top[0], top[1])) * sl);
                            base = run.m == -INFINITY ? 0.0f : run.m;
                        }
                        pin();
                        const bf16x8 now = f[i % kAhead];
                        if constexpr (i + kAhead < NA + NB) f[i % kAhead] = frag(std::integral_constant<int, i + kAhead>{});
                        if constexpr (i < NA) {
                            xn[i % SUBS] = mfma(now, q[i / SUBS], i < SUBS ? (f32x16){} : xn[i % SUBS]);
                        } else {
                            constexpr int c = (i - NA) / (D / 32), m = (i - NA) % (D / 32);
                            run.o[m] = mfma(now, as_bf16x8(p[c]), run.o[m]);
                        }
                        if constexpr (i < MX) {
#pragma unroll
                            for (int e = KT / 2 * i / MX; e < KT / 2 * (i + 1) / MX; ++e) top[e & 1] = fmaxf(top[e & 1], x[e / 16][e % 16]);
                        } else {
#pragma unroll
                            for (int t = pairs * (i - MX) / EL; t < (i - MX >= EL ? pairs : pairs * (i + 1 - MX) / EL); ++t) {
                                if (i - MX >= EL) break;
                                const int e = 2 * t, u = e / 16, w = e % 16;
                                x[u][w] = __builtin_amdgcn_exp2f(x[u][w] * sl - base);
                                x[u][w + 1] = __builtin_amdgcn_exp2f(x[u][w + 1] * sl - base);
                                sum[0] += x[u][w];
                                sum[1] += x[u][w + 1];
                                p[e / 8][(e % 8) / 2] = pack_bf16(x[u][w], x[u][w + 1]);
                            }
                        }
                    });
                    pin();
                    run.l += sum[0] + sum[1];
                } else if (j + 1 == n0) {
                    only_scores(xn, rat + (1 - slot) * TB);
                }
            };
            for (int j = 0; j < nt; j += 2) {
                step(x0, x1, j, std::integral_constant<int, 0>{});
                if (j + 1 < nt) step(x1, x0, j + 1, std::integral_constant<int, 1>{});
            }
            landed();
        }
        finish<D>(a, s, row, h, split, run, pair_sum(run.l));
        __syncthreads();
    }
}

// ---------------------------------------------------------------- a few rows against many keys
// At most 32 rows of a key head (one token's query heads, or a few tokens'): nothing is shared between rows, so
// every wave takes tiles of 32 keys of its own, with its own K and V tile in LDS and no barrier: the next keys
// are loaded when the scores are done, the next values when the product is. The NW waves' sums meet in LDS.
// Bound by memory, 2 * D * 2 bytes a key: one token, 24 over 4 heads of 256, 32768 keys 28.5 us (4.7 TB/s); 16 tokens, 32
// over 8 heads of 128, caches of 1 .. 4096 keys 29.4 us (5.4 TB/s).
template <int D, int NW>
__global__ __launch_bounds__(64 * NW, 1) void attn_few_kernel(Args a) {
    using T = Tile<D>;
    constexpr int KT = 32, TB = KT * T::RB;
    __shared__ __attribute__((aligned(16))) uint8_t lds[NW * 2 * TB];
    __shared__ float2 ml[NW][32];
    static_assert(2 * TB >= 32 * D * 4, "a wave's tiles hold its sums");
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, h = lane >> 5;
    const int bh = blockIdx.x, hk = bh % a.hk, split = blockIdx.y;
    const Seq s = sequence(a, bh / a.hk);
    const int rows = s.lq * a.g;
    const float sl = score_scale(a);
    const uint8_t* kb = kv_at(a.k, a, s, hk);
    const uint8_t* vb = kv_at(a.v, a, s, hk);
    const int64_t kts = 2 * a.k.ts, vts = 2 * a.v.ts;
    const Loader<D, KT, 64> kl(kts, a.d, lane), vl(vts, a.d, lane);
    uint8_t* own = lds + wave * 2 * TB;
    const uint32_t at = lds_at(own);
    for (int64_t tile = blockIdx.z; tile * 32 < rows; tile += gridDim.z) {
        const int r0 = (int)tile * 32;
        const Row row(a, hk, r0 + col, rows);
        const int rend = r0 + 31 < rows ? r0 + 31 : rows - 1;
        const Keys keys = keys_of(a, s, r0 / a.g, rend / a.g);
        int lo = keys.lo, hi = keys.hi;
        if (a.splits > 1) {
            lo = (int)clamp64((int64_t)lo + (int64_t)split * a.chunk, lo, hi);
            if (split < a.splits - 1 && hi - lo > a.chunk) hi = lo + a.chunk;  // the last range takes what is left
            if (lo >= hi) {  // nothing in this range
                if (wave == 0 && row.on && h == 0) a.stats[split * a.slots + stat_at(a, s, row.head, row.tok)] = make_float2(-INFINITY, 0.0f);
                continue;
            }
        }
        Running<D> run;
        run.clear();
        const int first = a.window ? (int)clamp64((int64_t)row.tok + s.off - a.window + 1, 0, s.lk) : 0;
        const int last = a.causal && row.tok + s.off < s.lk - 1 ? row.tok + s.off : s.lk - 1;
        int j0 = lo + KT * wave;
        if (j0 < hi) {
            Rows kr(kb, kts, j0, hi, a.d), vr(vb, vts, j0, hi, a.d);
            kl.load(kr, at);
            vl.load(vr, at + TB);
            bf16x8 q[D / 16];
            load_row<D>(q_at(a.q, a, s, row.head) + 2 * (row.tok * a.q.ts), row.on, fresh(a.d), lane, q);
            turn_sign<D>(a, q);
            settle(q);
            landed<Loader<D, KT, 64>::N>();  // the queries have been waited for: no more than the values are left
            for (; j0 < hi; j0 += KT * NW) {
                f32x16 x[1];
                scores<D, KT>(own, q, lane, x);
                // the keys are in registers: their tile is free
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                kr.step(NW * KT);
                kl.load(kr, at);
                if (j0 < keys.all_lo || j0 + KT > keys.all_hi) mask<KT>(x, first - j0, last - j0, h);
                run.rise(tile_max<KT>(x) * sl);
                landed<Loader<D, KT, 64>::N>();  // the values; the next keys may be on their way
                absorb<D, KT>(own + TB, x, sl, lane, run);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                vr.step(NW * KT);
                vl.load(vr, at + TB);
                landed<Loader<D, KT, 64>::N>();
            }
            landed();
        }
        // the waves' sums, each in its own tiles: relative to the largest maximum, then added in wave order
        const float l = pair_sum(run.l);
        if (h == 0) ml[wave][col] = make_float2(run.m, l);
        __syncthreads();
        float top = ml[0][col].x;
#pragma unroll
        for (int w = 1; w < NW; ++w) top = fmaxf(top, ml[w][col].x);
        const float turn = __builtin_amdgcn_exp2f(run.m - (top == -INFINITY ? 0.0f : top));
        float* sum = reinterpret_cast<float*>(own);
        if (row.on) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 v = {run.o[i][4 * e] * turn, run.o[i][4 * e + 1] * turn, run.o[i][4 * e + 2] * turn, run.o[i][4 * e + 3] * turn};
                    *reinterpret_cast<float4*>(sum + col * D + 32 * i + 8 * e + 4 * h) = v;
                }
        }
        __syncthreads();
        const int n = rows - r0 < 32 ? rows - r0 : 32;
        for (int i = tid; i < n * (D / 4); i += 64 * NW) {
            const int r = i / (D / 4), d0 = 4 * (i % (D / 4));
            if (d0 >= a.d) continue;
            float t = ml[0][r].x, total = 0.0f;
#pragma unroll
            for (int w = 1; w < NW; ++w) t = fmaxf(t, ml[w][r].x);
#pragma unroll
            for (int w = 0; w < NW; ++w) total += ml[w][r].y * __builtin_amdgcn_exp2f(ml[w][r].x - (t == -INFINITY ? 0.0f : t));
            float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float4 u = *reinterpret_cast<const float4*>(lds + w * 2 * TB + 4 * (r * D + d0));
                v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
            }
            const Row rr(a, hk, r0 + r, rows);
            const int64_t st = stat_at(a, s, rr.head, rr.tok);
            if (a.splits > 1) {
                const int64_t to = split * a.slots + st;
                *reinterpret_cast<float4*>(a.part + to * a.d + d0) = v;
                if (d0 == 0) a.stats[to] = make_float2(t, total);
                continue;
            }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            uint8_t* out = q_at(a.o, a, s, rr.head) + (a.o.f32 ? 4 : 2) * (rr.tok * a.o.ts);
            if (a.o.f32)
                *reinterpret_cast<float4*>(out + 4 * d0) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
            else
                *reinterpret_cast<uint2*>(out + 2 * d0) = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
            if (d0 == 0 && a.lse) a.lse[st] = log_sum(t, total);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- the ranges' results joined
// grid (batch * q heads, tokens). Each range's sums are relative to its own m. A row of d values takes `lanes` threads
// (d / 4, rounded up to a power of two); `groups` of them share a row's ranges, kBatch at once each, so that a row's
// loads all go out together, and their sums are added in order. `rows` rows a workgroup. Bound by latency: 5.8 us for the
// 43 ranges of one token's 24 heads of 256.
constexpr int kBatch = 8;
__global__ __launch_bounds__(1024) void attn_join_kernel(Args a, int lanes, int groups, int rows) {
    __shared__ __attribute__((aligned(16))) float4 acc[1024];
    __shared__ float2 stat[1024];
    const int tid = threadIdx.x, head = blockIdx.x % a.hq, per = lanes * groups;
    const Seq s = sequence(a, blockIdx.x / a.hq);
    const int lane = tid % lanes, group = tid % per / lanes, d0 = 4 * lane;
    for (int64_t t0 = (int64_t)blockIdx.y * rows; t0 < s.lq; t0 += (int64_t)gridDim.y * rows) {
        const int64_t tok = t0 + tid / per;
        const bool on = tok < s.lq;
        const int64_t at = on ? stat_at(a, s, head, (int)tok) : 0;
        float top = -INFINITY, l = 0.0f;
        float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i0 = group; on && i0 < a.splits; i0 += kBatch * groups) {
            float2 st[kBatch];
            float4 u[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int i = i0 + k * groups < a.splits ? i0 + k * groups : i0;
                st[k] = a.stats[i * a.slots + at];
                u[k] = *reinterpret_cast<const float4*>(a.part + (i * a.slots + at) * a.d + (d0 < a.d ? d0 : 0));
            }
            float most = top;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                if (i0 + k * groups >= a.splits) st[k].x = -INFINITY;
                most = fmaxf(most, st[k].x);
            }
            const float turn = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - most);
            l *= turn, v.x *= turn, v.y *= turn, v.z *= turn, v.w *= turn;
            top = most;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                if (st[k].x == -INFINITY) continue;  // an empty range wrote no sums: its place may hold anything
                const float f = __builtin_amdgcn_exp2f(st[k].x - top);
                l += st[k].y * f;
                v.x += u[k].x * f, v.y += u[k].y * f, v.z += u[k].z * f, v.w += u[k].w * f;
            }
        }
        if (groups > 1) {
            acc[tid] = v;
            stat[tid] = make_float2(top, l);
            __syncthreads();
            if (group == 0) {
                float most = top;
                for (int i = 1; i < groups; ++i) most = fmaxf(most, stat[tid + i * lanes].x);
                l = 0.0f;
                v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int i = 0; i < groups; ++i) {
                    const float2 st = stat[tid + i * lanes];
                    if (st.x == -INFINITY) continue;
                    const float f = __builtin_amdgcn_exp2f(st.x - most);
                    const float4 u = acc[tid + i * lanes];
                    l += st.y * f;
                    v.x += u.x * f, v.y += u.y * f, v.z += u.z * f, v.w += u.w * f;
                }
                top = most;
            }
            __syncthreads();
        }
        if (!on || group || d0 >= a.d) continue;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint8_t* out = q_at(a.o, a, s, head) + (a.o.f32 ? 4 : 2) * (tok * a.o.ts);
        if (a.o.f32)
            *reinterpret_cast<float4*>(out + 4 * d0) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        else
            *reinterpret_cast<uint2*>(out + 2 * d0) = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
        if (lane == 0 && a.lse) a.lse[at] = log_sum(top, l);
    }
}

// How a shape is cut: rows a workgroup, ranges of the keys. A range writes its sums and a second launch (some 5 us) joins
// them, so only where compute units would be idle. Measured (us at 1 / 2 / 4 / 8 / 16 / 32 ranges): one token, 24 over 4
// heads of 256, 32768 keys 601 / 312 / 168 / 98 / 63 / 43 (64: 39); 16 sequences of 1 .. 4096 keys, 32 over 8 heads of 128
// 58 / 47 / 44 / 46 / 52 / 67, all of 4096 keys 45 / 49 / 49 / 50 / 54 / 72; 64 rows over 4096 keys 67 / 42 / 29 / 23 / 22 /
// 24, over 1024 keys 22 / 19 / 16 / 14 / 15; 200 rows over 2000 keys, heads of 64 28 / 21 / 16 / 14 / 15; but 1300 tokens, 16
// over 4 heads 28 / 35 / 45 / 57, and 512 tokens 15 / 20 / 22 / 30. One token, 24 over 4 heads of 256, 1024 keys 19 / 17 / 15 /
// 14 and 512 keys 14 / 15 / 14 / 13; 32 over 8 heads of 128, 1024 keys 10 / 12 / 11 / 11.
struct Plan {
    bool few;
    int splits, chunk;
    int64_t tiles;
};
Plan plan_of(const Args& a) {
    Plan p = {};
    const int64_t rows = (int64_t)a.lq * a.g;
    p.few = rows <= 32;
    const int tile = p.few ? 32 : 128;
    p.tiles = (rows + tile - 1) / tile;
    p.splits = 1;
    // the keys a tile's rows may see
    int64_t most = mean_len(a.kv_starts, a.kv_tokens, a.lk, a.batch);
    if (a.window && (int64_t)a.window + tile / a.g + 1 < most) most = (int64_t)a.window + tile / a.g + 1;
    const int64_t have = a.hk * all_tiles(a.q_starts, a.q_tokens, a.lq, a.batch, a.g, tile);
    int64_t n = 1, unit;
    if (p.few) {  // lengths that differ leave workgroups idle: more of them
        const int64_t want = !a.kv_lens && !a.kv_starts ? 192 : a.d > 128 ? 256 : 512;
        unit = 128;
        if (have > 0 && have * 3 / 2 < want && most > (a.d > 128 ? 640 : 1024)) n = (want + have - 1) / have;
    } else {
        unit = have > 16 ? 512 : most < 512 ? most + 1 : most < 1024 ? 128 : most < 4096 ? most / 8 : 512;
        if (have > 0 && have * 2 <= 256) n = (256 + have - 1) / have;
    }
    if (n > most / unit) n = most / unit;
    if (n > kMostSplits) n = kMostSplits;
    // a workgroup for each range of each head in a grid, and the join's of up to 1024 threads for each query head
    if (n > most_groups(256) / ((int64_t)a.batch * a.hk)) n = most_groups(256) / ((int64_t)a.batch * a.hk);
    if ((int64_t)a.batch * a.hq > most_groups(1024)) n = 1;
    if (n > 1) {
        p.chunk = (int)(((most + n - 1) / n + 127) / 128 * 128);
        p.splits = (int)((most + p.chunk - 1) / p.chunk);
    }
    return p;
}

template <int D, int KT, int NW, int PER>
int run_tiles(const Args& a, const Plan& p, hipStream_t st) {
    const int64_t nb = (int64_t)a.batch * a.hk * p.splits, most = most_groups(64 * NW) / nb;
    const int64_t tiles = p.tiles < most ? p.tiles : most;
    hipLaunchKernelGGL((attn_fwd_kernel<D, KT, NW, PER>), dim3((unsigned)(tiles * nb)), dim3(64 * NW), 0, st, a);
    return launch_status("attn_fwd_kernel");
}
template <int D, int NW>
int run_few(const Args& a, const Plan& p, hipStream_t st) {
    hipLaunchKernelGGL((attn_few_kernel<D, NW>), dim3((unsigned)(a.batch * a.hk), p.splits, (unsigned)p.tiles), dim3(64 * NW), 0, st, a);
    return launch_status("attn_few_kernel");
}

}  // namespace

int64_t fwd_workspace(const Args& a) {
    const Plan p = plan_of(a);
    return p.splits > 1 ? p.splits * a.slots * (a.d + 2) * 4 : 0;
}

int launch_fwd(Args a, void* workspace, hipStream_t st) {
    const Plan p = plan_of(a);
    a.splits = p.splits;
    a.chunk = p.chunk;
    a.part = static_cast<float*>(workspace);
    a.stats = reinterpret_cast<float2*>(a.part + (p.splits > 1 ? p.splits * a.slots * a.d : 0));
    int e;
    if (p.few)
        e = a.d <= 64 ? run_few<64, 4>(a, p, st) : a.d <= 128 ? run_few<128, 4>(a, p, st) : run_few<256, 4>(a, p, st);
    else
        e = a.d <= 64    ? run_tiles<64, 64, 4, 2>(a, p, st)
            : a.d <= 128 ? run_tiles<128, 64, 4, 2>(a, p, st)
                         : run_tiles<256, 32, 4, 1>(a, p, st);
    if (e || p.splits == 1) return e;
    const int lanes = a.d <= 32 ? 8 : a.d <= 64 ? 16 : a.d <= 128 ? 32 : 64;
    int groups = 1;
    while (groups * lanes < 1024 && groups * kBatch < p.splits) groups *= 2;
    const int rows = groups * lanes < 256 ? 256 / (groups * lanes) : 1, blocks = (a.lq + rows - 1) / rows;
    hipLaunchKernelGGL(attn_join_kernel, dim3((unsigned)(a.batch * a.hq), (unsigned)(blocks < 65535 ? blocks : 65535)),
                       dim3((unsigned)(rows * groups * lanes)), 0, st, a, lanes, groups, rows);
    return launch_status("attn_join_kernel");
}

}  // namespace attn
}  // namespace r97q
