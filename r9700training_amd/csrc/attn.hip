// attn.hip -- the C entries of attention's forward and backward: checks and the kernels' arguments. The
// kernels are in attn_fwd.hip, attn_dq.hip and attn_dkdv.hip.
#include <cmath>

#include "attn.h"
#include "status.h"

namespace r97q {
namespace attn {

int64_t fwd_workspace(const Args& a);
int launch_fwd(Args a, void* workspace, hipStream_t st);
int64_t paged_workspace(const Args& a);
int launch_paged(Args a, void* workspace, hipStream_t st);
int launch_write(const Args& a, const Heads& k, const Heads& v, hipStream_t st);
int launch_dq(const Args& a, hipStream_t st);
int launch_base(const Args& a, hipStream_t st);
int launch_dq_kept(const Args& a, hipStream_t st);
int launch_sums(const Args& a, bool keys, hipStream_t st);
int launch_dkdv(const Args& a, hipStream_t st);
int launch_dkdv_wide(const Args& a, hipStream_t st);

namespace {

int refuse(int code, const char* who, const char* why) {
    set_error("%s: %s", who, why);
    return code;
}

// lens and forms; the sizes must keep every row index of a key head inside 31 bits
int check_shape(const R97qAttnShape* p, int32_t hq, int32_t hk, const char* who) {
    if (!p) return refuse(R97Q_EINVAL, who, "null shape");
    if (p->head_dim <= 0 || p->head_dim % 8 || p->head_dim > 256)
        return refuse(p->head_dim <= 0 ? R97Q_EINVAL : R97Q_EUNSUPPORTED, who, "head_dim is a multiple of 8, at most 256");
    if (hk <= 0 || hq <= 0 || hq % hk) return refuse(R97Q_EINVAL, who, "the query heads are a multiple of the key heads");
    if (p->batch < 0 || p->q_len < 0 || p->kv_len < 0) return refuse(R97Q_EINVAL, who, "a negative batch or length");
    if (p->batch > 65535 || hk > 65535) return refuse(R97Q_EUNSUPPORTED, who, "at most 65535 sequences and key heads");
    if ((int64_t)p->batch * hq > kMostHeads)
        return refuse(R97Q_EUNSUPPORTED, who, "the sequences' heads in all pass 2^23");
    if (p->q_len > 0x7FFFFF00 / (hq / hk) || p->kv_len > 0x7FFFFF00)
        return refuse(R97Q_EUNSUPPORTED, who, "a sequence's rows of one key head or its keys pass 31 bits");
    if (p->window < 0 || (p->window && !p->causal)) return refuse(R97Q_EINVAL, who, "a window is positive and needs causal");
    if (p->kv_starts && p->kv_lens) return refuse(R97Q_EINVAL, who, "kv_lens goes with the dense form of the keys");
    if ((p->q_starts && p->q_tokens < 0) || (p->kv_starts && p->kv_tokens < 0))
        return refuse(R97Q_EINVAL, who, "a negative count of packed tokens");
    if (!std::isfinite(p->scale)) return refuse(R97Q_EINVAL, who, "the scale is not finite");
    return R97Q_OK;
}

constexpr int64_t kMostStride = 1 << 24;

int check_heads(const R97qHeads* t, int32_t heads, bool f32, bool output, bool packed, int64_t batch, int64_t tokens,
                const char* who, const char* name) {
    if (!t || (!t->data && batch > 0 && tokens > 0)) {
        set_error("%s: %s is null", who, name);
        return R97Q_EINVAL;
    }
    if (t->heads != heads) {
        set_error("%s: %s has %d heads, not %d", who, name, t->heads, heads);
        return R97Q_EINVAL;
    }
    if (t->dtype != R97Q_BF16 && !(f32 && t->dtype == R97Q_F32)) {
        set_error("%s: %s is %s", who, name, f32 ? "bf16 or f32" : "bf16");
        return R97Q_EINVAL;
    }
    const int64_t unit = t->dtype == R97Q_F32 ? 4 : 8;
    if ((reinterpret_cast<uintptr_t>(t->data) & 15) || t->token_stride % unit || t->head_stride % unit ||
        (!packed && t->batch_stride % unit)) {
        set_error("%s: %s starts and strides on 16 bytes", who, name);
        return R97Q_EUNSUPPORTED;
    }
    // a tile's rows lie within 31 bits of its first
    if (tokens > 1 && t->token_stride > kMostStride) {
        set_error("%s: %s has its tokens more than %lld values apart", who, name, (long long)kMostStride);
        return R97Q_EUNSUPPORTED;
    }
    if (t->token_stride < 0 || t->head_stride < 0 || (!packed && t->batch_stride < 0) ||
        (output && ((tokens > 1 && !t->token_stride) || (heads > 1 && !t->head_stride) || (!packed && batch > 1 && !t->batch_stride)))) {
        set_error("%s: %s has a negative stride, or is written through a stride of zero", who, name);
        return R97Q_EINVAL;
    }
    return R97Q_OK;
}

Heads heads_of(const R97qHeads* t, int64_t tokens) {  // a lone token's stride says nothing
    return {static_cast<uint8_t*>(t->data), t->batch_stride, tokens > 1 ? t->token_stride : 0, t->head_stride, t->dtype == R97Q_F32};
}

Args args_of(const R97qAttnShape* p, int32_t hq, int32_t hk) {
    Args a = {};
    a.batch = p->batch;
    a.hq = hq;
    a.hk = hk;
    a.g = hq / hk;
    a.d = p->head_dim;
    a.lq = (int32_t)p->q_len;
    a.lk = (int32_t)p->kv_len;
    // a longest sequence of nothing is taken for a wrong one: what the starts say counts
    if (p->q_starts && p->q_tokens > 0 && a.lq == 0) a.lq = 1;
    if (p->kv_starts && p->kv_tokens > 0 && a.lk == 0) a.lk = 1;
    a.q_starts = p->q_starts;
    a.kv_starts = p->kv_starts;
    a.kv_lens = p->kv_lens;
    a.q_tokens = p->q_tokens;
    a.kv_tokens = p->kv_tokens;
    a.causal = p->causal != 0;
    a.window = (int32_t)(p->window < 0x7FFFFFFF ? p->window : 0x7FFFFFFF);  // past every length
    a.scale = p->scale;
    a.slots = p->q_starts ? hq * p->q_tokens : (int64_t)p->batch * hq * p->q_len;
    a.splits = 1;
    // half of an XCD's 4 MiB of L2
    const int64_t bytes = 4 * a.d * (a.batch ? mean_len(a.kv_starts, a.kv_tokens, a.lk, a.batch) : 0), most = ((int64_t)a.batch * hk + 7) / 8;
    const int64_t fit = (2 << 20) / (bytes > 0 ? bytes : 1);
    a.together = (int32_t)(fit < 1 ? 1 : fit > most ? (most < 1 ? 1 : most) : fit);
    return a;
}

// the cache's own sizes, and that every token of a sequence has a place inside 31 bits
int check_pages(const R97qAttnShape* p, const R97qPages* c, const char* who) {
    if (!c) return refuse(R97Q_EINVAL, who, "null pages");
    if (p->kv_starts) return refuse(R97Q_EINVAL, who, "kv_starts go with packed keys, not with pages");
    if (c->pages < 0 || c->max_pages < 0 || c->table_stride < 0) return refuse(R97Q_EINVAL, who, "a negative count of pages or stride of the table");
    if (c->page_size < 8 || c->page_size > (1 << 20) || (c->page_size & (c->page_size - 1)))
        return refuse(c->page_size < 1 ? R97Q_EINVAL : R97Q_EUNSUPPORTED, who, "a page holds a power of two of tokens, 8 to 2^20");
    if (c->pages > 0x7FFFFFFF || (int64_t)c->max_pages * c->page_size > 0x7FFFFF00)
        return refuse(R97Q_EUNSUPPORTED, who, "the pages' count or a sequence's tokens pass 31 bits");
    if (p->batch > 0 && ((!c->table && c->max_pages > 0) || !p->kv_lens)) return refuse(R97Q_EINVAL, who, "null table or kv_lens");
    return R97Q_OK;
}

int64_t q_rows(const R97qAttnShape* p) { return p->q_starts ? p->q_tokens : p->q_len; }
int64_t kv_rows(const R97qAttnShape* p) { return p->kv_starts ? p->kv_tokens : p->kv_len; }

// How the backward is cut where its grids leave compute units idle: a tile's steps over up to kMostCuts workgroups,
// whose f32 sums another launch adds. Measured on 16 over 4 heads (us at 1 / 2 / 4 / 8 cuts; a cut writes and reads
// its sums): dK and dV of 1 x 1300 tokens, heads of 128: 176 / 123 / 93 / 86; of 2 x 1300: 181 / 130 / 104 / 123; of
// 4 x 700: 112 / 92 / 85 / 105; of 512 tokens, heads of 64: 54 / 43 / 36 / 35; of 128, heads of 64 (8 steps a tile):
// 26 / 23 / 20 / 20, of 64 18 / 19 / 17; so up to some 320 workgroups of at least four steps, or eight cuts of at
// least two. dQ of 64 rows over 4096 keys: 103 / 70 / 53 / 46, but of 1 x 1300: 175 / 178 / 188 / 214 and of 512: 80
// / 84 / 86 / 92; so only below half the compute units and from 512 keys a cut. Where dK's and dV's tiles just fill
// the compute units and are long, the causal ones' first tile has twice the steps of the mean, and two cuts even that
// out (the whole backward with dS^T kept, us at 1 / 2 cuts): heads of 128, 4 x 2048 tokens 336 / 317, 24 heads 468 /
// 402, but 8 x 1024 194 / 186, 16 x 512 116 / 135, 6 x 2048 415 / 443; of 256, 4 x 2048 560 / 499, 8 x 1024 311 /
// 323; of 64, two workgroups a unit, 4 x 2048 201 / 164, 8 x 1024 117 / 103, 16 x 512 73 / 74.
constexpr int kMostCuts = 16;
int cuts(int64_t want, int64_t have, int64_t steps) {
    int64_t n = have > 0 ? (want + have - 1) / have : 1;
    if (n > steps) n = steps;
    return (int)(n < 1 ? 1 : n > kMostCuts ? kMostCuts : n);
}
void cut_backward(Args& a) {
    a.q_splits = a.k_splits = 1;
    if (a.batch > 0) {
        const int64_t tiles = a.hk * all_tiles(a.q_starts, a.q_tokens, a.lq, a.batch, a.g, 128);
        const int64_t keys = a.hk * all_tiles(a.kv_starts, a.kv_tokens, a.lk, a.batch, 1, 128);
        int64_t seen = mean_len(a.kv_starts, a.kv_tokens, a.lk, a.batch), seeing = mean_len(a.q_starts, a.q_tokens, a.lq, a.batch);
        if (a.window && (int64_t)a.window + 128 < seen) seen = (int64_t)a.window + 128;
        if (a.window && (int64_t)a.window + 128 < seeing) seeing = (int64_t)a.window + 128;
        a.q_splits = tiles * 2 <= 256 ? cuts(256, tiles, seen / 512) : 1;
        const int64_t rows = a.g * seeing;
        const int64_t steps = rows / (a.d > 128 ? 32 : 64), two = steps / 2 < 8 ? steps / 2 : 8;
        a.k_splits = keys * 3 / 2 < 320 ? cuts(320, keys, steps < 8 ? 1 : steps / 4 > two ? steps / 4 : two) : 1;
        // and a workgroup for each cut of each head in a grid
        const int most = (int)(most_groups(256) / ((int64_t)a.batch * a.hk));
        if (a.q_splits > most) a.q_splits = most;
        if (a.k_splits > most) a.k_splits = most;
        if (a.k_splits == 1 && most > 1 && a.causal && !a.window && (a.d <= 64 ? keys <= 384 && rows >= 3500 : keys <= 256 && rows >= 6144)) a.k_splits = 2;
    }
    a.kv_slots = a.kv_starts ? a.hk * a.kv_tokens : (int64_t)a.batch * a.hk * a.lk;
}
// Whether dS^T is kept between the launches (then dQ is one product from it, instead of three from scratch): the bytes,
// or 0. It costs its bytes written and read, and D's own launch. Measured, computed again / kept (us): heads of 256, 8 x
// 2048 tokens, 16 over 4 heads 1014 / 843, 4 x 2048 560 / 480, 1 x 512 tokens, 8 over 2 66 / 50; heads of 128, 16 over 4,
// 8 x 2048 501 / 535, 4 x 2048 275 / 303, 2 x 4096 472 / 520, 4 x 1300 157 / 151, 1 x 1300 81 / 68; heads of 64, 8 x 2048
// 287 / 382, 4 x 1300 92 / 106, 1 x 1300 54 / 51. So from heads of more than 64 columns, up to 256 MiB with heads of up to
// 128, and up to 2 GiB of workspace; not where dQ's rows are cut, since few rows over many keys are few workgroups here (64
// over 4096: 45 / 60).
int64_t kept_bytes(Args& a) {
    if (a.d <= 64 || a.q_splits > 1 || a.batch == 0) return 0;
    const double rows = a.kv_starts ? (double)a.hq * a.kv_tokens : (double)a.batch * a.hq * a.lk;
    a.pitch = a.q_starts ? (a.q_tokens + 64LL * (a.batch + 2) + 63) / 64 * 64 : ((int64_t)a.lq + 127) / 128 * 128;
    // what is touched of it: packed sequences leave most of it alone
    const double each = (double)mean_len(a.q_starts, a.q_tokens, a.lq, a.batch) * mean_len(a.kv_starts, a.kv_tokens, a.lk, a.batch);
    if (a.pitch > kMostStride || 2.0 * rows * a.pitch > (double)(2LL << 30)) return 0;
    if (a.d <= 128 && 2.0 * a.batch * a.hq * each > (double)(256LL << 20)) return 0;
    return (2 * (int64_t)rows * a.pitch + 255) / 256 * 256;
}
Args paged_args(const R97qAttnShape* p, const R97qPages* c, int32_t hq, int32_t hk) {
    Args a = args_of(p, hq, hk);
    a.held = a.lk;
    a.lk = c->max_pages * c->page_size;  // what kv_lens are clamped to
    if (a.held > a.lk) a.held = a.lk;
    a.table = c->table;
    a.table_stride = c->table_stride;
    a.pages = (int32_t)c->pages;
    a.max_pages = c->max_pages;
    a.page_shift = __builtin_ctz((unsigned)c->page_size);
    return a;
}
int64_t bwd_stats(const Args& a) { return (8 * a.slots + 255) / 256 * 256; }

}  // namespace
}  // namespace attn
}  // namespace r97q

using namespace r97q;
using namespace r97q::attn;

extern "C" {

int64_t r97q_attn_fwd_workspace_bytes(const R97qAttnShape* shape, int32_t q_heads, int32_t kv_heads) {
    clear_error();
    if (check_shape(shape, q_heads, kv_heads, "r97q_attn_fwd_workspace_bytes")) return -1;
    if (shape->batch == 0 || q_rows(shape) == 0) return 0;  // nothing runs; a packed q_len of 0 is a wrong one, and runs
    return fwd_workspace(args_of(shape, q_heads, kv_heads));
}

int r97q_attn_fwd(const R97qAttnShape* shape, const R97qHeads* q, const R97qHeads* k, const R97qHeads* v,
                  const R97qHeads* out, float* lse, void* workspace, int64_t workspace_bytes, R97IqrStream stream) {
    clear_error();
    const char* who = "r97q_attn_fwd";
    if (!q || !k) return refuse(R97Q_EINVAL, who, "null q or k");
    const int32_t hq = q->heads, hk = k->heads;
    if (int e = check_shape(shape, hq, hk, who)) return e;
    const int64_t n = q_rows(shape), m = kv_rows(shape), b = shape->batch;
    const bool pq = shape->q_starts, pk = shape->kv_starts;
    if (int e = check_heads(q, hq, false, false, pq, b, n, who, "q")) return e;
    if (int e = check_heads(k, hk, false, false, pk, b, m, who, "k")) return e;
    if (int e = check_heads(v, hk, false, false, pk, b, m, who, "v")) return e;
    if (int e = check_heads(out, hq, true, true, pq, b, n, who, "out")) return e;
    const int64_t need = r97q_attn_fwd_workspace_bytes(shape, hq, hk);
    if (need > 0 && (!workspace || workspace_bytes < need)) return refuse(R97Q_EWORKSPACE, who, "the workspace is too small");
    if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15)) return refuse(R97Q_EINVAL, who, "the workspace starts on 16 bytes");
    if (b == 0 || n == 0) return R97Q_OK;
    Args a = args_of(shape, hq, hk);
    a.q = heads_of(q, n);
    a.k = heads_of(k, m);
    a.v = heads_of(v, m);
    a.o = heads_of(out, n);
    a.lse = lse;
    return launch_fwd(a, workspace, (hipStream_t)stream);
}

int64_t r97q_paged_attn_fwd_workspace_bytes(const R97qAttnShape* shape, const R97qPages* pages, int32_t q_heads, int32_t kv_heads) {
    clear_error();
    const char* who = "r97q_paged_attn_fwd_workspace_bytes";
    if (check_shape(shape, q_heads, kv_heads, who) || check_pages(shape, pages, who)) return -1;
    if (shape->batch == 0 || q_rows(shape) == 0) return 0;
    return paged_workspace(paged_args(shape, pages, q_heads, kv_heads));
}

int r97q_paged_attn_fwd(const R97qAttnShape* shape, const R97qPages* pages, const R97qHeads* q, const R97qHeads* k, const R97qHeads* v,
                        const R97qHeads* out, float* lse, void* workspace, int64_t workspace_bytes, R97IqrStream stream) {
    clear_error();
    const char* who = "r97q_paged_attn_fwd";
    if (!q || !k) return refuse(R97Q_EINVAL, who, "null q or k");
    const int32_t hq = q->heads, hk = k->heads;
    if (int e = check_shape(shape, hq, hk, who)) return e;
    if (int e = check_pages(shape, pages, who)) return e;
    const int64_t n = q_rows(shape), b = shape->batch;
    const bool pq = shape->q_starts;
    if (int e = check_heads(q, hq, false, false, pq, b, n, who, "q")) return e;
    if (int e = check_heads(k, hk, false, false, false, pages->pages, pages->page_size, who, "k")) return e;
    if (int e = check_heads(v, hk, false, false, false, pages->pages, pages->page_size, who, "v")) return e;
    if (int e = check_heads(out, hq, true, true, pq, b, n, who, "out")) return e;
    if (b == 0 || n == 0) return R97Q_OK;
    Args a = paged_args(shape, pages, hq, hk);
    const int64_t need = paged_workspace(a);
    if (need > 0 && (!workspace || workspace_bytes < need)) return refuse(R97Q_EWORKSPACE, who, "the workspace is too small");
    if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15)) return refuse(R97Q_EINVAL, who, "the workspace starts on 16 bytes");
    a.q = heads_of(q, n);
    a.k = heads_of(k, pages->page_size);
    a.v = heads_of(v, pages->page_size);
    a.o = heads_of(out, n);
    a.lse = lse;
    return launch_paged(a, workspace, (hipStream_t)stream);
}

int r97q_paged_write(const R97qAttnShape* shape, const R97qPages* pages, const R97qHeads* k, const R97qHeads* v, const R97qHeads* k_pages,
                     const R97qHeads* v_pages, R97IqrStream stream) {
    clear_error();
    const char* who = "r97q_paged_write";
    if (!k || !v || !k_pages) return refuse(R97Q_EINVAL, who, "null k, v or pages");
    const int32_t hk = k_pages->heads;
    if (int e = check_shape(shape, hk, hk, who)) return e;
    if (int e = check_pages(shape, pages, who)) return e;
    const int64_t n = q_rows(shape), b = shape->batch;
    const bool pq = shape->q_starts;
    if (int e = check_heads(k, hk, true, false, pq, b, n, who, "k")) return e;
    if (int e = check_heads(v, hk, true, false, pq, b, n, who, "v")) return e;
    if (k->dtype != v->dtype) return refuse(R97Q_EINVAL, who, "k and v are both bf16 or both f32");
    if (int e = check_heads(k_pages, hk, false, true, false, pages->pages, pages->page_size, who, "k_pages")) return e;
    if (int e = check_heads(v_pages, hk, false, true, false, pages->pages, pages->page_size, who, "v_pages")) return e;
    if (b == 0 || n == 0 || pages->pages == 0 || pages->max_pages == 0) return R97Q_OK;
    Args a = paged_args(shape, pages, hk, hk);
    a.k = heads_of(k_pages, pages->page_size);
    a.v = heads_of(v_pages, pages->page_size);
    return launch_write(a, heads_of(k, n), heads_of(v, n), (hipStream_t)stream);
}

int64_t r97q_attn_bwd_workspace_bytes(const R97qAttnShape* shape, int32_t q_heads, int32_t kv_heads) {
    clear_error();
    if (check_shape(shape, q_heads, kv_heads, "r97q_attn_bwd_workspace_bytes")) return -1;
    Args a = args_of(shape, q_heads, kv_heads);
    cut_backward(a);
    const int64_t row = 4 * a.d, kept = kept_bytes(a);
    return bwd_stats(a) + kept + (a.q_splits > 1 ? a.q_splits * a.slots * row : 0) + (a.k_splits > 1 ? 2 * a.k_splits * a.kv_slots * row : 0);
}

int r97q_attn_bwd(const R97qAttnShape* shape, const R97qHeads* q, const R97qHeads* k, const R97qHeads* v,
                  const R97qHeads* out, const float* lse, const R97qHeads* d_out, const R97qHeads* dq,
                  const R97qHeads* dk, const R97qHeads* dv, void* workspace, int64_t workspace_bytes, R97IqrStream stream) {
    clear_error();
    const char* who = "r97q_attn_bwd";
    if (!q || !k) return refuse(R97Q_EINVAL, who, "null q or k");
    const int32_t hq = q->heads, hk = k->heads;
    if (int e = check_shape(shape, hq, hk, who)) return e;
    const int64_t n = q_rows(shape), m = kv_rows(shape), b = shape->batch;
    const bool pq = shape->q_starts, pk = shape->kv_starts;
    if (int e = check_heads(q, hq, false, false, pq, b, n, who, "q")) return e;
    if (int e = check_heads(k, hk, false, false, pk, b, m, who, "k")) return e;
    if (int e = check_heads(v, hk, false, false, pk, b, m, who, "v")) return e;
    if (int e = check_heads(out, hq, true, false, pq, b, n, who, "out")) return e;
    if (int e = check_heads(d_out, hq, false, false, pq, b, n, who, "d_out")) return e;
    if (int e = check_heads(dq, hq, true, true, pq, b, n, who, "dq")) return e;
    if (int e = check_heads(dk, hk, true, true, pk, b, m, who, "dk")) return e;
    if (int e = check_heads(dv, hk, true, true, pk, b, m, who, "dv")) return e;
    if (b == 0) return R97Q_OK;
    if (!lse && n > 0) return refuse(R97Q_EINVAL, who, "null lse");
    if (workspace_bytes < r97q_attn_bwd_workspace_bytes(shape, hq, hk) || (!workspace && n > 0))
        return refuse(R97Q_EWORKSPACE, who, "the workspace is too small");
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return refuse(R97Q_EINVAL, who, "the workspace starts on 16 bytes");
    Args a = args_of(shape, hq, hk);
    cut_backward(a);
    if (n == 0) a.lq = 0;
    if (m == 0) a.lk = 0;
    a.q = heads_of(q, n);
    a.k = heads_of(k, m);
    a.v = heads_of(v, m);
    a.o = heads_of(out, n);
    a.d_o = heads_of(d_out, n);
    a.dq = heads_of(dq, n);
    a.dk = heads_of(dk, m);
    a.dv = heads_of(dv, m);
    a.lse = const_cast<float*>(lse);
    a.base = static_cast<float*>(workspace);
    a.delta = a.base + a.slots;
    const int64_t kept = kept_bytes(a);
    uint8_t* rest = static_cast<uint8_t*>(workspace) + bwd_stats(a);
    if (kept) a.ds = reinterpret_cast<uint16_t*>(rest);
    a.dq_part = reinterpret_cast<float*>(rest + kept);
    a.dk_part = a.dq_part + (a.q_splits > 1 ? a.q_splits * a.slots * a.d : 0);
    a.dv_part = a.dk_part + a.k_splits * a.kv_slots * a.d;
    hipStream_t st = (hipStream_t)stream;
    if (int e = kept ? launch_base(a, st) : launch_dq(a, st)) return e;
    if (a.q_splits > 1)
        if (int e = launch_sums(a, false, st)) return e;
    if (int e = a.d > 128 ? launch_dkdv_wide(a, st) : launch_dkdv(a, st)) return e;
    if (kept)
        if (int e = launch_dq_kept(a, st)) return e;
    return a.k_splits > 1 ? launch_sums(a, true, st) : R97Q_OK;
}

}  // extern "C"
