"""The paged cache against float64: attention of one new token, a few, or a chunk over pages of every size, and the write of
new tokens into them. Whatever no query sees (slots past a sequence, expired places, unused pages and table entries) holds
NaN or nonsense. Tolerances are attention's (tests/between_ref.py)."""
import math

import pytest
import torch

import between_ref as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def rnd(seed, *shape, dtype=BF):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def close(got, want, tol, what):
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin), f"{what}: other places are finite"
    assert torch.equal(got[~fin], want[~fin]), what
    if want.numel():
        over = float(((got - want).abs() - tol)[fin].max()) if fin.any() else -1.0
        assert over <= 1e-30, f"{what}: {over} past the tolerance"


class Cache:
    """Sequences' keys and values scattered over pages; everything else is NaN, and unused entries of the table nonsense."""

    def __init__(self, lens, heads, dim, page, order="slots", seed=1, spare=3, room=2, first=0, junk=(-1, 1 << 30)):
        self.lens, self.page = list(lens), page
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare + first
        shape = (pages, page, heads, dim) if order == "slots" else (pages, heads, page, dim)
        self.k, self.v = (torch.full(shape, math.nan, dtype=BF, device="cuda") for _ in range(2))
        if order == "heads":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        ids = (first + torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed))).tolist()
        most = max(need, default=0) + room
        self.table = torch.tensor([[junk[(b + j) % 2] for j in range(most)] for b in range(len(lens))], dtype=torch.int32).reshape(len(lens), most)
        self.keys, self.values = [], []
        for b, n in enumerate(self.lens):
            k, v = rnd(100 + 2 * b + seed, n, heads, dim), rnd(101 + 2 * b + seed, n, heads, dim)
            for j in range(need[b]):
                at = self.table[b, j] = ids.pop()
                part = slice(j * page, min(n, (j + 1) * page))
                self.k[at, :part.stop - part.start], self.v[at, :part.stop - part.start] = k[part], v[part]
            self.keys.append(k)
            self.values.append(v)
        self.table = self.table.cuda()
        self.kv_lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def expire(self, before):
        """Tokens before `before[b]` hold NaN, their whole pages have no entry."""
        for b, n in enumerate(before):
            for j in range(-(-n // self.page)):
                at, upto = int(self.table[b, j]), min(self.page, n - j * self.page)
                self.k[at, :upto], self.v[at, :upto] = math.nan, math.nan
                if upto == self.page:
                    self.table[b, j] = -7


def expected(c, qs, heads, kv_heads, causal, window, scale, half):
    return R.reference([(q.double(), k.double(), v.double(), None) for q, k, v in zip(qs, c.keys, c.values)], heads, kv_heads,
                       causal, window, scale, half)


CASES = [
    # new tokens of each sequence, tokens of each, q_heads, kv_heads, head_dim, page, causal, window
    ([1], [1], 1, 1, 64, 8, True, 0),
    ([1, 1, 1], [77, 1, 500], 4, 1, 64, 16, True, 0),
    ([1, 1], [1000, 513], 24, 4, 256, 32, True, 0),
    ([1] * 9, [3000, 1, 8, 16, 17, 900, 2048, 0, 65], 32, 8, 128, 16, True, 0),
    ([1], [20000], 24, 4, 256, 64, True, 0),
    ([1] * 3, [12000, 0, 1], 4, 1, 64, 16, True, 0),      # one sequence takes nearly all workgroups
    ([2] * 5, [6000, 5, 1300, 127, 129], 8, 2, 128, 64, True, 0),
    ([1] * 4, [3000, 2500, 1, 700], 16, 2, 256, 8, True, 900),
    ([1] * 64, [37 * i % 1900 for i in range(64)], 4, 1, 64, 16, True, 0),
    ([1] * 65, [53 * i % 2500 for i in range(65)], 2, 1, 64, 32, True, 0),
    ([1, 1], [5000, 1700], 8, 2, 128, 8, True, 300),
    ([3, 3], [200, 2], 14, 2, 128, 16, True, 0),          # the second's first query has no key
    ([5], [4097], 6, 3, 80, 8, True, 33),
    ([31], [31], 2, 2, 64, 128, True, 0),
    ([33], [65], 3, 1, 80, 16, True, 0),
    ([128, 128], [128, 1000], 8, 2, 64, 8, True, 0),
    ([129], [2000], 4, 2, 128, 16, True, 0),
    ([255], [257], 2, 1, 256, 8, True, 0),
    ([300], [777], 2, 2, 64, 32, False, 0),
    ([97], [40], 2, 1, 64, 16, True, 0),                  # the first 57 queries see nothing
    ([70, 70], [0, 9], 4, 2, 64, 16, True, 0),
    ([190], [190], 2, 1, 64, 16, True, 1),
    ([190, 190], [260, 1900], 2, 1, 128, 64, True, 50),
    ([260], [3001], 4, 4, 256, 16, True, 333),
    ([200], [3001], 4, 4, 128, 8, True, 70),
    ([65], [70], 2, 1, 8, 16, True, 0),
    ([40], [40], 7, 1, 248, 512, True, 0),
    ([520], [6000], 12, 2, 128, 256, True, 0),
    ([520], [6000], 12, 2, 128, 64, True, 1000),
    ([64], [9000], 16, 4, 64, 16, True, 0),
    ([600], [1111], 6, 2, 72, 1024, True, 0),
    ([1200], [4000], 16, 4, 64, 64, True, 0),             # chunks that fill the card, cut into ranges all the same
    ([1024], [4100], 16, 4, 128, 16, True, 0),
    ([1300], [4200], 16, 4, 256, 64, True, 0),
]


@pytest.mark.parametrize("new,lens,hq,hk,d,page,causal,window", CASES)
@pytest.mark.parametrize("order", ["slots", "heads"])
def test_dense(new, lens, hq, hk, d, page, causal, window, order):
    from r9700training_amd.paged import paged_attention_fwd

    print(f"case paged {(new, lens, hq, hk, d, page, causal, window, order)}", flush=True)
    c = Cache(lens, hk, d, page, order)
    if window:
        c.expire([max(0, m - n - window + 1) for n, m in zip(new, lens)])
    q, scale = rnd(1, len(new), new[0], hq, d), 1.0 / math.sqrt(d)
    for dtype in (BF, torch.float32):
        ref = expected(c, q, hq, hk, causal, window, scale, R.HALF[dtype])
        for most in (None, max(lens), 1, 1 << 20):  # the plan's length: results go by kv_lens alone
            out, lse = paged_attention_fwd(q, c.k, c.v, c.table, c.kv_lens, causal=causal, window=window, max_kv=most, out_dtype=dtype)
            torch.cuda.synchronize()
            for b, r in enumerate(ref):
                close(out[b], *r["out"], f"out of sequence {b}, planned for {most}")
                close(lse[b], *r["lse"], f"lse of sequence {b}, planned for {most}")
            if dtype == torch.float32:
                break


PACKED = [
    ([1, 3, 1, 5], [400, 30, 1, 5], 8, 2, 64, 16, 0),
    ([70, 0, 1, 200], [500, 90, 300, 200], 8, 2, 128, 16, 0),
    ([40, 129, 300], [2000, 129, 310], 6, 1, 256, 64, 0),
    ([300, 17, 1], [3000, 17, 4000], 4, 4, 64, 8, 100),
    ([5, 100], [3, 60], 4, 2, 80, 32, 0),                 # more new tokens than the cache has room for
    ([0, 0], [7, 0], 2, 1, 64, 16, 0),
    ([700, 400, 1, 250], [5000, 900, 30, 2600], 16, 4, 64, 32, 0),
    ([900, 300, 0, 500], [3000, 301, 9, 2600], 16, 4, 64, 16, 2700),
]


@pytest.mark.parametrize("new,lens,hq,hk,d,page,window", PACKED)
def test_packed(new, lens, hq, hk, d, page, window):
    from r9700training_amd.paged import paged_attention_fwd

    print(f"case paged packed {(new, lens, hq, hk, d, page, window)}", flush=True)
    c = Cache(lens, hk, d, page)
    if window:
        c.expire([max(0, m - n - window + 1) for n, m in zip(new, lens)])
    starts = [2]
    for n in new:
        starts.append(starts[-1] + n)
    tokens = starts[-1] + 3                               # two tokens before the first sequence, three after the last
    q, scale = rnd(1, tokens, hq, d), 0.1
    at = torch.tensor(starts, dtype=torch.int32, device="cuda")
    qs = [q[a:b] for a, b in zip(starts, starts[1:])]
    ref = expected(c, qs, hq, hk, True, window, scale, R.HALF[BF])
    for most in (max(new), 0, 5000):
        out = torch.full((tokens, hq, d), 7.0, dtype=BF, device="cuda")
        lse = torch.full((hq, tokens), 7.0, device="cuda")
        paged_attention_fwd(q, c.k, c.v, c.table, c.kv_lens, window=window, scale=scale, q_starts=at, max_q=most, out=out, lse=lse)
        torch.cuda.synchronize()
        for b, r in enumerate(ref):
            part = slice(starts[b], starts[b + 1])
            close(out[part], *r["out"], f"out of sequence {b}")
            close(lse[:, part], *r["lse"], f"lse of sequence {b}")
        for part in (slice(0, 2), slice(starts[-1], tokens)):
            assert (out[part] == 7).all() and (lse[:, part] == 7).all()


@pytest.mark.parametrize("new,d,page", [(1, 128, 8), (100, 128, 8), (1, 64, 16), (200, 256, 16), (100, 80, 256), (1, 80, 256), (3, 200, 64),
                                        (90, 200, 128), (90, 40, 32)])
def test_entries_outside_the_pool_read_as_zeros(new, d, page):
    """Also where a head has fewer columns than its tile: what lies elsewhere in the pool is NaN."""
    from r9700training_amd.paged import paged_attention_fwd

    lens = [5 * page + 3, 7 * page]
    c = Cache(lens, 2, d, page)
    for b, j, e in [(0, 1, -1), (0, 2, c.k.shape[0]), (1, 0, 2 ** 31 - 1), (1, 5, -(1 << 31)), (1, 6, 1 << 30)]:
        c.table[b, j] = e
        c.keys[b][j * page:(j + 1) * page] = 0
        c.values[b][j * page:(j + 1) * page] = 0
    q = rnd(1, 2, new, 4, d)
    for window in (0, 3 * page):
        ref = expected(c, q, 4, 2, True, window, 0.1, R.HALF[BF])
        out, lse = paged_attention_fwd(q, c.k, c.v, c.table, c.kv_lens, scale=0.1, window=window)
        for b, r in enumerate(ref):
            close(out[b], *r["out"], f"out of sequence {b}")
            close(lse[b], *r["lse"], f"lse of sequence {b}")


@pytest.mark.parametrize("new,d", [(1, 128), (100, 128), (1, 64), (200, 256)])
def test_entries_outside_the_pool(new, d):
    """They read as zeros, wherever they stand; lengths past the table are the table's."""
    from r9700training_amd.paged import paged_attention_fwd

    page, n = 16, 300
    c = Cache([n, n], 2, d, page, room=0)
    bad = [(0, 0, -1), (0, 7, c.k.shape[0]), (0, 18, 1 << 30), (1, 3, -(1 << 31)), (1, 4, 2 ** 31 - 1)]
    for b, j, e in bad:
        c.table[b, j] = e
        c.keys[b][j * page:(j + 1) * page] = 0
        c.values[b][j * page:(j + 1) * page] = 0
    q = rnd(1, 2, new, 4, d)
    ref = expected(c, q, 4, 2, True, 0, 0.1, R.HALF[BF])
    out, lse = paged_attention_fwd(q, c.k, c.v, c.table, c.kv_lens, scale=0.1)
    for b, r in enumerate(ref):
        close(out[b], *r["out"], f"out of sequence {b}")
        close(lse[b], *r["lse"], f"lse of sequence {b}")
    # the table's 19 pages hold 304 tokens: the rest of the last page is made readable
    last = int(c.table[1, 18])
    c.k[last, n % page:], c.v[last, n % page:] = c.k[last, 0], c.v[last, 0]
    c.table[0, 18] = last
    full = paged_attention_fwd(q, c.k, c.v, c.table, torch.full((2,), 304, dtype=torch.int32, device="cuda"), scale=0.1)
    past = paged_attention_fwd(q, c.k, c.v, c.table, torch.tensor([2 ** 31 - 1, 305], dtype=torch.int32, device="cuda"), scale=0.1)
    assert torch.equal(full[0], past[0]) and torch.equal(full[1], past[1])
    none = paged_attention_fwd(q, c.k, c.v, c.table, torch.tensor([-5, 0], dtype=torch.int32, device="cuda"), scale=0.1)
    assert (none[0] == 0).all() and (none[1] == -math.inf).all()


@pytest.mark.parametrize("new,d", [(1, 128), (150, 64), (150, 256)])
def test_shared_pages(new, d):
    """Sequences that begin alike name the same pages."""
    from r9700training_amd.paged import paged_attention_fwd

    c = Cache([200, 230], 2, d, 16)
    c.table[1, :8] = c.table[0, :8]
    c.keys[1][:128], c.values[1][:128] = c.keys[0][:128], c.values[0][:128]
    q = rnd(1, 2, new, 4, d)
    ref = expected(c, q, 4, 2, True, 0, 0.1, R.HALF[BF])
    out, _ = paged_attention_fwd(q, c.k, c.v, c.table, c.kv_lens, scale=0.1)
    for b, r in enumerate(ref):
        close(out[b], *r["out"], f"out of sequence {b}")


@pytest.mark.parametrize("page,d", [(64, 128), (8, 64), (256, 256), (16, 128)])
@pytest.mark.parametrize("new", [1, 90])
def test_far_pages(new, page, d):
    """A pool of more than 2^32 bytes and 2^31 values: pages at its end."""
    from r9700training_amd.paged import paged_attention_fwd, paged_write

    heads, lens = 8, [130, 700]
    pages = 2 ** 31 // (page * heads * d) + 8
    c = Cache(lens, heads, d, page)
    k, v = (torch.empty((pages, page, heads, d), dtype=BF, device="cuda") for _ in range(2))
    first = pages - c.k.shape[0]
    k[first:], v[first:] = c.k, c.v
    ids = torch.where((c.table >= 0) & (c.table < pages), c.table + first, c.table)
    q = rnd(1, 2, new, heads, d)
    want = paged_attention_fwd(q, c.k, c.v, c.table, c.kv_lens)
    got = paged_attention_fwd(q, k, v, ids, c.kv_lens)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    nk, nv = rnd(5, 2, new, heads, d), rnd(6, 2, new, heads, d)
    paged_write(nk, nv, c.k, c.v, c.table, c.kv_lens)
    paged_write(nk, nv, k, v, ids, c.kv_lens)
    assert torch.equal(k[first:].view(torch.int16), c.k.view(torch.int16)) and torch.equal(v[first:].view(torch.int16), c.v.view(torch.int16))


WRITES = [
    # new tokens, tokens with them, heads, head_dim, page, packed
    ([1], [1], 1, 8, 8, False),
    ([1, 1, 1, 1], [16, 17, 1, 300], 8, 128, 16, False),
    ([5, 5], [5, 800], 3, 80, 32, False),
    ([700], [1000], 2, 256, 64, False),
    ([7, 7], [3, 20], 2, 64, 8, False),                   # four of the first's have no place
    ([300, 0, 1, 77], [300, 50, 1, 100], 4, 64, 128, True),
    ([2000, 3], [2001, 4000], 8, 128, 16, True),
    ([1] * 40, list(range(1, 41)), 2, 64, 8, False),
]


@pytest.mark.parametrize("new,lens,heads,d,page,packed", WRITES)
@pytest.mark.parametrize("order", ["slots", "heads"])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_write(new, lens, heads, d, page, packed, order, dtype):
    """Every new token in its place, rounded once from f32; all other places untouched, to the bit."""
    from r9700training_amd.paged import paged_write

    print(f"case write {(new, lens, heads, d, page, packed, order, dtype)}", flush=True)
    c = Cache(lens, heads, d, page, order)
    want_k, want_v = c.k.clone(), c.v.clone()
    starts = [1]
    for n in new:
        starts.append(starts[-1] + n)
    shape = (starts[-1] + 2, heads, d) if packed else (len(new), new[0], heads, d)
    kv = rnd(3, *shape[:-2], 2 * heads * d + 8, dtype=dtype)  # k and v side by side in a wider projection's rows
    k = kv[..., :heads * d].unflatten(-1, (heads, d))
    v = kv[..., heads * d:2 * heads * d].unflatten(-1, (heads, d))
    for b, (n, m) in enumerate(zip(new, lens)):
        kb, vb = (k[starts[b]:starts[b + 1]], v[starts[b]:starts[b + 1]]) if packed else (k[b], v[b])
        for i in range(max(0, n - m), n):
            at = m - n + i
            page_id = int(c.table[b, at // page])
            want_k[page_id, at % page], want_v[page_id, at % page] = kb[i].to(BF), vb[i].to(BF)
    extra = dict(q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda")) if packed else {}
    for most in ((max(new), 1) if packed else (None,)):
        ck, cv = c.k.clone(), c.v.clone()
        paged_write(k, v, ck, cv, c.table, c.kv_lens, max_q=most, **extra)
        torch.cuda.synchronize()
        assert torch.equal(ck.view(torch.int16), want_k.view(torch.int16))
        assert torch.equal(cv.view(torch.int16), want_v.view(torch.int16))
    # pages that are no pages take nothing
    gone = torch.full_like(c.table, -1)
    gone[:, ::2] = c.k.shape[0]
    ck, cv = c.k.clone(), c.v.clone()
    paged_write(k, v, ck, cv, gone, c.kv_lens, max_q=max(new), **extra)
    paged_write(k, v, ck, cv, c.table[:, :0], c.kv_lens, max_q=max(new), **extra)
    torch.cuda.synchronize()
    assert torch.equal(ck.view(torch.int16), c.k.view(torch.int16)) and torch.equal(cv.view(torch.int16), c.v.view(torch.int16))


@pytest.mark.parametrize("new,d", [(1, 128), (1, 256), (130, 64), (40, 128)])
def test_streams_and_graphs(new, d):
    """On a stream of its own, and captured: two graphs with their own workspaces replayed in turn as the cache grows."""
    from r9700training_amd.paged import paged_attention_fwd, paged_write

    heads, kv_heads, page, room = 8, 2, 16, 1500
    lens = [900, 300]
    c = Cache([room, room], kv_heads, d, page, room=0)
    c.k.nan_to_num_(), c.v.nan_to_num_()
    held = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q, k, v = rnd(1, 2, new, heads, d), rnd(2, 2, new, kv_heads, d), rnd(3, 2, new, kv_heads, d)

    def step(stream=None):
        paged_write(k, v, c.k, c.v, c.table, held, stream=stream)
        return paged_attention_fwd(q, c.k, c.v, c.table, held, stream=stream)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(side)
    torch.cuda.synchronize()
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, step()))
    for i in range(4):
        held.add_(new)
        q.copy_(rnd(10 + i, 2, new, heads, d)), k.copy_(rnd(20 + i, 2, new, kv_heads, d))
        want = [x.clone() for x in step()]
        c.k.view(-1)[:8].add_(0)  # the program's own work between the replays
        g, got = graphs[i % 2]
        got[0].fill_(5)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.parametrize("page,chunk", [(16, 100), (64, 333), (8, 1)])
def test_a_prompt_in_chunks(page, chunk):
    """Rotary with three axes, the write and attention, chunk by chunk, against the whole prompt at once in float64."""
    from r9700training_amd.paged import paged_attention_fwd, paged_write
    from r9700training_amd.rotary import rotary_axes, rotary_frequencies, rotary_pair_axes

    n, heads, kv_heads, d = (700 if chunk > 1 else 40), 8, 2, 64
    q, k, v = rnd(1, n, heads, d), rnd(2, n, kv_heads, d), rnd(3, n, kv_heads, d)
    pos = torch.stack([torch.arange(n) // 7, torch.arange(n) % 11, torch.arange(n)]).to(torch.int32).cuda()
    f, _ = rotary_frequencies(d)
    axis = rotary_pair_axes([12, 10, 10], "cycle")
    pages = -(-n // page) + 2
    kp, vp = (torch.full((pages, page, kv_heads, d), math.nan, dtype=BF, device="cuda") for _ in range(2))
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()[None]
    outs, kept = [], []
    for a in range(0, n, chunk):
        part = slice(a, min(n, a + chunk))
        qr, kr = rotary_axes(q[part], k[part], f, pos[:, part], axis)
        held = torch.tensor([part.stop], dtype=torch.int32, device="cuda")
        paged_write(kr[None], v[part][None], kp, vp, table, held)
        outs.append(paged_attention_fwd(qr[None], kp, vp, table, held)[0][0])
        kept.append((qr, kr))
    qr, kr = torch.cat([x for x, _ in kept]), torch.cat([x for _, x in kept])
    angles = pos.double()[axis.long()].T * f
    # turned in f32 and rounded once: a step of bf16 covers it
    for x, y in ((q, qr), (k, kr)):
        want = R.rotary(x.double(), angles, d, "half", 1.0, False)
        assert float(((y.double() - want).abs() - 2 * R.HALF[BF] * want.abs() - 1e-5).max()) <= 0
    ref = R.reference([(qr.double(), kr.double(), v.double(), None)], heads, kv_heads, True, 0, 1.0 / math.sqrt(d), R.HALF[BF])
    close(torch.cat(outs), *ref[0]["out"], "the prompt")


def test_nothing_to_do():
    from r9700training_amd.paged import paged_attention_fwd, paged_write

    c = Cache([10, 20], 2, 64, 16)
    q, k = rnd(1, 2, 0, 4, 64), rnd(2, 2, 0, 2, 64)
    paged_write(k, k, c.k, c.v, c.table, c.kv_lens)
    out, lse = paged_attention_fwd(q, c.k, c.v, c.table, c.kv_lens)
    assert out.shape == (2, 0, 4, 64) and lse.shape == (2, 4, 0)
    empty = torch.empty((0, 3), dtype=torch.int32, device="cuda")
    out, _ = paged_attention_fwd(rnd(1, 0, 5, 4, 64), c.k, c.v, empty, c.kv_lens[:0])
    assert out.shape == (0, 5, 4, 64)
    # a cache without a page
    none = c.k[:0]
    out, lse = paged_attention_fwd(rnd(1, 2, 3, 4, 64), none, none, c.table, c.kv_lens, out_dtype=torch.float32)
    assert (out == 0).all()
    # a table without an entry
    out, lse = paged_attention_fwd(rnd(1, 2, 3, 4, 64), c.k, c.v, c.table[:, :0], c.kv_lens)
    assert (out == 0).all() and (lse == -math.inf).all()


def past(new, lens, heads, d, page, entries, packed=False, dtype=BF):
    """Pools of finite values, new tokens of sequences whose table has so many entries, and the pools after the write."""
    pages = len(lens) * entries + 2
    pools = [rnd(60 + i, pages, page, heads, d) for i in range(2)]
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(5))[:len(lens) * entries].reshape(len(lens), entries)
    starts = torch.tensor([0] + list(new)).cumsum(0)
    shape = (int(starts[-1]), heads, d) if packed else (len(new), new[0], heads, d)
    k, v = rnd(70, *shape, dtype=dtype), rnd(71, *shape, dtype=dtype)
    want = [t.clone() for t in pools]
    for b, (n, m) in enumerate(zip(new, lens)):
        mine = [t[starts[b]:starts[b + 1]] if packed else t[b] for t in (k, v)]
        for i in range(n):
            at = m - n + i
            if 0 <= at < entries * page:
                for w, t in zip(want, mine):
                    w[int(ids[b, at // page]), at % page] = t[i].to(BF)
    kw = dict(q_starts=starts.to(torch.int32).cuda(), max_q=max(new)) if packed else {}
    return k, v, pools, want, ids.to(torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), kw


@pytest.mark.parametrize("new,lens,page,entries,packed", [
    ([1, 1, 1], [33, 32, 2 ** 31 - 1], 16, 2, False),     # one past the table's room, its last place, and far past it
    ([5, 5, 5], [34, 37, 38], 16, 2, False),              # the last two, all and all without a place
    ([40, 3, 1], [60, 50, 49], 8, 6, True),
    ([300, 1], [1100, 1025], 128, 8, True),
])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_write_past_the_table(new, lens, page, entries, packed, dtype):
    """A token whose position the table has no entry for is left out, and moves no other."""
    from r9700training_amd.paged import paged_write

    for heads, d in ((2, 64), (3, 80)):
        k, v, pools, want, ids, held, kw = past(new, lens, heads, d, page, entries, packed, dtype)
        paged_write(k, v, *pools, ids, held, **kw)
        torch.cuda.synchronize()
        for got, w in zip(pools, want):
            assert torch.equal(got.view(torch.int16), w.view(torch.int16))


def test_tokens_past_the_tables_room():
    """A captured step of one token that is replayed until its cache is full, and on: what the cache holds stays."""
    from r9700training_amd.paged import paged_write

    k, v, pools, _, ids, held, _ = past([1, 1], [30, 31], 2, 64, 16, 2)
    paged_write(k, v, *pools, ids, held)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held.add_(1)
        paged_write(k, v, *pools, ids, held)
    held.copy_(torch.tensor([30, 31], dtype=torch.int32, device="cuda"))
    want = [t.clone() for t in pools]
    for i in range(6):
        k.copy_(rnd(80 + i, 2, 1, 2, 64)), v.copy_(rnd(90 + i, 2, 1, 2, 64))
        for b in range(2):
            at = 30 + b + i
            if at < 32:
                want[0][int(ids[b, 1]), at % 16], want[1][int(ids[b, 1]), at % 16] = k[b, 0], v[b, 0]
        g.replay()
        torch.cuda.synchronize()
        for got, w in zip(pools, want):
            assert torch.equal(got.view(torch.int16), w.view(torch.int16)), i


@pytest.mark.parametrize("page", [8, 16])
@pytest.mark.parametrize("new,d", [(1, 80), (100, 80), (1, 40), (90, 40), (1, 200), (70, 200), (100, 128)])
def test_a_pool_just_under_2_GiB(new, d, page):
    """Heads of fewer columns than their tile, in pages smaller than it: the columns past a head are zeros whatever the pool's
    last pages hold, also where a tile's later places name the pool's first pages."""
    from r9700training_amd.paged import paged_attention_fwd

    heads, n = 8, 8 * page
    pages = 0x7FFFFFF0 // (2 * page * heads * d)
    k, v = (torch.zeros((pages, page, heads, d), dtype=BF, device="cuda") for _ in range(2))
    k[8:], v[8:] = math.nan, math.nan
    k[:8], v[:8] = rnd(1, 8, page, heads, d), rnd(2, 8, page, heads, d)
    ids = torch.tensor([[7, 0, 1, 2, 3, 4, 5, 6], [1, 0, 3, 2, 5, 4, 7, 6]], dtype=torch.int32, device="cuda")
    q = rnd(3, 2, new, heads, d)
    held = torch.full((2,), n, dtype=torch.int32, device="cuda")
    ref = R.reference([(q[b].double(), k[ids[b].long()].flatten(0, 1).double(), v[ids[b].long()].flatten(0, 1).double(), None)
                       for b in range(2)], heads, heads, True, 0, 0.1, R.HALF[BF])
    out, lse = paged_attention_fwd(q, k, v, ids, held, scale=0.1)
    torch.cuda.synchronize()
    for b, r in enumerate(ref):
        close(out[b], *r["out"], f"out of sequence {b}")
        close(lse[b], *r["lse"], f"lse of sequence {b}")


@pytest.mark.parametrize("new,n,hq,hk,d", [(1, 20000, 24, 4, 256), (2, 6000, 8, 2, 128), (1, 3000, 4, 4, 64), (64, 9000, 16, 4, 64), (1, 300, 4, 2, 64)])
def test_a_nan_query_in_ranges(new, n, hq, hk, d):
    """A row whose scores are all NaN is NaN, in one range of the keys or many, over pages and over rows; so is one whose keys
    are, if only in some of the ranges. The other rows are what they are without it."""
    from r9700training_amd.attention import attention_fwd
    from r9700training_amd.paged import paged_attention_fwd

    c = Cache([n, n], hk, d, 16)
    k, v = torch.stack(c.keys), torch.stack(c.values)
    q = rnd(1, 2, new, hq, d)
    bad = q.clone()
    bad[0, new - 1, hq - 1] = math.nan
    ref = expected(c, q, hq, hk, True, 0, 0.1, R.HALF[BF])
    for out, lse in (paged_attention_fwd(bad, c.k, c.v, c.table, c.kv_lens, scale=0.1), attention_fwd(bad, k, v, scale=0.1)):
        assert out[0, new - 1, hq - 1].isnan().all() and lse[0, hq - 1, new - 1].isnan()
        for b, r in enumerate(ref):
            (want, tol), (want_lse, tol_lse) = (tuple(t.clone() for t in r[name]) for name in ("out", "lse"))
            o, s = out[b].clone(), lse[b].clone()
            if b == 0:
                for t in (want, tol, o):
                    t[new - 1, hq - 1] = 0
                for t in (want_lse, tol_lse, s):
                    t[hq - 1, new - 1] = 0
            close(o, want, tol, f"out of sequence {b}")
            close(s, want_lse, tol_lse, f"lse of sequence {b}")
    # every key of a part of the cache, some ranges' whole
    k[0, :n // 2, 0] = math.nan
    for b in range(n // 2 // 16):
        c.k[int(c.table[0, b]), :, 0] = math.nan
    for out, lse in (paged_attention_fwd(q, c.k, c.v, c.table, c.kv_lens, scale=0.1), attention_fwd(q, k, v, scale=0.1)):
        assert out[0, :, :hq // hk].isnan().all() and lse[0, :hq // hk].isnan().all()
        assert out[1].isfinite().all() and out[0, :, hq // hk:].isfinite().all()
