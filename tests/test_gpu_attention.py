"""Attention's forward and backward against float64, at the lengths, head groups, masks and layouts where they
can go wrong. Every tolerance counts roundings at half a step (tests/between_ref.py)."""
import math

import pytest
import torch

import between_ref as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def rnd(seed, *shape, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (std * torch.randn(shape, generator=g, device="cuda")).to(BF)


def close(got, want, tol, what):
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin), f"{what}: other places are finite"
    assert torch.equal(got[~fin], want[~fin]), what
    off = (got - want).abs()[fin] - tol[fin]
    worst = float(off.max()) if off.numel() else -1.0
    print(f"{what}: largest |error| / tolerance {float(((got - want).abs()[fin] / (tol[fin] + 1e-300)).max()) if off.numel() else 0:.3f}",
          flush=True)
    # values that underflow: an absolute floor far below any of the inputs' products
    assert worst <= 1e-30, f"{what}: {worst} past the tolerance"


def run(q, k, v, do, seqs, heads, kv_heads, causal, window, scale, out_dtype=BF, grad_dtype=BF, back=True, **kw):
    """Both directions through the package, against the reference of the sequences `seqs`: (query rows, key rows,
    index) of each, as functions on the tensors."""
    from r9700training_amd.attention import attention_bwd, attention_fwd

    out, lse = attention_fwd(q, k, v, causal=causal, window=window, scale=scale, out_dtype=out_dtype, **kw)
    ref = R.reference([(s.q(q).double(), s.k(k).double(), s.k(v).double(), s.q(do).double() if back else None) for s in seqs],
                      heads, kv_heads, causal, window, scale, R.HALF[out_dtype], R.HALF[grad_dtype])
    torch.cuda.synchronize()
    for i, (s, r) in enumerate(zip(seqs, ref)):
        close(s.q(out), *r["out"], f"out of sequence {i}")
        close(s.stat(lse), *r["lse"], f"lse of sequence {i}")
    if not back:
        return out, lse
    dq, dk, dv = attention_bwd(q, k, v, out, lse, do, causal=causal, window=window, scale=scale, grad_dtype=grad_dtype, **kw)
    torch.cuda.synchronize()
    for i, (s, r) in enumerate(zip(seqs, ref)):
        close(s.q(dq), *r["dq"], f"dq of sequence {i}")
        close(s.k(dk), *r["dk"], f"dk of sequence {i}")
        close(s.k(dv), *r["dv"], f"dv of sequence {i}")
    return out, lse, dq, dk, dv


class Dense:
    def __init__(self, b, lk):
        self.b, self.lk = b, lk

    def q(self, x):
        return x[self.b]

    def k(self, x):
        return x[self.b, :self.lk]

    def stat(self, x):
        return x[self.b]


class Packed:
    def __init__(self, q0, q1, k0, k1):
        self.at = (q0, q1, k0, k1)

    def q(self, x):
        return x[self.at[0]:self.at[1]]

    def k(self, x):
        return x[self.at[2]:self.at[3]]

    def stat(self, x):
        return x[:, self.at[0]:self.at[1]]


DENSE = [
    # batch, q_len, kv_len, q_heads, kv_heads, head_dim, causal, window
    (1, 1, 1, 1, 1, 64, True, 0),
    (2, 1, 77, 4, 1, 64, True, 0),
    (1, 1, 1000, 6, 1, 128, True, 0),
    (2, 1, 513, 24, 4, 256, True, 0),
    (1, 3, 200, 14, 2, 128, True, 0),
    (1, 31, 31, 2, 2, 64, True, 0),
    (1, 32, 32, 2, 1, 128, True, 0),
    (1, 33, 65, 3, 1, 80, True, 0),
    (2, 128, 128, 8, 2, 64, True, 0),
    (1, 129, 129, 4, 2, 128, True, 0),
    (1, 255, 257, 2, 1, 256, True, 0),
    (1, 300, 300, 2, 2, 64, False, 0),
    (1, 100, 37, 3, 3, 128, False, 0),
    (1, 97, 40, 2, 1, 64, True, 0),       # the first 57 queries see nothing
    (1, 200, 1, 2, 2, 256, True, 0),
    (2, 70, 0, 4, 2, 64, True, 0),        # no keys at all
    (1, 190, 190, 2, 1, 64, True, 1),     # each query its own key
    (1, 190, 260, 2, 1, 128, True, 50),
    (1, 260, 200, 4, 4, 256, True, 33),
    (2, 400, 400, 6, 2, 64, True, 128),
    (1, 65, 65, 2, 1, 8, True, 0),
    (1, 65, 70, 2, 2, 40, True, 0),
    (1, 40, 40, 7, 1, 248, True, 0),
    (1, 50, 90, 5, 1, 72, False, 0),
    (3, 5, 2000, 8, 2, 64, True, 0),
    (1, 520, 520, 12, 2, 128, True, 0),
]


@pytest.mark.parametrize("b,lq,lk,hq,hk,d,causal,window", DENSE)
def test_dense(b, lq, lk, hq, hk, d, causal, window):
    print(f"case dense {(b, lq, lk, hq, hk, d, causal, window)}", flush=True)
    q, do = rnd(1, b, lq, hq, d), rnd(4, b, lq, hq, d)
    k, v = rnd(2, b, lk, hk, d), rnd(3, b, lk, hk, d)
    run(q, k, v, do, [Dense(i, lk) for i in range(b)], hq, hk, causal, window, 1.0 / math.sqrt(d))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_f32_outputs(d):
    q, do = rnd(1, 2, 150, 4, d), rnd(4, 2, 150, 4, d)
    k, v = rnd(2, 2, 150, 2, d), rnd(3, 2, 150, 2, d)
    run(q, k, v, do, [Dense(i, 150) for i in range(2)], 4, 2, True, 0, 0.1, out_dtype=torch.float32, grad_dtype=torch.float32)


PACKED = [
    # query lengths, key lengths, q_heads, kv_heads, head_dim, causal, window
    ([1, 129, 0, 64, 37], None, 4, 2, 64, True, 0),
    ([300, 5, 1, 211], None, 4, 1, 128, True, 0),
    ([130, 131], None, 2, 2, 256, True, 100),
    ([1, 1, 3, 1], [500, 1, 90, 33], 8, 2, 128, True, 0),
    ([40, 20, 7], [0, 20, 3], 2, 1, 64, True, 0),
    ([64, 65], [100, 10], 2, 1, 80, False, 0),
]


@pytest.mark.parametrize("lq,lk,hq,hk,d,causal,window", PACKED)
def test_packed(lq, lk, hq, hk, d, causal, window):
    print(f"case packed {(lq, lk, hq, hk, d, causal, window)}", flush=True)
    lk = lq if lk is None else lk
    qs = torch.tensor([0] + lq).cumsum(0).to(torch.int32).cuda()
    ks = torch.tensor([0] + lk).cumsum(0).to(torch.int32).cuda()
    q, do = rnd(1, sum(lq), hq, d), rnd(4, sum(lq), hq, d)
    k, v = rnd(2, sum(lk), hk, d), rnd(3, sum(lk), hk, d)
    seqs, a, b = [], 0, 0
    for x, y in zip(lq, lk):
        seqs.append(Packed(a, a + x, b, b + y))
        a, b = a + x, b + y
    run(q, k, v, do, seqs, hq, hk, causal, window, 1.0 / math.sqrt(d), q_starts=qs, kv_starts=ks, max_q=max(lq), max_kv=max(lk))


@pytest.mark.parametrize("lq", [1, 2, 40])
def test_cache_lengths(lq):
    """A cache longer than what is in use, its unused places NaN: they are not read."""
    lens = [0, 1, 64, 65, 300, 299]
    q, do = rnd(1, 6, lq, 8, 128), rnd(4, 6, lq, 8, 128)
    k, v = rnd(2, 6, 300, 2, 128), rnd(3, 6, 300, 2, 128)
    for i, n in enumerate(lens):
        k[i, n:] = float("nan")
        v[i, n:] = float("nan")
    got = run(q, k, v, do, [Dense(i, n) for i, n in enumerate(lens)], 8, 2, True, 0, 0.09,
              kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    for g in got[3:]:
        for i, n in enumerate(lens):
            assert torch.equal(g[i, n:], torch.zeros_like(g[i, n:]))


def test_packed_queries_over_a_cache():
    """New tokens of several sequences packed, each against its own part of a dense cache."""
    from r9700training_amd.attention import attention_fwd

    lq, lens = [5, 1, 17], [90, 33, 17]
    qs = torch.tensor([0, 5, 6, 23], dtype=torch.int32, device="cuda")
    q, k, v = rnd(1, 23, 4, 64), rnd(2, 3, 96, 2, 64), rnd(3, 3, 96, 2, 64)
    out, lse = attention_fwd(q, k, v, q_starts=qs, max_q=17, kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    ref = R.reference([(q[a:a + n].double(), k[i, :m].double(), v[i, :m].double(), None)
                       for i, (a, n, m) in enumerate(zip((0, 5, 6), lq, lens))], 4, 2, True, 0, 0.125, R.HALF[BF])
    for (a, n), r in zip(((0, 5), (5, 1), (6, 17)), ref):
        close(out[a:a + n], *r["out"], "out")
        close(lse[:, a:a + n], *r["lse"], "lse")


def test_longest_too_short_and_bad_starts():
    """The longest length only sizes the launch; starts that leave the tensors are clamped to them."""
    from r9700training_amd.attention import attention_bwd, attention_fwd

    q, k, v, do = (rnd(i, 300, 2, 64) for i in range(4))
    good = torch.tensor([0, 200, 300], dtype=torch.int32, device="cuda")
    a = attention_fwd(q, k, v, q_starts=good, kv_starts=good, max_q=200, max_kv=200)
    b = attention_fwd(q, k, v, q_starts=good, kv_starts=good, max_q=60, max_kv=10)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x = attention_bwd(q, k, v, a[0], a[1], do, q_starts=good, kv_starts=good, max_q=200, max_kv=200)
    y = attention_bwd(q, k, v, a[0], a[1], do, q_starts=good, kv_starts=good, max_q=60, max_kv=10)
    assert all(torch.equal(m, n) for m, n in zip(x, y))
    wild = torch.tensor([-7, 200, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    c = attention_fwd(q, k, v, q_starts=wild, kv_starts=wild, max_q=200, max_kv=200)
    assert torch.equal(a[0], c[0])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_layouts(d):
    """Views of a fused projection, of a [batch, heads, tokens, head_dim] cache, and a key broadcast over the batch
    give the bits of the contiguous tensors; gradients may go into such views."""
    from r9700training_amd.attention import attention_bwd, attention_fwd

    b, n, hq, hk = 2, 150, 4, 2
    fused = rnd(1, b, n, (hq + 2 * hk) * d)
    q = fused[..., :hq * d].unflatten(-1, (hq, d))
    k = fused[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    v = fused[..., (hq + hk) * d:].unflatten(-1, (hk, d))
    do = rnd(2, b, hq, n, d).transpose(1, 2)
    want, lse = attention_fwd(q.contiguous(), k.contiguous(), v.contiguous())
    out = torch.full((b, hq, n, d), float("nan"), dtype=BF, device="cuda").transpose(1, 2)
    got, lse2 = attention_fwd(q, k, v, out=out)
    assert torch.equal(got, want) and torch.equal(lse, lse2)
    grads = attention_bwd(q.contiguous(), k.contiguous(), v.contiguous(), want, lse, do.contiguous())
    into = torch.full_like(fused, float("nan"))
    parts = [into[..., :hq * d].unflatten(-1, (hq, d)), into[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d)),
             into[..., (hq + hk) * d:].unflatten(-1, (hk, d))]
    got = attention_bwd(q, k, v, out, lse, do, dq=parts[0], dk=parts[1], dv=parts[2])
    assert all(torch.equal(x, y) for x, y in zip(got, grads))
    one = k[:1].expand(b, n, hk, d)
    x = attention_fwd(q, one, v)
    y = attention_fwd(q, one.contiguous(), v)
    assert torch.equal(x[0], y[0])
    gx = attention_bwd(q, one, v, *x, do)
    gy = attention_bwd(q, one.contiguous(), v, *x, do)
    assert all(torch.equal(m, n) for m, n in zip(gx, gy))


@pytest.mark.parametrize("d,lq,lk", [(64, 130, 130), (128, 1, 700), (256, 70, 200)])
def test_steep_scores(d, lq, lk):
    """Scores of hundreds, rising along the keys so that the running maximum moves at every tile, and falling."""
    for rise in (1.0, -1.0):
        q = torch.ones((1, lq, 2, d), device="cuda").to(BF)
        ramp = rise * torch.arange(lk, device="cuda", dtype=torch.float32)[None, :, None, None] * 0.5
        k = (ramp.expand(1, lk, 1, d) / d + 0.01 * rnd(2, 1, lk, 1, d).float()).to(BF)
        run(q, k, rnd(3, 1, lk, 1, d), rnd(4, 1, lq, 2, d), [Dense(0, lk)], 2, 1, False, 0, 1.0)


def test_scale_zero_and_negative():
    for scale in (0.0, -0.2):
        run(rnd(1, 1, 90, 2, 64), rnd(2, 1, 90, 2, 64), rnd(3, 1, 90, 2, 64), rnd(4, 1, 90, 2, 64), [Dense(0, 90)], 2, 2, True, 0, scale)


def test_long_cache_offsets():
    """Keys whose byte offsets pass 32 bits: the last tokens of a cache of 9 x 2^30 bytes in one tensor."""
    from r9700training_amd.attention import attention_fwd

    n, d = 36000, 128
    k = torch.zeros((1, n, 1024, d), dtype=BF, device="cuda")[:, :, 1000:1001]  # a token 256 KiB from the next
    v = torch.zeros((1, n, 1024, d), dtype=BF, device="cuda")[:, :, 1000:1001]
    k.copy_(rnd(2, 1, n, 1, d))
    v.copy_(rnd(3, 1, n, 1, d))
    q = rnd(1, 1, 2, 4, d)
    got, lse = attention_fwd(q, k, v)
    want, lse2 = attention_fwd(q, k.contiguous(), v.contiguous())
    assert torch.equal(got, want) and torch.equal(lse, lse2)
    run(q, k.contiguous(), v.contiguous(), None, [Dense(0, n)], 4, 1, True, 0, 1.0 / math.sqrt(d), back=False)


def test_same_bits_and_graph_replay():
    """Repeated calls give the same bits, also on another stream, and captured into a graph and replayed with
    eager work between the replays."""
    from r9700training_amd.attention import attention_bwd, attention_fwd

    cases = [(1, 300, 300, 8, 2, 128), (2, 1, 900, 8, 2, 64), (1, 64, 64, 4, 4, 256)]
    for b, lq, lk, hq, hk, d in cases:
        q, k, v, do = rnd(1, b, lq, hq, d), rnd(2, b, lk, hk, d), rnd(3, b, lk, hk, d), rnd(4, b, lq, hq, d)

        def step():
            out, lse = attention_fwd(q, k, v)
            return (out, lse) + attention_bwd(q, k, v, out, lse, do)

        want = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = step()
            step()
        o2, l2 = attention_fwd(q, k, v, stream=side)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, again)) and torch.equal(o2, want[0]) and torch.equal(l2, want[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for seed in (11, 12, 13):
            q.copy_(rnd(seed, b, lq, hq, d))
            want = [x.clone() for x in step()]
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(want, held)), seed


def test_gradient_against_differences():
    """The kernels' gradient along a direction against the kernels' own forward, f32 out. The forward's outputs are off by at
    most 2^-8 of sum p |v| each, so the quotient by twice that over the step, and by the third derivative's
    step^2 (a step of 1/16 of inputs of size 1 under a scale of 1/8)."""
    from r9700training_amd.attention import attention_bwd, attention_fwd

    q, k, v, do = rnd(1, 1, 64, 2, 64), rnd(2, 1, 64, 1, 64), rnd(3, 1, 64, 1, 64), rnd(4, 1, 64, 2, 64)
    out, lse = attention_fwd(q, k, v, out_dtype=torch.float32)
    grads = attention_bwd(q, k, v, out, lse, do, grad_dtype=torch.float32)
    for name, x, g in zip("qkv", (q, k, v), grads):
        # a direction along the gradient's signs: the quotient is a sum of like terms, far above the roundings
        u = torch.sign(g) / 16
        hi, lo = (x.float() + u).to(BF), (x.float() - u).to(BF)
        moved = (hi.double() - lo.double()) / 2
        args = {n: t for n, t in zip("qkv", (q, k, v))}
        f = []
        for y in (hi, lo):
            o, _ = attention_fwd(*({**args, name: y}[n] for n in "qkv"), out_dtype=torch.float32)
            f.append(float((o.double() * do.double()).sum()))
        want = float((g.double() * moved).sum())
        got = (f[0] - f[1]) / 2
        noise = 2 ** -8 * float((do.double().abs() * v.double().abs().mean()).sum()) / math.sqrt(do.numel())
        assert abs(got - want) <= 0.02 * abs(want) + 4 * noise, (name, got, want, noise)


CUT = [
    # few workgroups over many keys: ranges of the keys joined, dQ's and dK's sums cut; the probabilities computed again
    (1, 40, 1200, 4, 2, 128, True, 0),
    (1, 64, 2100, 4, 1, 256, True, 0),
    (2, 33, 1500, 6, 2, 128, False, 0),
    (1, 90, 3000, 2, 1, 64, True, 1500),
    (1, 70, 2500, 4, 2, 128, True, 1100),
    (1, 1, 1500, 6, 1, 256, True, 0),
    (1, 3, 5000, 8, 1, 128, True, 1300),
    (2, 5, 2600, 12, 2, 80, True, 0),
    (1, 40, 1100, 2, 2, 8, True, 0),
    # dS^T kept: heads of 128 and 256, whole and ragged blocks, a window, queries without keys
    (1, 700, 700, 4, 2, 128, True, 0),
    (2, 260, 390, 6, 2, 256, True, 0),
    (1, 500, 500, 2, 1, 128, True, 70),
    (1, 400, 300, 2, 2, 256, True, 130),
    (1, 333, 200, 4, 1, 128, False, 0),
    (1, 200, 450, 3, 1, 200, False, 0),
]


@pytest.mark.parametrize("b,lq,lk,hq,hk,d,causal,window", CUT)
def test_cut_and_kept(b, lq, lk, hq, hk, d, causal, window):
    print(f"case cut {(b, lq, lk, hq, hk, d, causal, window)}", flush=True)
    q, do = rnd(1, b, lq, hq, d), rnd(4, b, lq, hq, d)
    k, v = rnd(2, b, lk, hk, d), rnd(3, b, lk, hk, d)
    run(q, k, v, do, [Dense(i, lk) for i in range(b)], hq, hk, causal, window, 1.0 / math.sqrt(d))


@pytest.mark.parametrize("d", [128, 256])
def test_packed_many(d):
    """Packed sequences of every length around the tiles, their kept dS^T beside one another."""
    lens = [1, 63, 64, 65, 127, 128, 129, 7, 0, 250, 33, 2]
    at = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    n = sum(lens)
    q, k, v, do = rnd(1, n, 4, d), rnd(2, n, 2, d), rnd(3, n, 2, d), rnd(4, n, 4, d)
    seqs = [Packed(int(at[i]), int(at[i + 1]), int(at[i]), int(at[i + 1])) for i in range(len(lens))]
    run(q, k, v, do, seqs, 4, 2, True, 0, 1.0 / math.sqrt(d), q_starts=at, kv_starts=at, max_q=250, max_kv=250)


@pytest.mark.parametrize("heads,n,d", [(16, 8300, 256), (16, 4300, 128)])
def test_too_long_to_keep(heads, n, d):
    """dS^T past what is kept: the probabilities are computed again. Two heads are checked, at rows of every part."""
    from r9700training_amd.attention import attention_bwd, attention_fwd

    q, k, v, do = (rnd(i, 1, n, heads, d) for i in range(1, 5))
    out, lse = attention_fwd(q, k, v)
    grads = attention_bwd(q, k, v, out, lse, do)
    for h in (0, heads - 1):
        one = [t[0, :, h:h + 1].double() for t in (q, k, v, do)]
        r = R.reference([tuple(one)], 1, 1, True, 0, 1.0 / math.sqrt(d), R.HALF[BF], R.HALF[BF])[0]
        close(out[0, :, h:h + 1], *r["out"], f"out of head {h}")
        for name, g in zip(("dq", "dk", "dv"), grads):
            close(g[0, :, h:h + 1], *r[name], f"{name} of head {h}")


def test_ragged_cache_of_many_keys():
    """A serving batch whose lengths differ by thousands: ranges with nothing in them, and places never written."""
    lens = [3000, 1, 0, 1025, 2047, 130]
    q, k, v = rnd(1, 6, 1, 8, 256), rnd(2, 6, 3000, 2, 256), rnd(3, 6, 3000, 2, 256)
    for i, n in enumerate(lens):
        k[i, n:] = float("nan")
        v[i, n:] = float("nan")
    run(q, k, v, None, [Dense(i, n) for i, n in enumerate(lens)], 8, 2, True, 0, 0.06, back=False,
        kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))


def test_workspace_of_a_larger_call_and_full_of_nan():
    """A workspace holds nothing between calls: one full of NaN, and larger than asked for, gives the same bits."""
    from r9700training_amd import lib
    from r9700training_amd.attention import attention_bwd, attention_fwd

    for lq, lk, d in ((700, 700, 128), (40, 2000, 128), (1, 4000, 256), (300, 300, 64)):
        q, k, v, do = rnd(1, 1, lq, 8, d), rnd(2, 1, lk, 2, d), rnd(3, 1, lk, 2, d), rnd(4, 1, lq, 8, d)
        out, lse = attention_fwd(q, k, v)
        grads = attention_bwd(q, k, v, out, lse, do)
        ws = torch.full((1 << 26,), float("nan"), device="cuda").view(torch.uint8)
        o2, l2 = attention_fwd(q, k, v, workspace=ws)
        assert torch.equal(out, o2) and torch.equal(lse, l2)
        ws.view(torch.float32).fill_(float("nan"))
        g2 = attention_bwd(q, k, v, out, lse, do, workspace=ws)
        assert all(torch.equal(x, y) for x, y in zip(grads, g2))
    assert lib() is not None


def test_kept_graph_and_stream():
    """The backward that keeps dS^T, on another stream and replayed from a graph with eager work between the replays."""
    from r9700training_amd.attention import attention_bwd, attention_fwd

    q, k, v, do = rnd(1, 2, 500, 8, 128), rnd(2, 2, 500, 2, 128), rnd(3, 2, 500, 2, 128), rnd(4, 2, 500, 8, 128)

    def step(**kw):
        out, lse = attention_fwd(q, k, v, **kw)
        return (out, lse) + attention_bwd(q, k, v, out, lse, do, **kw)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(stream=side)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (21, 22, 23):
        do.copy_(rnd(seed, 2, 500, 8, 128))
        want = [x.clone() for x in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, held)), seed


@pytest.mark.parametrize("d", [64, 128, 256])
def test_longest_of_nothing(d):
    """A longest length of 0 is only a wrong one: cut along the keys or not, the results are those of the right one."""
    from r9700training_amd.attention import attention_bwd, attention_fwd

    lq, lk = [3, 1, 40], [4000, 900, 1300]
    qs = torch.tensor([0, 3, 4, 44], dtype=torch.int32, device="cuda")
    ks = torch.tensor([0, 4000, 4900, 6200], dtype=torch.int32, device="cuda")
    q, do = rnd(1, 44, 4, d), rnd(4, 44, 4, d)
    k, v = rnd(2, 6200, 2, d), rnd(3, 6200, 2, d)
    seqs = [Packed(a, a + n, b, b + m) for a, n, b, m in zip((0, 3, 4), lq, (0, 4000, 4900), lk)]
    got = run(q, k, v, do, seqs, 4, 2, True, 0, 1.0 / math.sqrt(d), q_starts=qs, kv_starts=ks, max_q=0, max_kv=0)
    one = attention_fwd(q, k, v, q_starts=qs, kv_starts=ks, max_q=1, max_kv=1)
    assert torch.equal(got[0], one[0]) and torch.equal(got[1], one[1])
    grads = attention_bwd(q, k, v, *one, do, q_starts=qs, kv_starts=ks, max_q=1, max_kv=1)
    assert all(torch.equal(x, y) for x, y in zip(got[2:], grads))


def test_a_grid_cut_short():
    """A longest length far past the real ones asks for more workgroups than a launch takes: the workgroups there are take
    more tiles each, and the bits are those of the right length."""
    from r9700training_amd.attention import attention_bwd, attention_fwd

    lens = [1 + i % 3 for i in range(1023)] + [300]
    at = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    n = sum(lens)
    q, k, v, do = rnd(1, n, 32, 64), rnd(2, n, 8, 64), rnd(3, n, 8, 64), rnd(4, n, 32, 64)
    out = {}
    for longest in (300, 131072):
        print(f"case longest {longest}", flush=True)
        kw = dict(q_starts=at, kv_starts=at, max_q=longest, max_kv=longest)
        o, lse = attention_fwd(q, k, v, **kw)
        out[longest] = (o, lse) + attention_bwd(q, k, v, o, lse, do, **kw)
        torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(out[300], out[131072]))


PACKED_CUT = [
    # query lengths, key lengths, q_heads, kv_heads, causal, window: the mean of the keys is what the cuts go by, so the long
    # sequences' last range takes more than its share, and the short ones leave ranges empty
    ([1, 3, 1], [5000, 1, 1700], 8, 2, True, 0),
    ([40, 70], [4500, 300], 4, 2, True, 0),
    ([5, 0, 33, 2], [0, 1500, 7000, 40], 6, 2, True, 0),
    ([40, 70], [4500, 300], 4, 1, False, 0),
    ([60, 90], [3000, 5000], 2, 1, True, 2100),
    ([200, 3], [2500, 2400], 2, 2, True, 0),
]


def cut_of(lq, lk, hq, hk, d, causal, window):
    """Whether the forward's keys and dQ's keys are cut, from the sizes of the workspaces."""
    from r9700training_amd import AttnShape, lib

    s = AttnShape(batch=len(lq), head_dim=d, q_len=max(lq), kv_len=max(lk), q_starts=1 << 20, kv_starts=1 << 20, q_tokens=sum(lq),
                  kv_tokens=sum(lk), causal=causal, window=window, scale=1.0)
    slots = hq * sum(lq)
    parts = lib().r97q_attn_bwd_workspace_bytes(s, hq, hk) - (8 * slots + 255) // 256 * 256
    return lib().r97q_attn_fwd_workspace_bytes(s, hq, hk) > 0, parts >= 2 * slots * d * 4


@pytest.mark.parametrize("lq,lk,hq,hk,causal,window", PACKED_CUT)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_packed_and_cut(lq, lk, hq, hk, d, causal, window):
    print(f"case packed cut {(lq, lk, hq, hk, d, causal, window)}", flush=True)
    assert all(cut_of(lq, lk, hq, hk, d, causal, window))
    qs = torch.tensor([0] + lq).cumsum(0).to(torch.int32).cuda()
    ks = torch.tensor([0] + lk).cumsum(0).to(torch.int32).cuda()
    q, do = rnd(1, sum(lq), hq, d), rnd(4, sum(lq), hq, d)
    k, v = rnd(2, sum(lk), hk, d), rnd(3, sum(lk), hk, d)
    seqs, a, b = [], 0, 0
    for x, y in zip(lq, lk):
        seqs.append(Packed(a, a + x, b, b + y))
        a, b = a + x, b + y
    run(q, k, v, do, seqs, hq, hk, causal, window, 1.0 / math.sqrt(d), q_starts=qs, kv_starts=ks, max_q=max(lq), max_kv=max(lk))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lq", [1, 40])
def test_cache_cut_with_lengths(lq, d):
    """A dense cache cut along the keys whose sequences end before, inside and after the ranges; its unused places are NaN."""
    lens = [3000, 0, 700, 41, 1537]
    q, do = rnd(1, 5, lq, 4, d), rnd(4, 5, lq, 4, d)
    k, v = rnd(2, 5, 3000, 2, d), rnd(3, 5, 3000, 2, d)
    for i, n in enumerate(lens):
        k[i, n:] = float("nan")
        v[i, n:] = float("nan")
    got = run(q, k, v, do, [Dense(i, n) for i, n in enumerate(lens)], 4, 2, True, 0, 0.09,
              kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    for g in got[3:]:
        for i, n in enumerate(lens):
            assert torch.equal(g[i, n:], torch.zeros_like(g[i, n:]))


UNSEEN = [
    # batch, q_len, kv_len, lengths in use, q_heads, kv_heads, head_dim, window: the first keys are before every window
    (2, 1, 300, [300, 211], 4, 1, 64, 50),
    (2, 1, 5000, [5000, 3333], 8, 2, 128, 1300),
    (1, 5, 4000, [3999], 4, 1, 256, 1001),
    (2, 40, 700, [700, 457], 4, 2, 128, 100),
    (1, 200, 450, [450], 2, 1, 256, 77),
    (1, 200, 450, [449], 2, 1, 64, 77),
    (1, 150, 400, [390], 4, 1, 128, 33),
    (1, 40, 4000, [3990], 2, 1, 64, 1500),
]


@pytest.mark.parametrize("b,lq,lk,lens,hq,hk,d,window", UNSEEN)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_keys_before_every_window(b, lq, lk, lens, hq, hk, d, window, bad):
    """What no query sees is not read into anything, whatever it holds: a cache's expired keys, at any place in a tile."""
    from r9700training_amd.attention import attention_bwd, attention_fwd

    print(f"case unseen {(b, lq, lk, lens, hq, hk, d, window, bad)}", flush=True)
    q, do = rnd(1, b, lq, hq, d), rnd(4, b, lq, hq, d)
    clean = [rnd(2, b, lk, hk, d), rnd(3, b, lk, hk, d)]
    dirty = [t.clone() for t in clean]
    for i, n in enumerate(lens):
        for t, x in ((clean, 0.0), (dirty, bad)):
            for y in t:
                y[i, :n - lq - window + 1] = x
                y[i, n:] = x
    kw = dict(window=window, kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    res = []
    for k, v in (clean, dirty):
        out, lse = attention_fwd(q, k, v, **kw)
        res.append((out, lse) + attention_bwd(q, k, v, out, lse, do, **kw))
    for name, x, y in zip(("out", "lse", "dq", "dk", "dv"), *res):
        assert torch.equal(x, y), name
    for i, n in enumerate(lens):
        for g in res[1][3:]:
            assert not g[i, :n - lq - window + 1].any()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("packed", [False, True])
def test_a_nan_reaches_no_tile_past_its_window(d, packed):
    """A NaN key that the queries 390 .. 489 see: tiles of queries from 512 on begin inside its block of keys and do not see
    it, and are as without it; likewise the gradients of keys that only those queries see."""
    from r9700training_amd.attention import attention_bwd, attention_fwd

    n, window = 700, 100
    q, do = rnd(1, 1, n, 4, d), rnd(4, 1, n, 4, d)
    k, v = rnd(2, 1, n, 2, d), rnd(3, 1, n, 2, d)
    kw = dict(window=window)
    if packed:
        q, k, v, do = (t[0] for t in (q, k, v, do))
        at = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        kw.update(q_starts=at, kv_starts=at, max_q=n, max_kv=n)
    res = []
    for bad in (False, True):
        if bad:
            k, v = k.clone(), v.clone()
            for t in (k, v):
                (t if packed else t[0])[390] = float("nan")
        out, lse = attention_fwd(q, k, v, **kw)
        grads = attention_bwd(q, k, v, out, lse, do, **kw)
        res.append([t if packed else t[0] for t in (out, *grads)] + [(lse if packed else lse[0]).t()])
    for name, x, y in zip(("out", "dq", "dk", "dv", "lse"), *res):
        first = 640 if name in ("dk", "dv") else 512
        assert torch.equal(x[first:], y[first:]), name
        assert torch.equal(x[:256], y[:256]), name
        assert bool(y[400:480].isnan().any()), name


@pytest.mark.parametrize("d", [64, 128, 256])
def test_longest_too_short_and_bad_starts_with_kept_scores(d):
    """Wider heads keep dS^T between the launches, a row of it for each key: neither a longest length that is too small nor
    starts that leave the tensors change the results. (A length of a few rows takes the few rows' forward, which adds in
    another order: held to the reference. Otherwise the bits are the same.)"""
    n = 700
    q, k, v, do = rnd(1, n, 4, d), rnd(2, n, 2, d), rnd(3, n, 2, d), rnd(4, n, 4, d)
    good = torch.tensor([0, 430, 430, n], dtype=torch.int32, device="cuda")
    wild = torch.tensor([-(2 ** 31), 430, 430, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    seqs = [Packed(0, 430, 0, 430), Packed(430, n, 430, n)]
    want = {}
    for starts, longest in ((good, 430), (good, 100), (good, 0), (wild, 430), (wild, 1)):
        got = run(q, k, v, do, seqs, 4, 2, True, 0, 1.0 / math.sqrt(d), q_starts=starts, kv_starts=starts, max_q=longest, max_kv=longest)
        first = want.setdefault(longest > 16, got)
        assert all(torch.equal(x, y) for x, y in zip(first, got)), longest


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("packed", [False, True])
def test_no_queries(d, packed):
    """Nothing to answer: empty outputs, and every key's gradient is zero."""
    from r9700training_amd.attention import attention_bwd, attention_fwd

    q, k, v = rnd(1, 2, 0, 4, d), rnd(2, 2, 150, 2, d), rnd(3, 2, 150, 2, d)
    kw = {}
    if packed:
        q, k, v = q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1)
        kw = dict(q_starts=torch.zeros(3, dtype=torch.int32, device="cuda"), kv_starts=torch.tensor([0, 150, 300], dtype=torch.int32, device="cuda"),
                  max_q=0, max_kv=150)
    for longest in (0, 7):
        if packed:
            kw["max_q"] = longest
        out, lse = attention_fwd(q, k, v, **kw)
        dk, dv = (torch.full_like(k, float("nan")) for _ in range(2))
        dq, dk, dv = attention_bwd(q, k, v, out, lse, q.clone(), dk=dk, dv=dv, **kw)
        assert out.shape == dq.shape == q.shape and not dk.any() and not dv.any()
