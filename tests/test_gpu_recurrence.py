"""The gated recurrence against float64, forward and backward: sequences of no token, one, a tile and thousands, channels off
every piece, both types, packed and dense, gates far to both sides. Every tolerance counts roundings (tests/recurrence_ref.py)."""
import math

import pytest
import torch

import recurrence_ref as R

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
HALF = {t: torch.finfo(t).eps / 2 for t in (BF, F32)}
CHUNK = 128


def rnd(seed, *shape, dtype=F32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (std * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def rates(seed, n):
    """From a memory of thousands of tokens to none."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.exp(math.log(5e-4) + torch.rand(n, generator=g, device="cuda") * math.log(4e4))


def close(got, want, err, half, what):
    assert torch.isfinite(got).all(), what
    off = (got.double() - want).abs()
    tol = err + half * (want.abs() + err)
    if off.numel():
        print(f"{what}: largest |error| / tolerance {float((off / (tol + 1e-300)).max()):.3f}", flush=True)
        assert float((off - tol).max()) <= 1e-30, f"{what}: {float((off - tol).max())} past the tolerance"


def inputs(seed, shape, dtype, gated, batch, channels, std=2.0):
    x, gate = rnd(seed, *shape, dtype=dtype), rnd(seed + 1, *shape, dtype=dtype, std=std)
    gi = rnd(seed + 2, *shape, dtype=dtype) if gated else None
    return x, gate, gi, rates(seed + 3, channels), rnd(seed + 4, batch, channels)


def check(x, gate, gi, rate, h0, d_h, d_last, parts, kw, back=True):
    """Both directions through the package; parts: each sequence's rows, as functions on the tensors."""
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    half = HALF[x.dtype]
    h, last, states = recurrence_fwd(x, gate, rate, gi, h0=h0, want_states=back, **kw)
    torch.cuda.synchronize()
    zeros = torch.zeros(x.shape[-1], dtype=torch.float64, device="cuda")
    args = []
    for b, part in enumerate(parts):
        args.append((part(x).double(), part(gate).double(), rate.double(), None if gi is None else part(gi).double(),
                     zeros if h0 is None else h0[b].double()))
        ref = R.forward(*args[-1])
        close(part(h), *ref["h"], half, f"h of sequence {b}")
        close(last[b], *ref["last"], HALF[F32], f"last of sequence {b}")
    if not back:
        return h, last, states
    got = recurrence_bwd(x, gate, rate, states, d_h, gi, d_last=d_last, **kw)
    torch.cuda.synchronize()
    drate, e_rate = zeros.clone(), zeros.clone()
    for b, part in enumerate(parts):
        ref = R.backward(*args[b], part(d_h).double(), zeros if d_last is None else d_last[b].double())
        for name, t in zip(("dx", "dgate", "dinput_gate"), got):
            if t is not None:
                close(part(t), *ref[name], half, f"{name} of sequence {b}")
        close(got[4][b], *ref["dh0"], HALF[F32], f"dh0 of sequence {b}")
        drate, e_rate = drate + ref["drate"][0], e_rate + ref["drate"][1] + len(parts) * R.U * ref["drate"][0].abs()
    close(got[3], drate, e_rate, HALF[F32], "drate")
    return (h, last, states) + got


DENSE = [
    # batch, tokens, channels, type, gated, h0 and d_last
    (1, 1, 64, BF, True, True),
    (3, 1, 200, F32, True, True),
    (40, 1, 512, BF, True, True),
    (2, 2, 8, BF, False, False),
    (1, 3, 1, F32, True, True),
    (2, 17, 65, BF, True, True),
    (2, 33, 72, F32, False, True),
    (1, 127, 64, BF, True, False),
    (2, 128, 136, BF, False, True),
    (2, 129, 63, F32, True, True),
    (1, 255, 100, BF, True, True),
    (1, 256, 256, F32, True, False),
    (2, 257, 320, BF, True, True),
    (3, 385, 64, F32, False, True),
    (1, 513, 7, BF, True, True),
    (1, 1300, 192, F32, True, True),
    (2, 2048, 128, BF, True, True),
    (1, 5000, 64, BF, True, True),
    (1, 4100, 77, F32, True, True),
    (2, 300, 333, BF, True, True),        # slabs that share lines, dealt by XCD
    (1, 2000, 515, BF, False, True),
    (5, 140, 259, F32, True, True),
    (1, 1700, 1001, F32, True, False),
    (3, 16, 9, BF, True, True),
    (2, 9, 5, F32, True, True),
]


@pytest.mark.parametrize("batch,n,c,dtype,gated,ends", DENSE)
def test_dense(batch, n, c, dtype, gated, ends):
    print(f"case dense {(batch, n, c, dtype, gated, ends)}", flush=True)
    x, gate, gi, rate, h0 = inputs(1, (batch, n, c), dtype, gated, batch, c)
    d_h, d_last = rnd(8, batch, n, c, dtype=dtype), rnd(9, batch, c)
    if not ends:
        h0 = d_last = None
    check(x, gate, gi, rate, h0, d_h, d_last, [lambda t, b=b: t[b] for b in range(batch)], {})


PACKED = [
    ([1, 1, 1], 64, BF, True),
    ([5, 0, 130, 1], 72, F32, True),
    ([300, 128, 0, 0, 129], 128, BF, True),
    ([1000, 1, 4000, 256], 64, F32, False),
    ([3000, 50], 33, BF, False),
    ([0, 0], 64, BF, True),
]


@pytest.mark.parametrize("lens,c,dtype,gated", PACKED)
@pytest.mark.parametrize("most", ["longest", "nothing"])
def test_packed(lens, c, dtype, gated, most):
    """The longest length only plans; tokens outside every sequence keep what they held."""
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    print(f"case packed {(lens, c, dtype, gated, most)}", flush=True)
    starts = [3]
    for n in lens:
        starts.append(starts[-1] + n)
    tokens = starts[-1] + 2
    x, gate, gi, rate, h0 = inputs(1, (tokens, c), dtype, gated, len(lens), c)
    d_h, d_last = rnd(8, tokens, c, dtype=dtype), rnd(9, len(lens), c)
    kw = dict(starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), max_len=max(lens) if most == "longest" else 0)
    parts = [lambda t, a=a, b=b: t[a:b] for a, b in zip(starts, starts[1:])]
    h, last, states, *_ = check(x, gate, gi, rate, h0, d_h, d_last, parts, kw)
    out = [torch.full_like(x, 7.0) for _ in range(4)]
    recurrence_fwd(x, gate, rate, gi, h0=h0, out=out[0], **kw)
    recurrence_bwd(x, gate, rate, states, d_h, gi, dx=out[1], dgate=out[2], dinput_gate=out[3] if gated else None, **kw)
    torch.cuda.synchronize()
    assert torch.equal(out[0][3:-2], h[3:-2])
    for t in out[:4 if gated else 3]:
        assert (t[:3] == 7).all() and (t[-2:] == 7).all()
    # the states kept: each sequence's before its tokens 0, 128, ..
    for b, (a, n) in enumerate(zip(starts, lens)):
        ref = R.forward(x[a:a + n].double(), gate[a:a + n].double(), rate.double(), None if gi is None else gi[a:a + n].double(), h0[b].double())
        at = a // CHUNK + b
        value, err = (t[::CHUNK] for t in ref["before"]) if n else (x[:0].double(), x[:0].double())
        close(states[at:at + len(value)], value, err, HALF[F32], f"states of sequence {b}")


@pytest.mark.parametrize("bad", [[-5, 40, 300], [200, 100, 260], [0, 2 ** 31 - 1, 100], [500, 600, 700], [-(2 ** 31), -1, 0]])
def test_starts_outside_the_tensors(bad):
    """They are clamped: what a sequence of the clamped places gives, and nothing else is touched."""
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    c, tokens = 64, 260
    x, gate, gi, rate, h0 = inputs(1, (tokens, c), BF, True, 2, c)
    room = torch.full((tokens + 64, c), 7.0, dtype=BF, device="cuda")
    kw = dict(starts=torch.tensor(bad, dtype=torch.int32, device="cuda"), max_len=260)
    h, last, states = recurrence_fwd(x, gate, rate, gi, h0=h0, out=room[32:-32], want_states=True, **kw)
    grads = recurrence_bwd(x, gate, rate, states, x, gi, **kw)
    torch.cuda.synchronize()
    assert (room[:32] == 7).all() and (room[-32:] == 7).all()
    touched = torch.zeros(tokens, dtype=torch.bool)
    for b in range(2):
        a = min(max(bad[b], 0), tokens)
        e = min(max(bad[b + 1], a), tokens)
        touched[a:e] = True
        if e == a:
            assert torch.equal(last[b], h0[b]) and (grads[4][b] == 0).all()
    assert (h[~touched.cuda()] == 7).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("batch,n,c", [(2, 70, 64), (1, 300, 136), (3, 1, 128), (1, 3000, 64), (2, 200, 99), (3, 5, 13), (1, 2000, 300)])
def test_layouts(batch, n, c, dtype):
    """Slices of a fused projection's rows, token-major storage, places off 16 bytes, a broadcast sequence, and outputs over
    the inputs give the contiguous call's bits."""
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    x, gate, gi, rate, h0 = inputs(1, (batch, n, c), dtype, True, batch, c)
    d_h, d_last = rnd(8, batch, n, c, dtype=dtype), rnd(9, batch, c)
    h, last, states = recurrence_fwd(x, gate, rate, gi, h0=h0, want_states=True)
    grads = recurrence_bwd(x, gate, rate, states, d_h, gi, d_last=d_last)
    for off in (0, 8, 1):
        fused = torch.zeros((batch, n, 8 * c + 16), dtype=dtype, device="cuda")
        views = [fused[..., off + i * c:off + (i + 1) * c] for i in range(8)]
        for v, t in zip(views, (x, gate, gi, d_h)):
            v.copy_(t)
        got = recurrence_fwd(*views[:2], rate, views[2], h0=h0, out=views[4], want_states=True)
        assert torch.equal(got[0], h) and torch.equal(got[1], last) and torch.equal(got[2], states), off
        mine = recurrence_bwd(*views[:2], rate, got[2], views[3], views[2], d_last=d_last, dx=views[5], dgate=views[6], dinput_gate=views[7])
        for a, b in zip(grads, mine):
            assert torch.equal(a, b), off
        assert torch.equal(views[0], x) and (fused[..., :off] == 0).all() and (fused[..., off + 8 * c:] == 0).all()
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, gate, gi)]
    assert torch.equal(recurrence_fwd(turned[0], turned[1], rate, turned[2], h0=h0)[0], h)
    for over in range(3):
        mine = [x.clone(), gate.clone(), gi.clone()]
        state = h0.clone()
        got = recurrence_fwd(mine[0], mine[1], rate, mine[2], h0=state, last=state, out=mine[over])
        assert torch.equal(got[0], h) and torch.equal(state, last)
    one = recurrence_fwd(x[:1].expand(batch, n, c), gate, rate, gi[:1].expand(batch, n, c))[0]
    assert torch.equal(one, recurrence_fwd(x[:1].repeat(batch, 1, 1), gate, rate, gi[:1].repeat(batch, 1, 1))[0])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,c", [(1, 4099), (3, 261), (300, 65), (700, 1029), (2000, 130)])
def test_in_place_of_odd_widths(n, c, dtype):
    """The state and the outputs over the inputs, where the last piece of channels lies over its neighbour's."""
    from r9700training_amd.recurrence import recurrence_fwd

    x, gate, gi, rate, h0 = inputs(1, (6, n, c), dtype, True, 6, c)
    h, last, _ = recurrence_fwd(x, gate, rate, gi, h0=h0)
    for i in range(6):
        mine, state = [x.clone(), gate.clone(), gi.clone()], h0.clone()
        out = mine[i % 3] if i % 2 else None
        got = recurrence_fwd(*mine[:2], rate, mine[2], h0=state, last=state, out=out)[0]
        assert torch.equal(got, h) and torch.equal(state, last)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cuts", [[1] * 20, [100, 1, 156, 43], [600, 1, 1, 1300]])
def test_continued(dtype, cuts):
    """A sequence in pieces, each from the state the one before it left, is the whole sequence."""
    from r9700training_amd.recurrence import recurrence_fwd

    n, c = sum(cuts), 96
    x, gate, gi, rate, h0 = inputs(1, (2, n, c), dtype, True, 2, c)
    state, outs, at = h0.clone(), [], 0
    for m in cuts:
        part = slice(at, at + m)
        outs.append(recurrence_fwd(x[:, part], gate[:, part], rate, gi[:, part], h0=state, last=state)[0])
        at += m
    h = torch.cat(outs, 1)
    for b in range(2):
        ref = R.forward(x[b].double(), gate[b].double(), rate.double(), gi[b].double(), h0[b].double())
        # each piece's joins anew
        close(h[b], ref["h"][0], ref["h"][1] * (1 + len(cuts)), HALF[dtype], f"h of sequence {b}")
        close(state[b], ref["last"][0], ref["last"][1] * (1 + len(cuts)), HALF[F32], f"last of sequence {b}")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_gates_far_to_both_sides(dtype):
    """Gates from -60 to 60: decays of one, whose gradient has no bound and counts as none, and of the rate's own."""
    n, c = 300, 64
    x, _, gi, rate, h0 = inputs(1, (1, n, c), dtype, True, 1, c)
    gate = torch.linspace(-60, 60, n, device="cuda")[torch.randperm(n, generator=torch.Generator().manual_seed(1))]
    gate = gate[None, :, None].expand(1, n, c).to(dtype).contiguous()
    check(x, gate, gi * 20, rate, h0, rnd(8, 1, n, c, dtype=dtype), rnd(9, 1, c), [lambda t: t[0]], {})


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_rate_of_zero(dtype):
    """Nothing enters and nothing decays; gradients are finite."""
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    x, gate, gi, rate, h0 = inputs(1, (1, 400, 64), dtype, True, 1, 64)
    rate[:32] = 0.0
    gate[:, 7] = -math.inf
    gate[:, 9] = math.inf
    h, last, states = recurrence_fwd(x, gate, rate, gi, h0=h0, want_states=True)
    assert torch.equal(last[0, :32], h0[0, :32]) and torch.equal(h[0, :, :32], h0[0, :32].to(dtype).expand(400, 32))
    d_h = rnd(8, 1, 400, 64, dtype=dtype)
    grads = recurrence_bwd(x, gate, rate, states, d_h, gi)
    for t in grads:
        assert torch.isfinite(t).all()
    assert (grads[0][..., :32] == 0).all() and (grads[1][..., :32] == 0).all() and (grads[2][..., :32] == 0).all()
    total = d_h[0].double().sum(0)
    assert float((grads[4][0].double() - total)[:32].abs().max()) <= 400 * R.U * float(d_h[0].double().abs().sum(0).max())


def test_nan_and_infinity_stay_in_their_channel():
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    for dtype in (BF, F32):
        x, gate, gi, rate, h0 = inputs(1, (2, 700, 128), dtype, True, 2, 128)
        d_h = rnd(8, 2, 700, 128, dtype=dtype)
        want = recurrence_fwd(x, gate, rate, gi, h0=h0, want_states=True)
        wgrads = recurrence_bwd(x, gate, rate, want[2], d_h, gi)
        for t, value in ((0, math.nan), (1, math.nan), (2, math.nan), (0, math.inf)):
            bad = [x.clone(), gate.clone(), gi.clone()]
            bad[t][0, 333, 70] = value
            got = recurrence_fwd(bad[0], bad[1], rate, bad[2], h0=h0, want_states=True)
            grads = recurrence_bwd(bad[0], bad[1], rate, got[2], d_h, bad[2])
            assert not torch.isfinite(got[0][0, 333, 70]) and not torch.isfinite(got[1][0, 70])
            mask = torch.ones(2, 700, 128, dtype=torch.bool, device="cuda")
            mask[0, 333:, 70] = False
            assert torch.equal(got[0][mask], want[0][mask])
            mask[0, :, 70] = False
            for a, b in zip(wgrads[:3], grads[:3]):
                assert torch.equal(a[mask], b[mask])


@pytest.mark.parametrize("n,token_stride", [(2100, 1 << 20), (300, 1 << 23), (5, 1 << 29)])
@pytest.mark.parametrize("batch", [1, 2])
def test_offsets_past_32_bits(batch, n, token_stride):
    """Tokens far apart in one tensor of gigabytes: the bits of rows next to each other."""
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    c = 64
    memory = torch.empty(n * token_stride + 8192, dtype=BF, device="cuda")
    places = iter(range(0, 8192, c))

    def far(t=None):
        at = next(places) * batch
        v = memory.as_strided((batch, n, c), (c, token_stride, 1), at)
        return v.copy_(t) if t is not None else v

    near = [rnd(40 + i, batch, n, c, dtype=BF) for i in range(4)]
    rate, h0, d_last = rates(3, c), rnd(4, batch, c), rnd(5, batch, c)
    h, last, states = recurrence_fwd(near[0], near[1], rate, near[2], h0=h0, want_states=True)
    want = (h, last) + recurrence_bwd(near[0], near[1], rate, states, near[3], near[2], d_last=d_last)
    x, gate, gi, d_h = (far(t) for t in near)
    h, last, states = recurrence_fwd(x, gate, rate, gi, h0=h0, want_states=True, out=far())
    got = (h, last) + recurrence_bwd(x, gate, rate, states, d_h, gi, d_last=d_last, dx=far(), dgate=far(), dinput_gate=far())
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("batch,n,c", [(4, 1, 256), (1, 3000, 64)])
def test_streams_and_graphs(batch, n, c):
    """On a stream of its own, and both directions captured and replayed with the program's own work between, while an eager
    call's tensors live."""
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    x, gate, gi, rate, h0 = inputs(1, (batch, n, c), BF, True, batch, c)
    d_h = rnd(8, batch, n, c, dtype=BF)

    def both(stream=None):
        h, last, states = recurrence_fwd(x, gate, rate, gi, h0=h0, want_states=True, stream=stream)
        return (h, last) + recurrence_bwd(x, gate, rate, states, d_h, gi, d_last=last, stream=stream)

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = both(side)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, both()))
    for i in range(4):
        x.copy_(rnd(20 + i, batch, n, c, dtype=BF)), gate.copy_(rnd(30 + i, batch, n, c, dtype=BF)), h0.add_(1.0)
        want = both()
        g, got = graphs[i % 2]
        for t in got:
            t.fill_(3)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)


def test_nothing_to_do():
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    x, gate, gi, rate, h0 = inputs(1, (3, 0, 64), BF, True, 3, 64)
    h, last, states = recurrence_fwd(x, gate, rate, gi, h0=h0, want_states=True)
    assert h.shape == (3, 0, 64) and torch.equal(last, h0) and states.shape == (3, 0, 64)
    d_last = rnd(9, 3, 64)
    grads = recurrence_bwd(x, gate, rate, states, x, gi, d_last=d_last)
    assert torch.equal(grads[4], d_last) and (grads[3] == 0).all()
    none = rnd(1, 0, 5, 64, dtype=BF)
    h, last, states = recurrence_fwd(none, none, rate, want_states=True)
    grads = recurrence_bwd(none, none, rate, states, none)
    assert last.shape == (0, 64) and (grads[3] == 0).all() and grads[2] is None


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("c", [64, 100, 3])
@pytest.mark.parametrize("most", [1, 300, 2048])
def test_strides_of_a_lone_token(dtype, c, most):
    """A packed token alone, whose rows are as they come of a transposed column or an expanded one: its stride says nothing,
    whatever length is planned for."""
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    x, gate, gi, rate, h0 = inputs(1, (1, c), dtype, True, 3, c)
    d_h, d_last = rnd(8, 1, c, dtype=dtype), rnd(9, 3, c)
    kw = dict(starts=torch.tensor([0, 0, 1, 1], dtype=torch.int32, device="cuda"), max_len=most)
    h, last, states, *grads = check(x, gate, gi, rate, h0, d_h, d_last, [lambda t: t[:0], lambda t: t, lambda t: t[:0]], kw)

    def turned(t):
        return t.clone().as_strided((1, c), (1, 1))       # a column's, seen as a row

    def alone(t):
        return t.clone().as_strided((1, c), (0, 1))

    for way in (turned, alone):
        assert way(x).stride(0) < 2
        got = recurrence_fwd(way(x), way(gate), rate, way(gi), h0=h0, out=way(torch.zeros_like(x)), want_states=True, **kw)
        mine = recurrence_bwd(way(x), way(gate), rate, states, way(d_h), way(gi), d_last=d_last, **kw,
                              **{name: way(torch.zeros_like(x)) for name in ("dx", "dgate", "dinput_gate")})
        torch.cuda.synchronize()
        assert torch.equal(got[0], h) and torch.equal(got[1], last)
        for a, b in zip(grads, mine):
            assert torch.equal(a, b)


@pytest.mark.parametrize("n", [1, 5, 300])
def test_in_place_over_strides_that_say_nothing(n):
    """An output over an input of one sequence, or one token, whose views differ in the stride of what there is one of."""
    from r9700training_amd.recurrence import recurrence_fwd

    c = 64
    x, gate, gi, rate, h0 = inputs(1, (1, n, c), BF, True, 1, c)
    h, last, _ = recurrence_fwd(x, gate, rate, gi, h0=h0)
    over = x.clone()
    got = recurrence_fwd(over, gate, rate, gi, h0=h0, out=over.as_strided((1, n, c), (7 * c, c if n > 1 else 5 * c, 1)))
    assert torch.equal(got[0], h) and torch.equal(over, h) and torch.equal(got[1], last)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n", [1, 40, 300, 1500])
@pytest.mark.parametrize("c", [64, 3])
def test_a_rate_without_bound(dtype, n, c):
    """Infinite and nearly infinite rates: nothing is left of a state after a token, and the places past a sequence's last
    token decay as little as under any rate. The only sums left are products: a gate's sigmoid, off by (|g| + 8) U, with x or
    the cotangent, and their roundings."""
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    x, gate, gi, _, h0 = inputs(1, (2, n, c), dtype, True, 2, c)
    d_h, d_last = rnd(8, 2, n, c, dtype=dtype), rnd(9, 2, c)
    for value in (math.inf, 3e38, 1e36, 1e30):
        rate = torch.full((c,), value, device="cuda")
        h, last, states = recurrence_fwd(x, gate, rate, gi, h0=h0, want_states=True)
        grads = recurrence_bwd(x, gate, rate, states, d_h, gi, d_last=d_last)
        torch.cuda.synchronize()
        si = torch.sigmoid(gi.double())
        ei = (gi.double().abs() + 8) * R.U
        off = ei + 6 * R.U
        want, lam = si * x.double(), d_h.double()
        lam[:, -1] += d_last.double()
        e_lam = 4 * R.U * (d_h.double().abs() + lam.abs())
        close(h, want, want.abs() * off, HALF[dtype], f"h, rate {value}")
        close(last, want[:, -1], (want.abs() * off)[:, -1], HALF[F32], f"last, rate {value}")
        dx = lam * si
        e_dx = dx.abs() * off + e_lam * si
        di = dx * x.double() * (1 - si)
        e_di = e_dx * x.double().abs() * (1 - si) + (dx * x.double()).abs() * (si * ei + 4 * R.U) + di.abs() * 4 * R.U
        close(grads[0], dx, e_dx, HALF[dtype], f"dx, rate {value}")
        close(grads[2], di, e_di, HALF[dtype], f"dinput_gate, rate {value}")
        assert (grads[1] == 0).all() and (grads[4] == 0).all(), value
        # up to 127 places past a sequence's end, each shut by a gate that f32 counts as -87: e^-87 < 2e-38 times the cotangent
        # behind them and the state before them (products and sums under twice that again)
        leak = 127 * 4e-38 * (d_last.double() * last.double()).abs().sum(0)
        assert (grads[3].double().abs() <= leak).all(), value


def scan(a, b):
    """v[t] = a[t] v[t - 1] + b[t] from nothing, f64 [tokens, channels]: spans joined by doubling."""
    a, b, s = a.clone(), b.clone(), 1
    while s < len(a):
        b[s:] += a[s:] * b[:-s].clone()
        a[s:] *= a[:-s].clone()
        s *= 2
    return b


def carried(gate, rate, e, root=True, roundings=2):
    """The state before nothing, carried through v[t] = a[t] v[t - 1] + u[t] (u: sqrt(1 - a^2) e, or a e), how far wrong logarithms
    and inputs may put it, and the standard deviation of what the roundings add: `roundings` a token, each up to U of a state and
    of either sign, so U / sqrt(3) of it. A bound of them all would grow with the tokens; an error with a sign does as well."""
    _, la, a, q, _ = R.parts(e, gate, rate, None)
    eg = (gate.abs() + 8) * R.U
    u = torch.sqrt(q) * e if root else a * e
    size = scan(a, u.abs())
    before = torch.cat([torch.zeros_like(size[:1]), size[:-1]])
    wrong = scan(a, a * before * la.abs() * (eg + 4 * R.U) + u.abs() * ((eg + 12 * R.U) / 2 + 6 * R.U + la.abs() * eg))
    var = scan(a * a, size ** 2 * roundings * R.U ** 2 / 3)
    return scan(a, u), wrong, torch.sqrt(var)


def without_a_sign(got, want, wrong, std, what):
    """Each channel's within six standard deviations, and the channels' mean, whose gates are independent, within its own."""
    off = got.double() - want
    n = want.shape[-1]
    print(f"{what}: mean error {float((off / want).mean() / R.U):.1f} U, largest {float((off / want).abs().max() / R.U):.1f} U, "
          f"mean tolerance {float(((wrong + 6 * std / n ** 0.5) / want.abs()).mean() / R.U):.1f} U", flush=True)
    assert bool((off.abs() <= wrong + 6 * std + 2 * R.U * want.abs()).all()), what
    mean, tol = (off / want).mean(-1).abs(), (wrong / want.abs()).mean(-1) + 6 * (std / want.abs()).pow(2).sum(-1).sqrt() / n + 2 * R.U
    assert bool((mean <= tol).all()), f"{what}: {mean / R.U} against {tol / R.U} U"


def slow(n, c, dtype, rate):
    """Inputs of one sign and decays next to one."""
    x, d_h = ((1 + rnd(50 + i, 1, n, c, std=0.25)).to(dtype) for i in range(2))
    g = torch.Generator(device="cuda").manual_seed(53)
    return x, rnd(52, 1, n, c, dtype=dtype), d_h, rate * (0.5 + torch.rand(c, generator=g, device="cuda"))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rate", [1e-4, 1e-3, 1e-2])
def test_thousands_of_single_tokens(dtype, rate):
    """A state, and backward a cotangent, carried through thousands of calls of one token: no error with a sign adds up."""
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    n, c = 4000, 256
    x, gate, d_h, rates_ = slow(n, c, dtype, rate)
    state, m = torch.zeros((1, c), device="cuda"), torch.zeros((1, c), device="cuda")
    for t in range(n):
        recurrence_fwd(x[:, t:t + 1], gate[:, t:t + 1], rates_, h0=state, last=state)
    out = [torch.empty_like(x[:, :1]) for _ in range(2)] + [torch.empty(c, device="cuda"), torch.empty((1, c), device="cuda")]
    for t in reversed(range(n)):
        recurrence_bwd(x[:, t:t + 1], gate[:, t:t + 1], rates_, state[None], d_h[:, t:t + 1], d_last=m, dx=out[0], dgate=out[1],
                       drate=out[2], dh0=out[3])
        m, out[3] = out[3], m
    torch.cuda.synchronize()
    g64, r64 = gate[0].double(), rates_.double()
    without_a_sign(state[0], *(t[-1] for t in carried(g64, r64, x[0].double())), "the state")
    back = carried(g64.flip(0), r64, d_h[0].double().flip(0), root=False, roundings=3)
    without_a_sign(m[0], *(t[-1] for t in back), "the cotangent")


@pytest.mark.parametrize("rate", [1e-4, 1e-3])
def test_long_runs_of_a_range(rate):
    """A quarter of a million tokens in ranges, whose spans walk runs of thousands of tokens: the states and cotangents that the
    ranges begin from have no error with a sign."""
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd

    n, c = 1 << 18, 4096
    x, gate, d_h, rates_ = slow(n, c, F32, rate)
    _, _, states = recurrence_fwd(x, gate, rates_, want_states=True)
    dx = recurrence_bwd(x, gate, rates_, states, d_h)[0][0, :, ::64]
    torch.cuda.synchronize()
    x, gate, d_h, r64 = (t[..., ::64].double() for t in (x[0], gate[0], d_h[0], rates_))
    want = carried(gate, r64, x)
    for t in range(n // 16, n, n // 16):
        without_a_sign(states[0, t // CHUNK, ::64], *(v[t - 1] for v in want), f"the state before token {t}")
    # dx = l sqrt(q), of which sqrt(q) is off by its gate's sigmoid; l before its decay: l[t] = m[t] / a[t]
    m, wrong, std = (v.flip(0) for v in carried(gate.flip(0), r64, d_h.flip(0), root=False, roundings=3))
    _, _, a, q, _ = R.parts(x, gate, r64, None)
    for t in range(n // 16 - 1, n, n // 16):
        by = torch.sqrt(q[t]) / a[t]
        value = m[t] * by
        root = value.abs() * (((gate[t].abs() + 8) * R.U + 12 * R.U) / 2 + 8 * R.U)
        without_a_sign(dx[t], value, wrong[t] * by + root, std[t] * by, f"dx of token {t}")
