"""Rotary positions against float64: both pairings, partial and whole heads, far positions, both types,
layouts and widths off the 16-byte pieces. Tolerances: the f32 sine and cosine (the angle's fraction of a turn rounded
to f32, their own error of 4 ulp), two products and a sum in f32, and the output's rounding."""
import pytest
import torch

import between_ref as R

pytestmark = pytest.mark.gpu


def rnd(seed, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def check(x, got, angles, rot, pairs, mscale, inverse, what):
    want = R.rotary(x.double(), angles, rot, pairs, mscale, inverse)
    half = R.HALF[x.dtype]
    # a turn's fraction to 2^-25 of a turn is 2 pi 2^-25 of an angle; sine, cosine, mscale, product, sum
    trig = (2 * 3.1416 / 2 + 4 + 4) * 2 * R.U32
    pair = torch.zeros_like(want)
    i, j = (slice(0, rot // 2), slice(rot // 2, rot)) if pairs == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    size = (x.double()[..., i].abs() + x.double()[..., j].abs()) * abs(mscale)
    pair[..., i], pair[..., j] = size, size
    off = (got.double() - want).abs() - (half * want.abs() + trig * pair)
    assert float(off.max()) <= 0.0, f"{what}: {float(off.max())} past the tolerance"
    assert torch.equal(got[..., rot:], x[..., rot:]), f"{what}: what does not turn is copied"


CASES = [
    # tokens, q_heads, kv_heads, dim, rot, pairs, dtype
    (1, 24, 4, 256, 64, "half", torch.bfloat16),
    (1, 1, 1, 2, 2, "interleaved", torch.float32),
    (7, 3, 1, 64, 64, "half", torch.float32),
    (300, 8, 2, 128, 128, "interleaved", torch.bfloat16),
    (1001, 8, 2, 128, 64, "half", torch.bfloat16),
    (65, 2, 2, 80, 20, "half", torch.bfloat16),
    (65, 2, 2, 80, 20, "interleaved", torch.bfloat16),
    (33, 5, 1, 96, 96, "half", torch.bfloat16),
    (33, 5, 1, 9, 6, "half", torch.float32),
    (12, 2, 1, 1024, 1024, "interleaved", torch.float32),
    (3000, 16, 16, 64, 32, "interleaved", torch.float32),
    (3, 2, 1, 8192, 8192, "half", torch.bfloat16),
]


@pytest.mark.parametrize("tokens,hq,hk,dim,rot,pairs,dtype", CASES)
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary(tokens, hq, hk, dim, rot, pairs, dtype, inverse):
    from r9700training_amd.rotary import rotary, rotary_frequencies

    print(f"case rotary {(tokens, hq, hk, dim, rot, pairs, dtype, inverse)}", flush=True)
    q, k = rnd(1, tokens, hq, dim, dtype=dtype), rnd(2, tokens, hk, dim, dtype=dtype)
    f, m = rotary_frequencies(rot, 1e4, "ramp", factor=8.0, original=2048.0)
    for start, width in ((0, torch.int32), (3_000_000, torch.int32), (-50, torch.int64), (2 ** 33, torch.int64)):
        pos = torch.arange(start, start + tokens, device="cuda").to(width)
        angles = pos.double()[:, None] * f
        qo, ko = rotary(q, k, f, pos, pairs=pairs, mscale=m, inverse=inverse)
        # f64's own error on the angle: position * frequency to 2^-53, in radians
        check(q, qo, angles, rot, pairs, m, inverse, f"q from {start}")
        check(k, ko, angles, rot, pairs, m, inverse, f"k from {start}")
    qo, ko = rotary(q, None, f, None, pairs=pairs, inverse=inverse)
    check(q, qo, torch.arange(tokens, device="cuda").double()[:, None] * f, rot, pairs, 1.0, inverse, "q alone, no positions")
    assert ko is None


@pytest.mark.parametrize("dim,rot", [(64, 32), (72, 24)])
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts_and_in_place(dim, rot, pairs, dtype):
    """Slices of a fused projection, head-major tensors, odd offsets (the narrow kernel) and the inputs themselves as
    outputs give the contiguous call's bits."""
    from r9700training_amd.rotary import rotary, rotary_frequencies

    t, hq, hk = 77, 4, 2
    f, _ = rotary_frequencies(rot)
    fused = rnd(1, t, (hq + hk) * dim + 3, dtype=dtype)
    for off in (0, 1, 3):
        q = fused[:, off:off + hq * dim].unflatten(1, (hq, dim))
        k = fused[:, off + hq * dim:off + (hq + hk) * dim].unflatten(1, (hk, dim))
        want = rotary(q.contiguous(), k.contiguous(), f, pairs=pairs)
        got = rotary(q, k, f, pairs=pairs)
        tall = [torch.empty((n, t, dim), dtype=dtype, device="cuda").transpose(0, 1) for n in (hq, hk)]
        rotary(q, k, f, pairs=pairs, q_out=tall[0], k_out=tall[1])
        mine = fused.clone()
        mq = mine[:, off:off + hq * dim].unflatten(1, (hq, dim))
        mk = mine[:, off + hq * dim:off + (hq + hk) * dim].unflatten(1, (hk, dim))
        rotary(mq, mk, f, pairs=pairs, q_out=mq, k_out=mk)
        for a, b, c, d in zip(want, got, tall, (mq, mk)):
            assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)
        keep = torch.ones(fused.shape[1], dtype=torch.bool)
        keep[off:off + (hq + hk) * dim] = False
        assert torch.equal(mine[:, keep.cuda()], fused[:, keep.cuda()])


def test_broadcast_input_stream_and_graph():
    from r9700training_amd.rotary import rotary, rotary_frequencies

    f, _ = rotary_frequencies(64)
    one = rnd(1, 1, 1, 64)
    x = one.expand(50, 4, 64)
    want = rotary(x.contiguous(), None, f)[0]
    assert torch.equal(rotary(x, None, f)[0], want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = rotary(x, None, f, stream=side)[0]
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    q, pos = rnd(2, 50, 4, 64), torch.arange(50, dtype=torch.int32, device="cuda")
    rotary(q, None, f, pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rotary(q, None, f, pos)[0]
    for i in range(3):
        q.copy_(rnd(3 + i, 50, 4, 64))
        pos.add_(1000)
        want = rotary(q, None, f, pos)[0]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


def test_no_tokens():
    from r9700training_amd.rotary import rotary, rotary_frequencies

    f, _ = rotary_frequencies(64)
    q, k = rotary(rnd(1, 0, 4, 64), rnd(2, 0, 2, 64), f)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)


@pytest.mark.parametrize("dim,rot", [(96, 24), (90, 12), (20, 4), (66, 22), (96, 40)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pieces_of_every_width(dim, rot, dtype):
    """Halves and rests of 2, 4, 6, 10, 11, 12 and 20 values, and heads that begin off 16, 8 and 4 bytes."""
    from r9700training_amd.rotary import rotary, rotary_frequencies

    f, m = rotary_frequencies(rot, 1e4, "ramp", factor=8.0, original=2048.0)
    t, hq = 50, 3
    angles = torch.arange(t, device="cuda").double()[:, None] * f
    for gap in (0, 1, 2, 4):
        wide = rnd(1, t, hq, dim + gap, dtype=dtype)
        x = wide[..., gap:]
        for pairs in ("half", "interleaved"):
            got = rotary(x, None, f, None, pairs=pairs, mscale=m)[0]
            check(x, got, angles, rot, pairs, m, False, f"gap {gap} {pairs}")


def test_more_tokens_than_a_launch_takes_across():
    """Tokens past the first dimension's workgroups: single values of odd places, a token a workgroup, in place."""
    from r9700training_amd.rotary import rotary, rotary_frequencies

    tokens, dim = 16_777_300, 2052  # 1026 pairs of single values a token
    f, _ = rotary_frequencies(dim)
    whole = torch.empty(tokens * dim + 1, dtype=torch.bfloat16, device="cuda")  # 69 GB
    x = whole[1:].view(tokens, 1, dim)
    ends = [slice(a, a + 40) for a in (0, 8_388_600, 16_777_200, tokens - 40)]
    kept = []
    for i, part in enumerate(ends):
        x[part] = rnd(i, 40, 1, dim)
        kept.append(x[part].clone())
    rotary(x, None, f, q_out=x)
    for part, was in zip(ends, kept):
        pos = torch.arange(part.start, part.stop, dtype=torch.int32, device="cuda")
        assert torch.equal(x[part], rotary(was, None, f, pos)[0]), part
