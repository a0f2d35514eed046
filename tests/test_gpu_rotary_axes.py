"""Rotary positions with several axes against float64, with tests/test_gpu_rotary.py's tolerances."""
import pytest
import torch

from test_gpu_rotary import check, rnd

pytestmark = pytest.mark.gpu

CASES = [
    # tokens, q_heads, kv_heads, dim, sections, order, pairs, dtype
    (1, 24, 4, 256, [11, 11, 10], "cycle", "half", torch.bfloat16),
    (1, 1, 1, 4, [1, 1], "blocks", "interleaved", torch.float32),
    (7, 3, 1, 64, [16, 8, 8], "blocks", "half", torch.float32),
    (300, 8, 2, 128, [16, 24, 24], "blocks", "interleaved", torch.bfloat16),
    (1001, 8, 2, 128, [0, 32], "cycle", "half", torch.bfloat16),
    (65, 2, 2, 80, [3, 4, 3], "cycle", "half", torch.bfloat16),
    (33, 5, 1, 9, [1, 0, 1, 1], "blocks", "half", torch.float32),
    (500, 16, 16, 64, [32], "blocks", "interleaved", torch.float32),
]


def positions(axes, tokens, start, dtype):
    t = torch.arange(tokens, device="cuda")
    return torch.stack([start + (t // (a + 1)) * (1 if a % 2 == 0 else -1) for a in range(axes)]).to(dtype)


@pytest.mark.parametrize("tokens,hq,hk,dim,sections,order,pairs,dtype", CASES)
@pytest.mark.parametrize("inverse", [False, True])
def test_axes(tokens, hq, hk, dim, sections, order, pairs, dtype, inverse):
    from r9700training_amd.rotary import rotary_axes, rotary_frequencies, rotary_pair_axes

    print(f"case axes {(tokens, hq, hk, dim, sections, order, pairs, dtype, inverse)}", flush=True)
    rot = 2 * sum(sections)
    q, k = rnd(1, tokens, hq, dim, dtype=dtype), rnd(2, tokens, hk, dim, dtype=dtype)
    f, m = rotary_frequencies(rot, 1e4, "ramp", factor=8.0, original=2048.0)
    axis = rotary_pair_axes(sections, order)
    for start, width in ((0, torch.int32), (3_000_000, torch.int32), (-50, torch.int64), (2 ** 33, torch.int64)):
        pos = positions(len(sections), tokens, start, width)
        angles = pos.double()[axis.long()].T * f
        qo, ko = rotary_axes(q, k, f, pos, axis, pairs=pairs, mscale=m, inverse=inverse)
        check(q, qo, angles, rot, pairs, m, inverse, f"q from {start}")
        check(k, ko, angles, rot, pairs, m, inverse, f"k from {start}")
        # rows of a wider table of positions
        wide = torch.full((len(sections), tokens + 5), 77, dtype=width, device="cuda")
        wide[:, 2:2 + tokens] = pos
        again, none = rotary_axes(q, None, f, wide[:, 2:2 + tokens], axis, pairs=pairs, mscale=m, inverse=inverse)
        assert torch.equal(again, qo) and none is None


def test_one_axis_is_rotary():
    """The same position on every axis, and all pairs on one of several axes, are rotary's bits."""
    from r9700training_amd.rotary import rotary, rotary_axes, rotary_frequencies, rotary_pair_axes

    q, k = rnd(1, 200, 8, 128), rnd(2, 200, 2, 128)
    f, _ = rotary_frequencies(64)
    pos = torch.arange(1000, 1200, dtype=torch.int32, device="cuda")
    want = rotary(q, k, f, pos)
    axis = rotary_pair_axes([12, 10, 10], "cycle")
    for p, a in ((pos.expand(3, 200), axis), (torch.stack([pos + 5, pos, pos - 5]), torch.ones_like(axis))):
        got = rotary_axes(q, k, f, p, a)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_pairs_of_no_axis_are_only_scaled():
    from r9700training_amd.rotary import rotary_axes, rotary_frequencies

    q = rnd(1, 50, 4, 64, dtype=torch.float32)
    f, _ = rotary_frequencies(64)
    pos = torch.arange(100, dtype=torch.int32, device="cuda").view(2, 50)
    axis = torch.tensor([0, 1, -1, 2, 2 ** 31 - 1, -(2 ** 31), 1, 0] * 4, dtype=torch.int32, device="cuda")
    got = rotary_axes(q, None, f, pos, axis, mscale=0.5)[0]
    for i in range(32):
        if int(axis[i]) not in (0, 1):
            assert torch.equal(got[..., i], 0.5 * q[..., i]) and torch.equal(got[..., 32 + i], 0.5 * q[..., 32 + i])
    angles = torch.where((axis >= 0) & (axis < 2), pos.double()[axis.clamp(0, 1).long()].T * f, 0.0)
    check(q, got, angles, 64, "half", 0.5, False, "q")


def test_in_place_stream_graph_and_no_tokens():
    from r9700training_amd.rotary import rotary_axes, rotary_frequencies, rotary_pair_axes

    f, _ = rotary_frequencies(64)
    axis = rotary_pair_axes([12, 10, 10])
    q, k, pos = rnd(1, 60, 4, 64), rnd(2, 60, 2, 64), positions(3, 60, 9, torch.int32)
    want = rotary_axes(q, k, f, pos, axis)
    mine = q.clone(), k.clone()
    rotary_axes(*mine, f, pos, axis, q_out=mine[0], k_out=mine[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = rotary_axes(q, k, f, pos, axis, stream=side)
    torch.cuda.synchronize()
    for a, b, c in zip(want, mine, got):
        assert torch.equal(a, b) and torch.equal(a, c)
    # forward and back
    back = rotary_axes(*want, f, pos, axis, inverse=True)
    assert float((back[0].float() - q.float()).abs().max()) <= 2 ** -6 * float(q.float().abs().max())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rotary_axes(q, k, f, pos, axis)
    for i in range(3):
        q.copy_(rnd(3 + i, 60, 4, 64))
        pos.add_(1000)
        want = rotary_axes(q, k, f, pos, axis)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])
    none = rotary_axes(q[:0], k[:0], f, pos[:, :0], axis)
    assert none[0].shape == (0, 4, 64) and none[1].shape == (0, 2, 64)
