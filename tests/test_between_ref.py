"""The float64 references of the operators between the projections against central differences (CPU)."""
import math

import pytest
import torch

import between_ref as R


def rnd(seed, *shape):
    return torch.randn(shape, dtype=torch.float64, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("lq,lk,causal,window", [(5, 7, True, 0), (6, 3, True, 0), (4, 9, False, 0), (7, 7, True, 2), (3, 0, False, 0)])
def test_attention_gradients_are_the_differences(lq, lk, causal, window):
    q, k, v, do = rnd(1, lq, 4, 6), rnd(2, lk, 2, 6), rnd(3, lk, 2, 6), rnd(4, lq, 4, 6)

    def loss(q, k, v):
        return float((R.reference([(q, k, v, None)], 4, 2, causal, window, 0.4, 0.0)[0]["out"][0] * do).sum())

    got = R.reference([(q, k, v, do)], 4, 2, causal, window, 0.4, 0.0, 0.0)[0]
    for n, x in (("dq", q), ("dk", k), ("dv", v)):
        for at in range(0, x.numel(), 5):
            step = torch.zeros(x.numel(), dtype=torch.float64)
            step[at] = 1e-5
            step = step.view(x.shape)
            args = [(q, k, v), (q, k, v)]
            i = "qkv".index(n[1])
            hi, lo = list(args[0]), list(args[1])
            hi[i], lo[i] = x + step, x - step
            # central differences: an error of step^2 and 1e-16 / step
            assert abs((loss(*hi) - loss(*lo)) / 2e-5 - float(got[n][0].flatten()[at])) < 1e-7, (n, at)


def test_rotary_inverse_is_the_adjoint():
    x, y, a = rnd(1, 5, 3, 16), rnd(2, 5, 3, 16), rnd(3, 5, 5)
    for pairs in ("half", "interleaved"):
        lhs = (R.rotary(x, a, 10, pairs, 1.3, False) * y).sum()
        rhs = (x * R.rotary(y, a, 10, pairs, 1.3, True)).sum()
        assert abs(float(lhs - rhs)) < 1e-12
        back = R.rotary(R.rotary(x, a, 10, pairs, 1.0, False), a, 10, pairs, 1.0, True)
        assert float((back - x).abs().max()) < 1e-14


def test_norm_gradient_is_the_differences():
    h, w, gc, gy, gh = rnd(1, 3, 10), rnd(2, 10), rnd(3, 3, 10), rnd(4, 3, 10), rnd(5, 3, 10)
    eps, wadd, group = 1e-3, 0.5, 4
    rs = 1.0 / torch.sqrt((h * h).mean(1) + eps)
    scale = R.group_scale(h * rs[:, None] * (w + wadd), group)

    def loss(h, w):
        _, _, y = R.norm(h, None, w, eps, wadd, torch.float64)
        return float((y * (gc / scale[:, R.group_index(10, group, h.device)] + gy) + h * gh).sum())

    dx, dw, _ = R.norm_backward(h, rs, w, wadd, scale, group, gc, gy, gh)
    for x, d, f in ((h, dx, lambda t: loss(t, w)), (w, dw, lambda t: loss(h, t))):
        for at in range(x.numel()):
            step = torch.zeros(x.numel(), dtype=torch.float64)
            step[at] = 1e-5
            step = step.view(x.shape)
            got = (f(x + step) - f(x - step)) / 2e-5
            assert abs(got - float(d.flatten()[at])) < 1e-7 * max(1.0, float(gc.abs().max() / scale.min())), at


def test_frequencies_on_the_host():
    from r9700training_amd.rotary import rotary_frequencies

    f, m = rotary_frequencies(64, 1e6, device="cpu")
    want = 1e6 ** (-torch.arange(32, dtype=torch.float64) / 32)
    assert m == 1.0 and float(((f - want) / want).abs().max()) < 1e-14
    g, m = rotary_frequencies(64, 1e6, "linear", factor=4.0, device="cpu")
    assert m == 1.0 and torch.equal(g, f / 4.0)
    g, m = rotary_frequencies(64, 1e6, "ramp", factor=8.0, original=4096.0, slow=1.0, fast=32.0, device="cpu")
    turns = 4096.0 * want / (2 * math.pi)
    assert abs(m - (0.1 * math.log(8.0) + 1.0)) < 1e-6
    assert torch.equal(g[turns > 32], f[turns > 32]) and int((turns > 32).sum()) > 0
    slow = turns < 1
    assert int(slow.sum()) > 0 and float((g[slow] / (f[slow] / 8) - 1).abs().max()) < 1e-14
    mid = ~slow & (turns <= 32)
    assert int(mid.sum()) > 0 and bool((g[mid] < f[mid]).all()) and bool((g[mid] > f[mid] / 8).all())
