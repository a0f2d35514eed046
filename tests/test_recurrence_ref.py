"""The recurrence's reference gradients against differences of its forward (no GPU needed)."""
import pytest
import torch

import recurrence_ref as R


@pytest.mark.parametrize("gated", [True, False])
def test_gradients_are_the_forwards(gated):
    g = torch.Generator().manual_seed(1)
    n, c = 7, 5
    rnd = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    x, gate, gi, h0 = rnd(n, c), rnd(n, c), rnd(n, c), rnd(c)
    rate = torch.tensor([0.01, 0.3, 1.0, 4.0, 9.0], dtype=torch.float64)
    dh, dl = rnd(n, c), rnd(c)
    gi = gi if gated else None

    def loss(**kw):
        v = dict(x=x, gate=gate, rate=rate, input_gate=gi, h0=h0)
        v.update(kw)
        r = R.forward(**v)
        return float((r["h"][0] * dh).sum() + (r["last"][0] * dl).sum())

    grads = R.backward(x, gate, rate, gi, h0, dh, dl)
    for name, value in (("x", x), ("gate", gate), ("rate", rate), ("input_gate", gi), ("h0", h0)):
        if value is None:
            continue
        got = grads["d" + name][0].reshape(-1)
        for i in range(value.numel()):
            step = torch.zeros(value.numel(), dtype=torch.float64)
            step[i] = 1e-5 * max(1e-3, abs(float(value.reshape(-1)[i])))
            step = step.reshape(value.shape)
            diff = (loss(**{name: value + step}) - loss(**{name: value - step})) / (2 * float(step.sum()))
            assert abs(diff - float(got[i])) <= 1e-6 * (1 + abs(diff)), (name, i, diff, float(got[i]))


def test_tokens_are_the_definition():
    x, gate = torch.tensor([[2.0], [-1.0]], dtype=torch.float64), torch.tensor([[0.0], [1.0]], dtype=torch.float64)
    rate, h0 = torch.tensor([0.5], dtype=torch.float64), torch.tensor([3.0], dtype=torch.float64)
    r = R.forward(x, gate, rate, None, h0)
    a0 = torch.exp(torch.tensor(-0.25, dtype=torch.float64))
    h1 = a0 * 3 + torch.sqrt(1 - a0 ** 2) * 2
    assert abs(float(r["h"][0][0, 0] - h1)) < 1e-14 and float(r["before"][0][1, 0]) == float(r["h"][0][0, 0])
