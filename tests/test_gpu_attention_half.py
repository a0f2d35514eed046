"""The attention half of a layer (examples/attention_half.py): every stage's output against float64 from the stage's own
inputs, so that a wrong operand, layout or scale anywhere on the way shows, and the layer a token at a time against the
whole sequence."""
import importlib.util
import math
import os

import pytest
import torch

import between_ref as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("attention_half", os.path.join(ROOT, "examples", "attention_half.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def rel(got, want):
    return float((got.double() - want).norm() / want.norm())


def weight(pair):
    codes, scale = pair
    return codes.double() * scale.view(BF).double().repeat_interleave(128, 1)


# one rounding to bf16, at most half a step of each value, and f32 sums far below it
ONE = 2 ** -8 * 1.01
# a product of operands rounded once before it (probabilities, dS, the adapter's t or the coded path's operand), then
# its own rounding: at most three half steps in norm
SUM = 3 * 2 ** -8


@pytest.mark.parametrize("lens", [[130, 1, 64, 300], [257]])
def test_stages(lens):
    m = example()
    layer = m.AttentionHalf(512, 8, 2, 64, seed=3)
    g = torch.Generator(device="cuda").manual_seed(1)
    n = sum(lens)
    x, r, dz, dh = (torch.randn((n, 512), generator=g, device="cuda").to(BF) for _ in range(4))
    starts = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    z, h, s = layer.forward(x, r, starts, max(lens))
    back = layer.backward(s, dz, dh)
    torch.cuda.synchronize()

    wh, wrs, wy = R.norm(x, r, layer.gain, 1e-6, 0.0, BF)
    assert torch.equal(h.double(), wh) and float(((s["rstd"].double() - wrs) / wrs).abs().max()) < 1e-4
    # the codes stand for wy: half a step of their scale
    again = m.add_rmsnorm_i8g(x, r, layer.gain, 128)
    codes, scale = again[0], again[1]
    assert torch.equal(scale, s["scale"])
    assert bool(((codes.double() * scale.double().repeat_interleave(128, 1) - wy).abs()
                 <= 0.5001 * scale.double().repeat_interleave(128, 1)).all())
    W, Wo = weight(layer.qkv), weight(layer.out)
    y = (codes.double() * scale.double().repeat_interleave(128, 1)) @ W.t()
    pos = torch.cat([torch.arange(k, device="cuda") for k in lens]).double()
    angles = pos[:, None] * layer.inv_freq
    yq, yk, yv = layer.split(y)
    q, k, v = layer.split(s["y"])
    # the projection's rounding, then the rotation's
    assert rel(q, R.rotary(yq.to(BF).double(), angles, 64, "half", layer.mscale, False)) <= 2 * ONE
    assert rel(k, R.rotary(yk.to(BF).double(), angles, 64, "half", layer.mscale, False)) <= 2 * ONE
    assert rel(v, yv) <= ONE
    seqs, at = [], 0
    for c in lens:
        seqs.append(tuple(t[at:at + c].double() for t in (q, k, v)) + (back["do"].view(n, 8, 64)[at:at + c].double(),))
        at += c
    ref = R.reference(seqs, 8, 2, True, 0, 1.0 / math.sqrt(64), 2 ** -8, 2 ** -8)
    assert rel(s["o"], torch.cat([t["out"][0] for t in ref])) <= SUM
    o = s["o"].flatten(1).double()
    assert rel(z, o @ Wo.t() + (o @ layer.A.double().t()) @ layer.B.double().t()) <= SUM

    assert rel(back["do"], dz.double() @ Wo + (dz.double() @ layer.B.double()) @ layer.A.double()) <= SUM
    dq, dk, dv = layer.split(back["dy"])
    # attention's gradient, turned back
    turn = lambda t: R.rotary(t, angles, 64, "half", layer.mscale, True)  # noqa: E731
    assert rel(dq, turn(torch.cat([t["dq"][0] for t in ref]))) <= 2 * SUM
    assert rel(dk, turn(torch.cat([t["dk"][0] for t in ref]))) <= 2 * SUM
    assert rel(dv, torch.cat([t["dv"][0] for t in ref])) <= 2 * SUM
    assert rel(back["g_codes"], (back["dy"].double() @ W) * scale.double().repeat_interleave(128, 1)) <= SUM
    wdx, wdw, _ = R.norm_backward(h.double(), s["rstd"].double(), layer.gain, 0.0, scale, 128, back["g_codes"], None, dh)
    assert rel(back["dx"], wdx) <= ONE and rel(back["dgain"], wdw) <= 1e-4
    assert rel(back["dB"], dz.double().t() @ (o @ layer.A.double().t())) <= 1e-3
    assert rel(back["dA"], (dz.double() @ layer.B.double()).t() @ o) <= 1e-3


def test_token_by_token():
    """Every token through the cache gives the whole sequence's output: the same codes and rotation (the same kernels on one
    row), keys and values rounded alike; attention and the projection sum in another order and round twice."""
    m = example()
    layer = m.AttentionHalf(512, 8, 2, 64, seed=4)
    g = torch.Generator(device="cuda").manual_seed(2)
    x, r = (torch.randn((2 * 40, 512), generator=g, device="cuda").to(BF) for _ in range(2))
    starts = torch.tensor([0, 40, 80], dtype=torch.int32, device="cuda")
    z, h, _ = layer.forward(x, r, starts, 40)
    cache = layer.cache(2, 48)
    for i in range(40):
        zi, hi = layer.token(x[[i, 40 + i]], r[[i, 40 + i]], cache)
        assert torch.equal(hi, h[[i, 40 + i]])
        assert rel(zi, z[[i, 40 + i]].double()) <= 2 * SUM, i
    assert cache["lens"].tolist() == [40, 40]
