"""The operators between the projections in float64, from their definitions, and how far a correct f32 /
bf16 implementation may lie from them (every rounding counted at half a step)."""
from __future__ import annotations

import math

import torch

HALF = {torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2, torch.float32: torch.finfo(torch.float32).eps / 2}
U32 = HALF[torch.float32]


def visible(lq, lk, causal, window, device):
    """True where query i (the last query stands at the last key) sees key j."""
    at = torch.arange(lq, device=device)[:, None] + (lk - lq)
    j = torch.arange(lk, device=device)[None, :]
    see = torch.ones((lq, lk), dtype=torch.bool, device=device)
    if causal:
        see &= j <= at
    if window:
        see &= j > at - window
    return see


def head_forward(q, k, v, see, scale):
    """(out, lse, P) of one head, f64; a query that sees nothing: zeros, -inf."""
    s = (q @ k.t()) * scale
    s = torch.where(see, s, torch.full_like(s, -math.inf))
    top = s.amax(1, keepdim=True) if s.shape[1] else s.new_full((s.shape[0], 1), -math.inf)
    p = torch.where(see, torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top)), torch.zeros_like(s))
    total = p.sum(1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    lse = torch.where(total > 0, torch.where(torch.isinf(top), torch.zeros_like(top), top) + torch.log(total),
                      torch.full_like(total, -math.inf))
    return p @ v, lse[:, 0], p


def head_backward(q, k, v, p, do, scale):
    """(dq, dk, dv, dS) of one head, f64."""
    dp = do @ v.t()
    ds = p * (dp - (p * dp).sum(1, keepdim=True))
    return scale * (ds @ k), scale * (ds.t() @ q), p.t() @ do, ds


def score_error(q, k, scale):
    """How far f32 scores can be off: head_dim roundings of sums of |q||k|, and the exponential's own."""
    most = (q.abs() @ k.abs().t()).max() * abs(scale) if k.shape[0] and q.shape[0] else torch.zeros((), dtype=q.dtype)
    return float(2 * q.shape[1] * U32 * most + 2 ** -20)


def reference(seqs, q_heads, kv_heads, causal, window, scale, out_half, grad_half=None):
    """seqs: [(q, k, v, do or None)] with q [n, Hq, d], k, v [m, Hk, d], f64. Returns, a sequence, a dict of name ->
    (value, tolerance), token-major: out, lse [Hq, n] and with do dq, dk, dv. out_half, grad_half: half a
    step of the outputs' types."""
    share = q_heads // kv_heads
    bf = HALF[torch.bfloat16]
    res = []
    for q, k, v, do in seqs:
        see = visible(q.shape[0], k.shape[0], causal, window, q.device)
        r = {n: (torch.zeros_like(x), torch.zeros_like(x)) for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", k))}
        lse = torch.zeros((q_heads, q.shape[0]), dtype=q.dtype, device=q.device)
        r["lse"] = (lse, torch.zeros_like(lse))
        for h in range(q_heads):
            qh, kh, vh = q[:, h], k[:, h // share], v[:, h // share]
            o, l, p = head_forward(qh, kh, vh, see, scale)
            e = score_error(qh, kh, scale)
            # the probabilities' rounding to bf16 and the scores' error act on sums of p |v|
            o_tol = (bf + 3 * e) * (p @ vh.abs()) + out_half * o.abs()
            r["out"][0][:, h], r["out"][1][:, h] = o, o_tol
            lse[h] = l
            r["lse"][1][h] = 2 * e + 4 * U32 * torch.where(torch.isinf(l), torch.zeros_like(l), l.abs())
            if do is None:
                continue
            g = do[:, h]
            dq, dk, dv, ds = head_backward(qh, kh, vh, p, g, scale)
            # dS: its own rounding and P's error, and P times the errors of dO V^T and of sum dO O (O as given)
            err = (bf + 3 * e) * ds.abs() + p * (2 * q.shape[2] * U32 * (g.abs() @ vh.abs().t())
                                                 + (g.abs() * o_tol).sum(1, keepdim=True))
            r["dq"][0][:, h] = dq
            r["dq"][1][:, h] = abs(scale) * (err @ kh.abs()) + grad_half * dq.abs()
            r["dk"][0][:, h // share] += dk
            r["dk"][1][:, h // share] += abs(scale) * (err.t() @ qh.abs())
            r["dv"][0][:, h // share] += dv
            r["dv"][1][:, h // share] += (bf + 3 * e) * (p.t() @ g.abs())
        if do is not None:
            for n in ("dk", "dv"):
                r[n][1].add_(grad_half * r[n][0].abs() + 64 * U32 * r[n][1])
        res.append(r)
    return res


def rotary(x, angles, rot, pairs, mscale, inverse):
    """x f64 [tokens, heads, dim] turned by angles f64 [tokens, rot / 2]."""
    a = -angles if inverse else angles
    c, s = (torch.cos(a) * mscale)[:, None], (torch.sin(a) * mscale)[:, None]
    y = x.clone()
    i, j = (slice(0, rot // 2), slice(rot // 2, rot)) if pairs == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., i] * s + x[..., j] * c
    return y


def norm(x, residual, w, eps, wadd, dtype):
    """(h as stored, rs, y) f64."""
    h = x.double() if residual is None else (x.double() + residual.double()).to(dtype).double()
    rs = 1.0 / torch.sqrt((h * h).mean(1) + eps)
    return h, rs, h * rs[:, None] * (w.double() + wadd)


def group_index(n, group, device):
    g = n if group <= 0 or group > n else group
    return torch.arange(n, device=device) // g


def group_scale(y, group):
    """amax / 127 a group (1 where all are zero), f64."""
    idx = group_index(y.shape[1], group, y.device)
    top = torch.zeros((y.shape[0], int(idx[-1]) + 1), dtype=y.dtype, device=y.device)
    top.scatter_reduce_(1, idx.expand_as(y), y.abs(), "amax")
    return torch.where(top > 0, top / 127, torch.ones_like(top))


def norm_backward(h, rs, w, wadd, scale, group, g_codes, g_y, g_h):
    """(dx, dw, e) f64 from the definition's derivative, the scales held."""
    e = torch.zeros_like(h)
    if g_codes is not None:
        e = e + g_codes.double() / scale.double()[:, group_index(h.shape[1], group, h.device)]
    if g_y is not None:
        e = e + g_y.double()
    we = (w.double() + wadd) * e
    r = rs[:, None]
    dx = r * we - h * r ** 3 * (we * h).mean(1, keepdim=True)
    if g_h is not None:
        dx = dx + g_h.double()
    return dx, (e * h * r).sum(0), e
