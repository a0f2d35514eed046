"""The gated recurrence in float64, token by token, from its definition, and how far a correct f32 implementation may lie from
it: every rounding counted at half a step, errors carried along the sequence by the recurrence itself.

U is half a step of f32. A hardware exponential, reciprocal or root is off by 2 U; a sigmoid's exponent g log2 e is rounded, an
absolute error, so its relative error is (|g| + 8) U; the decay's logarithm, rate times that, and the root of 1 - a^2 follow
from it. A product of decays is off by what its logarithms are, and by a rounding for each token (joins of spans make fewer,
but up to 100 at once: a thread's tokens, a wave's spans, the waves, the ranges)."""
from __future__ import annotations

import torch

U = torch.finfo(torch.float32).eps / 2
JOIN = 100


def parts(x, gate, rate, input_gate):
    """(s, log a, a, q = 1 - a^2, sigmoid of the input's gate) f64"""
    s = torch.sigmoid(gate)
    la = -rate * s
    return s, la, torch.exp(la), -torch.expm1(2 * la), torch.ones_like(x) if input_gate is None else torch.sigmoid(input_gate)


def carry(a, e, first):
    """v[t] = a[t] (v[t - 1] + e[t]), from v[-1] = first"""
    out = []
    for t in range(a.shape[0]):
        first = a[t] * (first + e[t])
        out.append(first)
    return torch.stack(out) if out else torch.zeros_like(a)


def forward(x, gate, rate, input_gate, h0):
    """x f64 [tokens, channels], rate and h0 [channels]. A dict: h, last, before (each token's state before it) as (value,
    error without the output's rounding)."""
    s, la, a, q, si = parts(x, gate, rate, input_gate)
    eg = (gate.abs() + 8) * U
    ei = 0.0 if input_gate is None else (input_gate.abs() + 8) * U
    w = si * x
    root = torch.sqrt(q)
    u = root * w
    eu = ei + (eg + 12 * U) / 2 + 6 * U                      # relative
    before, size, h, g = [], [], h0, h0.abs()
    for t in range(x.shape[0]):
        before.append(h)
        size.append(g)
        h = a[t] * h + u[t]
        g = a[t] * g + u[t].abs()
    before, size = torch.stack(before + [h]), torch.stack(size + [g])
    # the error's own recurrence: of the state's size, what this decay and its rounding put wrong; of the input, its own
    off = torch.zeros_like(h0)
    err = [off]
    for t in range(x.shape[0]):
        off = a[t] * (off + size[t] * (la[t].abs() * (eg[t] + 4 * U) + U)) + u[t].abs() * eu[t]
        err.append(off)
    err = torch.stack(err) + JOIN * U * size
    return dict(h=(before[1:], err[1:]), last=(before[-1], err[-1]), before=(before[:-1], err[:-1]))


def backward(x, gate, rate, input_gate, h0, d_h, d_last):
    """A dict: dx, dgate, dinput_gate, drate, dh0 as (value, error without the output's rounding)."""
    s, la, a, q, si = parts(x, gate, rate, input_gate)
    eg = (gate.abs() + 8) * U
    ei = torch.zeros_like(x) if input_gate is None else (input_gate.abs() + 8) * U
    w, root = si * x, torch.sqrt(q)
    inv = torch.where(q > 0, 1 / torch.where(q > 0, root, torch.ones_like(root)), torch.zeros_like(q))
    before, e_before = forward(x, gate, rate, input_gate, h0)["before"]
    n = x.shape[0]
    lam, size, err = [None] * n, [None] * n, [None] * n
    m, g, off = d_last, d_last.abs(), torch.zeros_like(d_last)
    for t in range(n - 1, -1, -1):
        lam[t], size[t] = m + d_h[t], g + d_h[t].abs()
        err[t] = off + 2 * U * size[t]
        off = a[t] * (err[t] + size[t] * (la[t].abs() * (eg[t] + 4 * U) + U))
        m, g = a[t] * lam[t], a[t] * size[t]
    dh0 = (m, off + JOIN * U * g)
    if not n:
        return dict(dx=(x, x), dgate=(x, x), dinput_gate=(x, x), drate=(torch.zeros_like(rate), torch.zeros_like(rate)), dh0=dh0)
    lam, size, err = torch.stack(lam), torch.stack(size), torch.stack(err)
    err = err + JOIN * U * size
    near = a * w * inv
    e_near = near.abs() * (ei + (eg + 12 * U) / 2 + la.abs() * eg + 10 * U)
    dlog = lam * a * (before - near)
    e_dlog = a * (err * (before - near).abs() + (lam.abs() + err) * (e_before + e_near + 2 * U * (before.abs() + near.abs()))) \
        + dlog.abs() * (la.abs() * eg + 8 * U)
    d = s * dlog
    e_d = s * e_dlog + d.abs() * (eg + U)
    dgate = -rate * (1 - s) * d
    e_dgate = rate * ((1 - s) * e_d + d.abs() * (s * eg + 4 * U)) + dgate.abs() * 6 * U
    dw = lam * root
    e_dw = err * root + dw.abs() * ((eg + 12 * U) / 2 + 6 * U)
    dx = dw * si
    e_dx = e_dw * si + dx.abs() * (ei + 2 * U)
    di = dx * x * (1 - si)
    e_di = e_dx * x.abs() * (1 - si) + (dx * x).abs() * (si * ei + 4 * U) + di.abs() * 4 * U
    return dict(dx=(dx, e_dx), dgate=(dgate, e_dgate), dinput_gate=(di, e_di),
                drate=(-d.sum(0), e_d.sum(0) + (n / 8 + JOIN) * U * d.abs().sum(0)), dh0=dh0)
