"""Rotary positions of the query and key heads on the card, with one position a token or several axes (a front over
r97q_rotary, r97q_rotary_axes and r97q_rotary_frequencies, include/r97q.h)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import (R97Q_BF16, R97Q_F32, R97Q_ROTARY_HALF, R97Q_ROTARY_INTERLEAVED, R97Q_ROTARY_LINEAR, R97Q_ROTARY_PLAIN,
               R97Q_ROTARY_RAMP, Heads, _device, _empty_like, _ptr, _stream, check, lib)

PAIRS = {"half": R97Q_ROTARY_HALF, "interleaved": R97Q_ROTARY_INTERLEAVED}
SCALINGS = {"plain": R97Q_ROTARY_PLAIN, "linear": R97Q_ROTARY_LINEAR, "ramp": R97Q_ROTARY_RAMP}


def rotary_frequencies(rot: int, base: float = 10000.0, scaling: str = "plain", factor: float = 1.0,
                       original: float = 0.0, slow: float = 1.0, fast: float = 32.0, device="cuda"):
    """(inv_freq f64 [rot / 2] on `device`, mscale): base^(-2i / rot), for a context `factor` times the
    `original` length divided by factor ("linear") or divided where a pair turns fewer than `slow` times over
    the original length, kept where it turns more than `fast` times and blended between ("ramp")."""
    if scaling not in SCALINGS:
        raise ValueError(f"rotary_frequencies: scaling {scaling!r} is not one of {sorted(SCALINGS)}")
    f = np.zeros(max(int(rot) // 2, 1), np.float64)
    m = C.c_float(1.0)
    check(lib().r97q_rotary_frequencies(int(rot), float(base), SCALINGS[scaling], float(factor), float(original),
                                        float(slow), float(fast), f.ctypes.data_as(C.c_void_p), C.byref(m)),
          "r97q_rotary_frequencies")
    return torch.from_numpy(f).to(device), float(m.value)


_DTYPES = {torch.bfloat16: R97Q_BF16, torch.float32: R97Q_F32}


def _heads(x: torch.Tensor, what: str, shape=None) -> Heads:
    st, own = x.stride(), x.shape
    if len(own) != 3 or st[2] != 1 or not x.is_cuda:
        raise ValueError(f"rotary: {what} is a device [tokens, heads, head_dim] tensor, head_dim consecutive")
    if shape is not None and own != shape:
        raise ValueError(f"rotary: {what} has {what[0]}'s shape")
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise ValueError(f"rotary: {what} is bf16 or f32")
    return Heads(x.data_ptr(), 0, st[0], st[1], own[1], dt)


def rotary(q: torch.Tensor, k: torch.Tensor | None, inv_freq: torch.Tensor, positions: torch.Tensor | None = None,
           pairs: str = "half", mscale: float = 1.0, inverse: bool = False, q_out: torch.Tensor | None = None,
           k_out: torch.Tensor | None = None, stream=None, *, _axes: tuple | None = None):
    """(q, k) [tokens, heads, head_dim] turned by positions * inv_freq (positions None: 0, 1, ..); k may be
    None. The first 2 * len(inv_freq) values of a head turn, the rest are copied. inverse: the adjoint
    (turned back, scaled by the same mscale). q_out / k_out may be q / k."""
    if pairs not in PAIRS:
        raise ValueError(f"rotary: pairs {pairs!r} are not one of {sorted(PAIRS)}")
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous() or not inv_freq.is_cuda:
        raise ValueError("rotary: inv_freq is a contiguous f64 [rot / 2] device tensor")
    qs = q.shape
    tokens, _, dim = qs if len(qs) == 3 else (0, 0, 0)
    wide = 0
    if positions is not None and _axes is None:
        if positions.dtype not in (torch.int32, torch.int64) or positions.shape != (tokens,) \
                or not positions.is_contiguous() or not positions.is_cuda:
            raise ValueError("rotary: positions are a contiguous int32 or int64 [tokens] device tensor")
        wide = int(positions.dtype == torch.int64)
    hq = _heads(q, "q")
    if q_out is None:
        q_out = _empty_like(q, q.dtype, stream)
    ho = _heads(q_out, "q_out", qs)
    hk = hko = None
    if k is not None:
        hk, ks = _heads(k, "k"), k.shape
        if k_out is None:
            k_out = _empty_like(k, k.dtype, stream)
        hko = _heads(k_out, "k_out", ks)
        if ks[0] != tokens or ks[2] != dim:
            raise ValueError("rotary: k has q's tokens and head_dim")
    elif k_out is not None:
        raise ValueError("rotary: k_out without k")
    if _axes is not None:  # rotary_axes's call: its positions and pairs' axes, checked
        check(lib().r97q_rotary_axes(hq, ho, hk, hko, tokens, dim, 2 * inv_freq.shape[0], PAIRS[pairs], _ptr(inv_freq), *_axes,
                                     float(mscale), int(bool(inverse)), _stream(stream)), "r97q_rotary_axes")
        return q_out, k_out
    check(lib().r97q_rotary(hq, ho, hk, hko, tokens, dim, 2 * inv_freq.shape[0], PAIRS[pairs], _ptr(inv_freq),
                            _ptr(positions), wide, float(mscale), int(bool(inverse)), _stream(stream)), "r97q_rotary")
    return q_out, k_out


def rotary_pair_axes(sections, order: str = "blocks", device="cuda"):
    """int32 [sum(sections)] on `device`: each pair's axis, sections[a] pairs for axis a. "blocks": the first axis's pairs,
    then the second's, ..; "cycle": the axes in turn, each as long as it has pairs left."""
    left = [int(n) for n in sections]
    if not left or min(left) < 0 or sum(left) < 1:
        raise ValueError("rotary_pair_axes: sections are counts of pairs, one or more in all")
    if order == "blocks":
        axis = [a for a, n in enumerate(left) for _ in range(n)]
    elif order == "cycle":
        axis = [a for i in range(max(left)) for a, n in enumerate(left) if i < n]
    else:
        raise ValueError(f"rotary_pair_axes: order {order!r} is not 'blocks' or 'cycle'")
    return torch.tensor(axis, dtype=torch.int32).to(device)


def rotary_axes(q: torch.Tensor, k: torch.Tensor | None, inv_freq: torch.Tensor, positions: torch.Tensor,
                pair_axis: torch.Tensor, pairs: str = "half", mscale: float = 1.0, inverse: bool = False,
                q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None, stream=None):
    """rotary with a position on each of several axes: positions int32 or int64 [axes, tokens], and pair i turns by
    positions[pair_axis[i]] * inv_freq[i] (pair_axis int32 [rot / 2]: rotary_pair_axes)."""
    device = _device(q, stream, "rotary_axes")
    for t in (k, inv_freq, positions, pair_axis, q_out, k_out):
        if t is not None and t.get_device() != device:
            raise ValueError("rotary_axes: all tensors are on q's device")
    if positions.dtype not in (torch.int32, torch.int64) or positions.dim() != 2 or positions.shape[1] != q.shape[0] \
            or (positions.shape[1] > 1 and positions.stride(1) != 1) or not positions.is_cuda:
        raise ValueError("rotary_axes: positions are an int32 or int64 [axes, tokens] device tensor, tokens consecutive")
    if pair_axis.dtype != torch.int32 or pair_axis.shape != inv_freq.shape or not pair_axis.is_contiguous() or not pair_axis.is_cuda:
        raise ValueError("rotary_axes: pair_axis is a contiguous int32 device tensor of inv_freq's shape")
    return rotary(q, k, inv_freq, positions, pairs, mscale, inverse, q_out, k_out, stream,
                  _axes=(_ptr(pair_axis), positions.shape[0], _ptr(positions), int(positions.dtype == torch.int64), positions.stride(0)))
