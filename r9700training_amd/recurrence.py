"""A gated linear recurrence over long sequences on the card, forward and backward (a front over r97q_recurrence_fwd and
r97q_recurrence_bwd, include/r97q.h):

    a = exp(-rate * sigmoid(gate)),  h[t] = a[t] * h[t - 1] + sqrt(1 - a[t]^2) * sigmoid(input_gate[t]) * x[t]

Tensors are [batch, tokens, channels], or [tokens, channels] where sequences of different lengths are packed one after the
other and int32 `starts` [batch + 1] says where each begins (max_len: the longest). All are bf16 or all f32, of any strides
with channels consecutive: a view of a fused projection's output, too. rate is f32 [channels], not negative; states are f32."""
from __future__ import annotations

import torch

from . import R97Q_BF16, R97Q_F32, Recurrence, Rows, _device, _empty, _empty_like, _space, _stream, check, lib

_DTYPES = {torch.bfloat16: R97Q_BF16, torch.float32: R97Q_F32}
_F32 = torch.float32


def _shape(x, starts, max_len) -> Recurrence:
    xs, dtype = x.shape, _DTYPES.get(x.dtype, -1)
    if len(xs) != (3 if starts is None else 2):
        raise ValueError("recurrence: x is [batch, tokens, channels], packed [tokens, channels]")
    if starts is not None:
        if starts.dtype != torch.int32 or starts.dim() != 1 or not starts.shape[0] or not starts.is_contiguous() or starts.get_device() != x.get_device():
            raise ValueError("recurrence: starts are a contiguous int32 device tensor, one more than the sequences")
        if max_len is None:
            raise ValueError("recurrence: packed sequences need max_len, the longest one's tokens")
        return Recurrence(starts.shape[0] - 1, xs[1], int(max_len), starts.data_ptr(), xs[0], dtype)
    return Recurrence(xs[0], xs[2], xs[1], None, 0, dtype)


def _rows(t: torch.Tensor, like, what: str) -> Rows:
    """like: x's shape, type and device, read once a call."""
    st, shape = t.stride(), like[0]
    if t.shape != shape or t.dtype is not like[1] or t.get_device() != like[2] or (st[-1] != 1 and shape[-1] > 1):
        raise ValueError(f"recurrence: {what} is a device tensor of x's shape and type, channels consecutive")
    return Rows(t.data_ptr(), st[0] if len(st) == 3 else 0, st[-2])


def _f32(t, shape, like, what: str):
    if t is None:
        return None
    if t.dtype is not _F32 or t.shape != shape or not t.is_contiguous() or t.get_device() != like[2]:
        raise ValueError(f"recurrence: {what} is a contiguous f32 device tensor of shape {tuple(shape)}")
    return t.data_ptr()


def _state_shape(s: Recurrence) -> tuple:
    rows = lib().r97q_recurrence_state_rows(s)
    return (max(rows, 0), s.channels) if s.starts else (s.batch, rows // s.batch if s.batch > 0 else 0, s.channels)


def recurrence_fwd(x, gate, rate, input_gate=None, h0=None, starts=None, max_len: int | None = None, out=None, last=None,
                   states=None, want_states: bool = False, workspace=None, stream=None):
    """(h, last, states): h in x's shape and type; last f32 [batch, channels], the state behind each sequence, from which the
    next tokens begin (h0: the state before it, None: zeros; last may be h0); states, where want_states asks for them or they
    are given: f32 [batch, ceil(tokens / 128), channels], packed [tokens // 128 + batch, channels], what the backward needs.
    Packed tokens outside every sequence are not written. out may be x, gate or input_gate."""
    s, like = _shape(x, starts, max_len), (x.shape, x.dtype, _device(x, stream, "recurrence"))
    ends = (s.batch, s.channels)
    if out is None:
        out = _empty_like(x, x.dtype, stream)
    if last is None:
        last = _empty(ends, torch.float32, x.device, stream)
    if want_states and states is None:
        states = _empty(_state_shape(s), torch.float32, x.device, stream)
    if workspace is None:
        need = lib().r97q_recurrence_fwd_workspace_bytes(s)
        if need > 0:
            workspace = _empty(need, torch.uint8, x.device, stream)
    check(lib().r97q_recurrence_fwd(s, _rows(x, like, "x"), _rows(gate, like, "gate"),
                                    None if input_gate is None else _rows(input_gate, like, "input_gate"),
                                    _f32(rate, (s.channels,), like, "rate"), _f32(h0, ends, like, "h0"), _rows(out, like, "out"),
                                    _f32(last, ends, like, "last"), _f32(states, states is not None and _state_shape(s), like, "states"),
                                    *_space(workspace, "recurrence"), _stream(stream)), "r97q_recurrence_fwd")
    return out, last, states


def recurrence_bwd(x, gate, rate, states, d_h, input_gate=None, d_last=None, starts=None, max_len: int | None = None,
                   dx=None, dgate=None, dinput_gate=None, drate=None, dh0=None, workspace=None, stream=None):
    """(dx, dgate, dinput_gate, drate, dh0), written: the adjoint of recurrence_fwd with the same arguments, from the states
    it kept and the cotangents d_h (x's shape and type) and d_last (f32, None: zeros). dinput_gate is None without an
    input_gate; none may be one of the inputs; drate f32 [channels] is the sum over all tokens, dh0 f32 [batch, channels]."""
    s, like = _shape(x, starts, max_len), (x.shape, x.dtype, _device(x, stream, "recurrence"))
    ends = (s.batch, s.channels)
    dx = _empty_like(x, x.dtype, stream) if dx is None else dx
    dgate = _empty_like(x, x.dtype, stream) if dgate is None else dgate
    if input_gate is not None and dinput_gate is None:
        dinput_gate = _empty_like(x, x.dtype, stream)
    if drate is None:
        drate = _empty((s.channels,), torch.float32, x.device, stream)
    if dh0 is None:
        dh0 = _empty(ends, torch.float32, x.device, stream)
    if workspace is None:
        need = lib().r97q_recurrence_bwd_workspace_bytes(s)
        if need > 0:
            workspace = _empty(need, torch.uint8, x.device, stream)
    check(lib().r97q_recurrence_bwd(s, _rows(x, like, "x"), _rows(gate, like, "gate"),
                                    None if input_gate is None else _rows(input_gate, like, "input_gate"),
                                    _f32(rate, (s.channels,), like, "rate"), _f32(states, _state_shape(s), like, "states"),
                                    _rows(d_h, like, "d_h"), _f32(d_last, ends, like, "d_last"), _rows(dx, like, "dx"), _rows(dgate, like, "dgate"),
                                    None if dinput_gate is None else _rows(dinput_gate, like, "dinput_gate"),
                                    _f32(drate, (s.channels,), like, "drate"), _f32(dh0, ends, like, "dh0"),
                                    *_space(workspace, "recurrence"), _stream(stream)), "r97q_recurrence_bwd")
    return dx, dgate, dinput_gate, drate, dh0
