"""Attention on the card, forward and backward (a front over r97q_attn_fwd and r97q_attn_bwd,
include/r97q.h).

Tensors are token-major: [batch, tokens, heads, head_dim], or [tokens, heads, head_dim] where sequences of
different lengths are packed one after the other and int32 `q_starts` / `kv_starts` [batch + 1] say where
each begins. Any strides will do, with head_dim consecutive and rows on 16 bytes: a view of a fused
projection's output, or of a [batch, heads, tokens, head_dim] cache (transpose(1, 2))."""
from __future__ import annotations

import math

import torch

from . import R97Q_BF16, R97Q_F32, AttnShape, Heads, _empty, _empty_like, _ptr, _space, _stream, check, lib


_DTYPES = {torch.bfloat16: R97Q_BF16, torch.float32: R97Q_F32}


def _heads(x: torch.Tensor, packed: bool, what: str, like=None) -> Heads:
    st, shape = x.stride(), x.shape
    if like is not None and shape != like:
        raise ValueError(f"attention: {what} has shape {tuple(like)}")
    if len(shape) != (3 if packed else 4) or not x.is_cuda or (st[-1] != 1 and x.numel()):
        raise ValueError(f"attention: {what} is a device [{'' if packed else 'batch, '}tokens, heads, head_dim] tensor, "
                         "head_dim consecutive")
    return Heads(x.data_ptr(), 0 if packed else st[0], st[-3], st[-2], shape[-2], _DTYPES.get(x.dtype, -1))


def _index(t: torch.Tensor, n: int | None, what: str) -> torch.Tensor:
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or not t.is_cuda or (n is not None and t.shape[0] != n):
        raise ValueError(f"attention: {what} is a contiguous int32 device tensor{'' if n is None else f' of {n} values'}")
    return t


def _shape(q, k, v, causal, window, scale, q_starts, kv_starts, max_q, max_kv, kv_lens) -> AttnShape:
    s = AttnShape()
    pq, pk = q_starts is not None, kv_starts is not None
    qs, ks = q.shape, k.shape
    if len(qs) != (3 if pq else 4) or len(ks) != (3 if pk else 4) or v.shape != ks or qs[-1] != ks[-1]:
        raise ValueError("attention: q and k are [batch, tokens, heads, head_dim], packed [tokens, heads, head_dim]; v has "
                         "k's shape")
    s.head_dim = qs[-1]
    s.batch = q_starts.shape[0] - 1 if pq else qs[0]
    if s.batch < 0 or s.batch != (kv_starts.shape[0] - 1 if pk else ks[0]):
        raise ValueError("attention: q and k hold as many sequences")
    if pq:
        _index(q_starts, None, "q_starts")
        if max_q is None:
            raise ValueError("attention: packed queries need max_q, their longest sequence")
        s.q_starts, s.q_tokens, s.q_len = q_starts.data_ptr(), qs[0], int(max_q)
    else:
        s.q_len = qs[1]
    if pk:
        _index(kv_starts, None, "kv_starts")
        if max_kv is None:
            raise ValueError("attention: packed keys need max_kv, their longest sequence")
        s.kv_starts, s.kv_tokens, s.kv_len = kv_starts.data_ptr(), ks[0], int(max_kv)
    else:
        s.kv_len = ks[1]
    if kv_lens is not None:
        s.kv_lens = _index(kv_lens, s.batch, "kv_lens").data_ptr()
    s.causal, s.window = int(bool(causal)), int(window)
    s.scale = 1.0 / math.sqrt(s.head_dim) if scale is None else float(scale)
    return s


def _lse_shape(s, packed):
    return (s[1], s[0]) if packed else (s[0], s[2], s[1])


def _check_lse(lse, s, packed):
    if lse.dtype != torch.float32 or lse.shape != _lse_shape(s, packed) or not lse.is_contiguous() or not lse.is_cuda:
        raise ValueError("attention: lse is a contiguous f32 [batch, heads, tokens] device tensor, packed [heads, tokens]")


def attention_fwd(q, k, v, causal: bool = True, window: int = 0, scale: float | None = None, q_starts=None,
                  kv_starts=None, max_q: int | None = None, max_kv: int | None = None, kv_lens=None, out=None,
                  out_dtype=torch.bfloat16, lse=None, workspace=None, stream=None):
    """(out, lse): out = softmax(scale q k^T) v (q's shape, `out_dtype`), lse f32 [batch, heads, tokens]. scale:
    1 / sqrt(head_dim). The last query stands at the last key; causal: a query sees no later key, window:
    and only the last `window` ones. kv_lens int32 [batch]: how much of a dense k and v is in use. Packed tokens
    outside every sequence are not written."""
    s = _shape(q, k, v, causal, window, scale, q_starts, kv_starts, max_q, max_kv, kv_lens)
    pq, pk = q_starts is not None, kv_starts is not None
    qs = q.shape
    if out is None:
        out = _empty_like(q, out_dtype, stream)
    ho = _heads(out, pq, "out", qs)
    if lse is None:
        lse = _empty(_lse_shape(qs, pq), torch.float32, q.device, stream)
    _check_lse(lse, qs, pq)
    hq, hk = _heads(q, pq, "q"), _heads(k, pk, "k")
    if workspace is None:
        need = lib().r97q_attn_fwd_workspace_bytes(s, hq.heads, hk.heads)
        if need > 0:
            workspace = _empty(need, torch.uint8, q.device, stream)
    check(lib().r97q_attn_fwd(s, hq, hk, _heads(v, pk, "v"), ho, _ptr(lse), *_space(workspace, "attention"),
                              _stream(stream)), "r97q_attn_fwd")
    return out, lse


def attention_bwd(q, k, v, out, lse, d_out, causal: bool = True, window: int = 0, scale: float | None = None,
                  q_starts=None, kv_starts=None, max_q: int | None = None, max_kv: int | None = None, kv_lens=None,
                  dq=None, dk=None, dv=None, grad_dtype=torch.bfloat16, workspace=None, stream=None):
    """(dq, dk, dv), written: the adjoint of attention_fwd with the same arguments, from its out and lse and
    the output's cotangent d_out (bf16). Packed tokens outside every sequence are not written."""
    s = _shape(q, k, v, causal, window, scale, q_starts, kv_starts, max_q, max_kv, kv_lens)
    pq, pk = q_starts is not None, kv_starts is not None

    def grad(x, like, shape, packed, what):
        if x is None:
            x = _empty_like(like, grad_dtype, stream)
        return x, _heads(x, packed, what, shape)

    qs, ks = q.shape, k.shape
    dq, hdq = grad(dq, q, qs, pq, "dq")
    dk, hdk = grad(dk, k, ks, pk, "dk")
    dv, hdv = grad(dv, v, ks, pk, "dv")
    ho, hdo = _heads(out, pq, "out", qs), _heads(d_out, pq, "d_out", qs)
    _check_lse(lse, qs, pq)
    hq, hk = _heads(q, pq, "q"), _heads(k, pk, "k")
    if workspace is None:
        need = lib().r97q_attn_bwd_workspace_bytes(s, hq.heads, hk.heads)
        workspace = _empty(max(need, 1), torch.uint8, q.device, stream)
    check(lib().r97q_attn_bwd(s, hq, hk, _heads(v, pk, "v"), ho, _ptr(lse), hdo, hdq, hdk, hdv,
                              *_space(workspace, "attention"), _stream(stream)), "r97q_attn_bwd")
    return dq, dk, dv
