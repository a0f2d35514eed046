"""The residual's addition, the RMS norm and the 8-bit group quantiser in one pass on the card, and their
adjoint (a front over r97q_add_rmsnorm_i8g and r97q_add_rmsnorm_i8g_bwd, include/r97q.h)."""
from __future__ import annotations

import torch

from . import R97Q_BF16, R97Q_F32, _empty, _ptr, _space, _stream, check, lib


def _rows(x: torch.Tensor, what: str, like: torch.Tensor | None = None) -> None:
    if x.dim() != 2 or not x.is_contiguous() or not x.is_cuda or (
            like is not None and (x.shape != like.shape or x.dtype != like.dtype)):
        raise ValueError(f"add_rmsnorm_i8g: {what} is a contiguous [rows, n] device tensor"
                         + (" of the stream's type" if like is not None else ""))


def _stream_dtype(x: torch.Tensor) -> int:
    if x.dtype == torch.bfloat16:
        return R97Q_BF16
    if x.dtype == torch.float32:
        return R97Q_F32
    raise ValueError("add_rmsnorm_i8g: the stream is bf16 or f32")


def _vector(t: torch.Tensor, dtype, shape, what: str) -> None:
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous() or not t.is_cuda:
        raise ValueError(f"add_rmsnorm_i8g: {what} is a contiguous {dtype} device tensor of shape {shape}")


def _groups(n: int, group: int) -> int:
    return 1 if group <= 0 or group > n else (n + group - 1) // group


def add_rmsnorm_i8g(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, group: int = 0,
                    eps: float = 1e-6, wadd: float = 0.0, want_codes: bool = True, want_y: bool = False,
                    codes: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                    h: torch.Tensor | None = None, y: torch.Tensor | None = None,
                    rstd: torch.Tensor | None = None, stream=None):
    """(codes int8 [rows, n], scale f32 [rows, groups], h, y, rstd f32 [rows]) of h = x + residual and
    y = h / rms(h) * (weight + wadd): h in x's dtype (x itself without a residual), a scale every `group`
    columns (<= 0: one a row), y bf16 when wanted. codes, scale, h, y and rstd may be given (h may be x or
    residual)."""
    _rows(x, "x")
    rows, n = x.shape
    dt = _stream_dtype(x)
    _vector(weight, x.dtype, (n,), "weight")

    def new(shape, dtype):
        return _empty(shape, dtype, x.device, stream)

    if residual is not None:
        _rows(residual, "residual", x)
        h = new((rows, n), x.dtype) if h is None else h
        _rows(h, "h", x)
    elif h is not None:
        raise ValueError("add_rmsnorm_i8g: without a residual h is x")
    if want_codes:
        codes = new((rows, n), torch.int8) if codes is None else codes
        scale = new((rows, _groups(n, group)), torch.float32) if scale is None else scale
        _vector(codes, torch.int8, (rows, n), "codes")
        _vector(scale, torch.float32, (rows, _groups(n, group)), "scale")
    else:
        codes = scale = None
    if want_y:
        y = new((rows, n), torch.bfloat16) if y is None else y
        _vector(y, torch.bfloat16, (rows, n), "y")
    else:
        y = None
    rstd = new((rows,), torch.float32) if rstd is None else rstd
    _vector(rstd, torch.float32, (rows,), "rstd")
    check(lib().r97q_add_rmsnorm_i8g(_ptr(x), _ptr(residual), _ptr(weight), dt, rows, n, int(group), float(eps),
                                     float(wadd), _ptr(h), _ptr(codes), _ptr(scale), _ptr(y), _ptr(rstd),
                                     _stream(stream)), "r97q_add_rmsnorm_i8g")
    return codes, scale, (x if residual is None else h), y, rstd


def add_rmsnorm_i8g_bwd(h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor, group: int = 0,
                        scale: torch.Tensor | None = None, g_codes: torch.Tensor | None = None,
                        g_y: torch.Tensor | None = None, g_h: torch.Tensor | None = None, wadd: float = 0.0,
                        dx: torch.Tensor | None = None, dw: torch.Tensor | None = None, want_dw: bool = True,
                        accumulate: bool = False, workspace: torch.Tensor | None = None, stream=None):
    """(dx, dw): the gradient of x and of the residual (h's dtype, written) and of the gain (f32 [n], written
    or, with accumulate, added to) from the cotangents of the codes (with the forward's scale), of y and of
    h, each [rows, n] in h's dtype and each optional. dx may be one of the cotangents."""
    _rows(h, "h")
    rows, n = h.shape
    dt = _stream_dtype(h)
    _vector(weight, h.dtype, (n,), "weight")
    _vector(rstd, torch.float32, (rows,), "rstd")
    for g, what in ((g_codes, "g_codes"), (g_y, "g_y"), (g_h, "g_h"), (dx, "dx")):
        if g is not None:
            _rows(g, what, h)
    if g_codes is not None:
        if scale is None:
            raise ValueError("add_rmsnorm_i8g_bwd: the codes' cotangent needs the forward's scale")
        _vector(scale, torch.float32, (rows, _groups(n, group)), "scale")
    if dx is None:
        dx = _empty((rows, n), h.dtype, h.device, stream)
    if want_dw:
        if dw is None:
            dw, accumulate = _empty(n, torch.float32, h.device, stream), False
        _vector(dw, torch.float32, (n,), "dw")
        if workspace is None:
            workspace = _empty(max(lib().r97q_add_rmsnorm_i8g_bwd_workspace_bytes(rows, n), 1), torch.uint8, h.device,
                               stream)
    else:
        dw = None
    check(lib().r97q_add_rmsnorm_i8g_bwd(_ptr(h), _ptr(weight), dt, rows, n, int(group), float(wadd), _ptr(rstd),
                                         _ptr(scale), _ptr(g_codes), _ptr(g_y), _ptr(g_h), _ptr(dx), _ptr(dw),
                                         int(bool(accumulate)),
                                         *_space(workspace if want_dw else None, "add_rmsnorm_i8g_bwd"), _stream(stream)),
          "r97q_add_rmsnorm_i8g_bwd")
    return dx, dw
