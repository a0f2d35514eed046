"""A paged cache on the card: the write of new keys and values into it and attention of new tokens over it (a front over
r97q_paged_write and r97q_paged_attn_fwd, include/r97q.h).

k_pages and v_pages are pools [pages, page_size, heads, head_dim] in bf16 (any strides, head_dim consecutive: also a view of
[pages, heads, page_size, head_dim]). page_table int32 [batch, most pages]: token j of sequence b lies in slot j % page_size of
page page_table[b, j // page_size]. kv_lens int32 [batch]: the tokens that each sequence has, its new ones with them. New
tokens are [batch, tokens, heads, head_dim], or [tokens, heads, head_dim] where sequences with different numbers of them are
packed one after the other and int32 q_starts [batch + 1] says where each begins (max_q: the longest)."""
from __future__ import annotations

import math

import torch

from . import AttnShape, Pages, _device, _empty, _empty_like, _ptr, _space, _stream, check, lib
from .attention import _check_lse, _heads, _index, _lse_shape


def _cache(q, k_pages, v_pages, page_table, kv_lens, q_starts, max_q, max_kv=None, causal=0, window=0, scale=1.0, stream=None):
    """(shape, pages) of a call whose new tokens are shaped like q."""
    packed = q_starts is not None
    qs, ks, ts, st = q.shape, k_pages.shape, page_table.shape, page_table.stride()
    if len(qs) != (3 if packed else 4) or len(ks) != 4 or v_pages.shape != ks or qs[-1] != ks[-1]:
        raise ValueError("paged: new tokens are [batch, tokens, heads, head_dim], packed [tokens, heads, head_dim]; k_pages and "
                         "v_pages [pages, page_size, heads, head_dim]")
    if page_table.dtype != torch.int32 or len(ts) != 2 or (ts[1] > 1 and st[1] != 1):
        raise ValueError("paged: page_table is an int32 [batch, most pages] device tensor, a row's entries consecutive")
    device = _device(q, stream, "paged")
    if k_pages.get_device() != device or v_pages.get_device() != device or page_table.get_device() != device \
            or kv_lens.get_device() != device or (packed and q_starts.get_device() != device):
        raise ValueError("paged: the pages, the table, the lengths and the starts are on the new tokens' device")
    batch, starts, tokens = ts[0], None, 0
    if packed:
        starts = _index(q_starts, batch + 1, "q_starts").data_ptr()
        if max_q is None:
            raise ValueError("paged: packed tokens need max_q, the longest sequence's")
        tokens, length = qs[0], int(max_q)
    else:
        if qs[0] != batch:
            raise ValueError("paged: page_table has a row for each sequence")
        length = qs[1]
    held = ts[1] * ks[1] if max_kv is None else int(max_kv)
    return (AttnShape(batch, qs[-1], length, held, starts, None, tokens, 0, _index(kv_lens, batch, "kv_lens").data_ptr(), window, causal, scale),
            Pages(page_table.data_ptr(), st[0], ks[0], ks[1], ts[1]))


def paged_write(k, v, k_pages, v_pages, page_table, kv_lens, q_starts=None, max_q: int | None = None, stream=None):
    """The new tokens' keys and values (bf16 or f32) into the pools: the last n of a sequence's kv_lens tokens are its n new
    ones. Tokens before the sequence, past the table's room or without a page are left out."""
    packed = q_starts is not None
    if v.shape != k.shape or v.get_device() != k.get_device():
        raise ValueError("paged: v has k's shape and device")
    s, p = _cache(k, k_pages, v_pages, page_table, kv_lens, q_starts, max_q, stream=stream)
    check(lib().r97q_paged_write(s, p, _heads(k, packed, "k"), _heads(v, packed, "v"), _heads(k_pages, False, "k_pages"),
                                 _heads(v_pages, False, "v_pages"), _stream(stream)), "r97q_paged_write")


def paged_attention_fwd(q, k_pages, v_pages, page_table, kv_lens, causal: bool = True, window: int = 0,
                        scale: float | None = None, q_starts=None, max_q: int | None = None, max_kv: int | None = None,
                        out=None, out_dtype=torch.bfloat16, lse=None, workspace=None, stream=None):
    """(out, lse) as attention_fwd's, of new tokens q over the cache that holds them: the last query stands at a sequence's
    last token, causal: a query sees no later one, window: and only the last `window`. scale: 1 / sqrt(head_dim). max_kv: the
    longest sequence's tokens where the program knows them (the call is planned for it), else what the table has room for.
    Packed tokens outside every sequence are not written."""
    packed = q_starts is not None
    qs = q.shape
    s, p = _cache(q, k_pages, v_pages, page_table, kv_lens, q_starts, max_q, max_kv, int(bool(causal)), int(window),
                  1.0 / math.sqrt(max(qs[-1], 1)) if scale is None else float(scale), stream)
    if out is None:
        out = _empty_like(q, out_dtype, stream)
    ho = _heads(out, packed, "out", qs)
    if lse is None:
        lse = _empty(_lse_shape(qs, packed), torch.float32, q.device, stream)
    _check_lse(lse, qs, packed)
    if out.get_device() != q.get_device() or lse.get_device() != q.get_device():
        raise ValueError("paged: out and lse are on q's device")
    hq, hk = _heads(q, packed, "q"), _heads(k_pages, False, "k_pages")
    if workspace is None:
        need = lib().r97q_paged_attn_fwd_workspace_bytes(s, p, hq.heads, hk.heads)
        if need > 0:
            workspace = _empty(need, torch.uint8, q.device, stream)
    check(lib().r97q_paged_attn_fwd(s, p, hq, hk, _heads(v_pages, False, "v_pages"), ho, _ptr(lse),
                                    *_space(workspace, "paged"), _stream(stream)), "r97q_paged_attn_fwd")
    return out, lse
