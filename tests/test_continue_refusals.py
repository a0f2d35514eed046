"""What the operators that continue a sequence refuse, on the host before any GPU work (no GPU needed: the pointers below are
never dereferenced, each call returns its status first)."""
import ctypes as C

import pytest
import torch

from r9700training_amd import AttnShape, Heads, Pages, R97qError, Recurrence, Rows, lib

OK, EINVAL, EUNSUPPORTED, EWORKSPACE = 0, 1, 2, 4
FAKE = 0x10000
BF16, F32 = 1, 0


def fields(s, kw):
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def heads(n=4, d=64, data=FAKE, dtype=BF16, **kw):
    return fields(Heads(data, 100 * n * d, n * d, d, n, dtype), kw)


# ------------------------------------------------------------------ rotary with axes
def axes(q=None, q_out=None, k=None, k_out=None, tokens=10, dim=64, rot=64, pairs=0, freq=FAKE, pair_axis=FAKE, n=3, pos=FAKE,
         stride=10):
    return lib().r97q_rotary_axes(q or heads(), q_out or heads(), k, k_out, tokens, dim, rot, pairs, freq, pair_axis, n, pos, 0,
                                  stride, 1.0, 0, None)


@pytest.mark.parametrize("bad,code", [
    (dict(pair_axis=None), EINVAL), (dict(pos=None), EINVAL), (dict(n=0), EINVAL), (dict(n=-1), EINVAL), (dict(stride=-10), EINVAL),
    (dict(freq=None), EINVAL), (dict(rot=0), EINVAL), (dict(rot=7), EINVAL), (dict(rot=66), EINVAL), (dict(pairs=2), EINVAL),
    (dict(tokens=-1), EINVAL), (dict(tokens=1 << 31), EINVAL), (dict(k=heads(2)), EINVAL), (dict(k_out=heads(2)), EINVAL),
    (dict(q=heads(dtype=2)), EINVAL), (dict(q_out=heads(dtype=F32)), EINVAL), (dict(q_out=heads(2)), EINVAL),
    (dict(q_out=heads(token_stride=0)), EINVAL), (dict(q=heads(data=0)), EINVAL), (dict(dim=1 << 20, rot=16386), EUNSUPPORTED)])
def test_rotary_axes(bad, code):
    assert axes(**bad) == code and b"r97q_rotary_axes" in lib().r97q_last_error()


def test_rotary_axes_of_no_tokens():
    assert axes(tokens=0, pos=None) == OK


# ------------------------------------------------------------------ the paged cache
def shape(**kw):
    return fields(AttnShape(batch=2, head_dim=64, q_len=10, kv_len=100, kv_lens=FAKE, causal=1, scale=0.125), kw)


def pages(**kw):
    return fields(Pages(FAKE, 8, 100, 16, 8), kw)


def pool(n=2, d=64, page=16, **kw):
    return fields(Heads(FAKE, page * n * d, n * d, d, n, BF16), kw)


def fwd(s=None, p=None, q=None, k=None, v=None, out=None, ws=FAKE, nws=1 << 40):
    return lib().r97q_paged_attn_fwd(s or shape(), p or pages(), q or heads(), k or pool(), v or pool(), out or heads(), FAKE, ws, nws, None)


def write(s=None, p=None, k=None, v=None, kp=None, vp=None):
    return lib().r97q_paged_write(s or shape(), p or pages(), k or heads(2), v or heads(2), kp or pool(), vp or pool(), None)


SHAPES = [
    (dict(head_dim=0), EINVAL), (dict(head_dim=12), EUNSUPPORTED), (dict(head_dim=264), EUNSUPPORTED), (dict(batch=-1), EINVAL),
    (dict(q_len=-1), EINVAL), (dict(kv_len=-5), EINVAL), (dict(batch=65536), EUNSUPPORTED), (dict(q_len=1 << 31), EUNSUPPORTED),
    (dict(kv_len=1 << 31), EUNSUPPORTED), (dict(window=-1), EINVAL), (dict(window=4, causal=0), EINVAL), (dict(kv_lens=None), EINVAL),
    (dict(kv_lens=None, kv_starts=FAKE), EINVAL), (dict(kv_starts=FAKE), EINVAL), (dict(q_starts=FAKE, q_tokens=-1), EINVAL),
    (dict(scale=float("nan")), EINVAL), (dict(scale=float("inf")), EINVAL),
]


@pytest.mark.parametrize("bad,code", SHAPES)
def test_paged_shapes(bad, code):
    assert fwd(shape(**bad)) == code and b"r97q_paged_attn_fwd" in lib().r97q_last_error()
    assert write(shape(**bad)) == code and b"r97q_paged_write" in lib().r97q_last_error()
    assert lib().r97q_paged_attn_fwd_workspace_bytes(shape(**bad), pages(), 4, 2) == -1


PAGES = [
    (dict(pages=-1), EINVAL), (dict(max_pages=-1), EINVAL), (dict(table_stride=-8), EINVAL), (dict(page_size=0), EINVAL),
    (dict(page_size=-16), EINVAL), (dict(page_size=4), EUNSUPPORTED), (dict(page_size=24), EUNSUPPORTED), (dict(page_size=1 << 21), EUNSUPPORTED),
    (dict(pages=1 << 31), EUNSUPPORTED), (dict(max_pages=1 << 27), EUNSUPPORTED), (dict(table=None), EINVAL),
]


@pytest.mark.parametrize("bad,code", PAGES)
def test_pages(bad, code):
    assert fwd(p=pages(**bad)) == code
    assert write(p=pages(**bad)) == code
    assert lib().r97q_paged_attn_fwd_workspace_bytes(shape(), pages(**bad), 4, 2) == -1
    assert lib().r97q_paged_attn_fwd(shape(), None, heads(), pool(), pool(), heads(), FAKE, FAKE, 1 << 40, None) == EINVAL


HEADS = [
    (dict(data=0), EINVAL), (dict(dtype=7), EINVAL), (dict(data=FAKE + 2), EUNSUPPORTED), (dict(token_stride=260), EUNSUPPORTED),
    (dict(head_stride=65), EUNSUPPORTED), (dict(batch_stride=1001), EUNSUPPORTED), (dict(token_stride=-256), EINVAL),
    (dict(head_stride=-64), EINVAL), (dict(batch_stride=-2560), EINVAL), (dict(heads=3), EINVAL), (dict(token_stride=(1 << 24) + 8), EUNSUPPORTED),
]


@pytest.mark.parametrize("bad,code", HEADS)
def test_paged_tensors(bad, code):
    for which in ("k", "v"):
        assert fwd(**{which: pool(**bad)}) == code, which
        assert write(**{which: heads(2, **bad)}) == code, which
    assert fwd(q=heads(**bad)) == code
    assert fwd(out=heads(**bad)) == code
    for which in ("kp", "vp"):
        assert write(**{which: pool(**bad)}) == code, which


def test_paged_types_and_outputs():
    assert fwd(q=heads(dtype=F32)) == EINVAL and fwd(k=pool(dtype=F32)) == EINVAL
    assert write(k=heads(2, dtype=F32)) == EINVAL and write(kp=pool(dtype=F32)) == EINVAL
    assert write(kp=pool(token_stride=0)) == EINVAL and write(vp=pool(batch_stride=0)) == EINVAL
    assert fwd(out=heads(token_stride=0)) == EINVAL
    assert lib().r97q_paged_write(shape(), pages(), None, heads(2), pool(), pool(), None) == EINVAL
    assert lib().r97q_paged_attn_fwd(shape(), pages(), None, pool(), pool(), heads(), FAKE, FAKE, 0, None) == EINVAL


def test_paged_workspace():
    """Few rows over many tokens are cut: their workspace is asked for, and checked."""
    s, p = shape(q_len=1, kv_len=30000), pages(max_pages=2000)
    need = lib().r97q_paged_attn_fwd_workspace_bytes(s, p, 4, 2)
    assert need > 0
    for ws, n in ((FAKE, need - 1), (None, need), (FAKE, 0)):
        assert fwd(s, p, ws=ws, nws=n) == EWORKSPACE
    assert fwd(s, p, ws=FAKE + 4, nws=need) == EINVAL
    assert lib().r97q_paged_attn_fwd_workspace_bytes(shape(q_len=0), pages(), 4, 2) == 0


def test_paged_of_nothing():
    assert fwd(shape(batch=0)) == OK and fwd(shape(q_len=0)) == OK and write(shape(batch=0)) == OK and write(shape(q_len=0)) == OK
    assert write(p=pages(pages=0)) == OK and write(p=pages(max_pages=0, table=None)) == OK


# ------------------------------------------------------------------ the recurrence
def rec(**kw):
    return fields(Recurrence(2, 64, 10, None, 0, BF16), kw)


def rows(**kw):
    return fields(Rows(FAKE, 640, 64), kw)


def rfwd(s=None, x=None, gate=None, gi=None, rate=FAKE, h=None, ws=FAKE, nws=1 << 40):
    return lib().r97q_recurrence_fwd(s or rec(), x or rows(), gate or rows(), gi or rows(), rate, FAKE, h or rows(), FAKE, FAKE, ws, nws, None)


def rbwd(s=None, x=None, gate=None, gi=None, rate=FAKE, states=FAKE, d_h=None, dx=None, dgate=None, dgi=None, drate=FAKE, ws=FAKE, nws=1 << 40):
    return lib().r97q_recurrence_bwd(s or rec(), x or rows(), gate or rows(), gi or rows(), rate, states, d_h or rows(), FAKE, dx or rows(),
                                     dgate or rows(), dgi or rows(), drate, FAKE, ws, nws, None)


@pytest.mark.parametrize("bad,code", [
    (dict(batch=-1), EINVAL), (dict(len=-1), EINVAL), (dict(channels=0), EINVAL), (dict(channels=-4), EINVAL), (dict(dtype=2), EINVAL),
    (dict(dtype=-1), EINVAL), (dict(starts=FAKE, tokens=-1), EINVAL), (dict(batch=65536), EUNSUPPORTED), (dict(len=1 << 31), EUNSUPPORTED),
    (dict(starts=FAKE, tokens=1 << 31), EUNSUPPORTED), (dict(channels=(1 << 27) + 1), EUNSUPPORTED)])
def test_recurrence_shapes(bad, code):
    assert rfwd(rec(**bad)) == code and b"r97q_recurrence_fwd" in lib().r97q_last_error()
    assert rbwd(rec(**bad)) == code and b"r97q_recurrence_bwd" in lib().r97q_last_error()
    for query in (lib().r97q_recurrence_state_rows, lib().r97q_recurrence_fwd_workspace_bytes, lib().r97q_recurrence_bwd_workspace_bytes):
        assert query(rec(**bad)) == -1


@pytest.mark.parametrize("bad", [dict(data=0), dict(data=FAKE + 1), dict(token_stride=-64), dict(batch_stride=-640)])
def test_recurrence_tensors(bad):
    for which in ("x", "gate", "gi", "h"):
        assert rfwd(**{which: rows(**bad)}) == EINVAL, which
    for which in ("x", "gate", "gi", "d_h", "dx", "dgate", "dgi"):
        assert rbwd(**{which: rows(**bad)}) == EINVAL, which


@pytest.mark.parametrize("bad", [dict(token_stride=0), dict(batch_stride=0), dict(token_stride=63)])
def test_recurrence_outputs(bad):
    """Not through a stride of zero, nor with tokens over each other."""
    assert rfwd(h=rows(**bad)) == EINVAL
    for which in ("dx", "dgate", "dgi"):
        assert rbwd(**{which: rows(**bad)}) == EINVAL, which


def test_recurrence_missing():
    x = rows()
    assert rfwd(rate=None) == EINVAL and rbwd(rate=None) == EINVAL and rbwd(drate=None) == EINVAL and rbwd(states=None) == EINVAL
    assert lib().r97q_recurrence_fwd(rec(), None, x, x, FAKE, None, x, None, None, None, 0, None) == EINVAL
    # the gate on the input and its gradient come together
    assert lib().r97q_recurrence_bwd(rec(), x, x, None, FAKE, FAKE, x, None, x, x, x, FAKE, None, FAKE, 1 << 40, None) == EINVAL
    assert lib().r97q_recurrence_bwd(rec(), x, x, x, FAKE, FAKE, x, None, x, x, None, FAKE, None, FAKE, 1 << 40, None) == EINVAL


def test_recurrence_outputs_over_inputs():
    """The backward reads its inputs while its outputs are written; the forward's output may be an input, strides and all."""
    own = {n: rows(data=FAKE + 0x10000 * i) for i, n in enumerate(("x", "gate", "gi", "d_h", "dx", "dgate", "dgi"))}
    for out in ("dx", "dgate", "dgi"):
        for other in own:
            if other != out:
                assert rbwd(**{**own, out: rows(data=own[other].data)}) == EINVAL and b"over" in lib().r97q_last_error(), (out, other)
    x = own["x"]
    call = lib().r97q_recurrence_bwd
    assert call(rec(), x, own["gate"], None, FAKE, FAKE, own["d_h"], FAKE, own["dx"], own["dgate"], None, FAKE, FAKE, FAKE, 1 << 40, None) == EINVAL
    for which in ("x", "gate", "gi"):
        assert rfwd(**{**{n: own[n] for n in ("x", "gate", "gi")}, "h": rows(data=own[which].data, token_stride=128)}) == EINVAL, which


def test_recurrence_workspace():
    s = rec(batch=1, len=16384)
    for call, need in ((rfwd, lib().r97q_recurrence_fwd_workspace_bytes(s)), (rbwd, lib().r97q_recurrence_bwd_workspace_bytes(s))):
        assert need > 0
        for ws, n in ((FAKE, need - 1), (None, need), (FAKE, 0)):
            assert call(s, ws=ws, nws=n) == EWORKSPACE
        assert call(s, ws=FAKE + 4, nws=need) == EINVAL
    assert lib().r97q_recurrence_fwd_workspace_bytes(rec()) == 0
    assert lib().r97q_recurrence_state_rows(rec(len=300)) == 6
    assert lib().r97q_recurrence_state_rows(rec(starts=FAKE, tokens=300, batch=3)) == 5


def test_recurrence_of_nothing():
    assert rfwd(rec(batch=0)) == OK


# ------------------------------------------------------------------ the fronts
def test_fronts_take_device_tensors_of_the_right_shapes():
    from r9700training_amd.paged import paged_attention_fwd, paged_write
    from r9700training_amd.recurrence import recurrence_bwd, recurrence_fwd
    from r9700training_amd.rotary import rotary_axes, rotary_pair_axes

    t = torch.zeros
    ints = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(ValueError):
        paged_write(bf(2, 3, 2, 64), bf(2, 3, 2, 64), bf(9, 16, 2, 64), bf(9, 16, 2, 64), ints(2, 4), ints(2))
    with pytest.raises(ValueError):
        paged_attention_fwd(bf(2, 3, 4, 64), bf(9, 16, 2, 64), bf(9, 16, 2, 64), ints(2, 4), ints(2))
    with pytest.raises(ValueError):
        paged_attention_fwd(bf(2, 3, 4, 64), bf(9, 16, 2, 32), bf(9, 16, 2, 32), ints(2, 4), ints(2))
    for call in (lambda: recurrence_fwd(bf(2, 3), bf(2, 3), t(3)), lambda: recurrence_fwd(bf(2, 3, 4), bf(2, 3, 4), t(4)),
                 lambda: recurrence_bwd(bf(2, 3, 4), bf(2, 3, 4), t(4), t(2, 1, 4), bf(2, 3, 4))):
        with pytest.raises((ValueError, R97qError)):
            call()
    with pytest.raises(ValueError):
        rotary_axes(bf(5, 2, 8), None, t(4, dtype=torch.float64), ints(3, 5), ints(4))
    assert rotary_pair_axes([3, 2, 1], device="cpu").tolist() == [0, 0, 0, 1, 1, 2]
    assert rotary_pair_axes([3, 2, 1], "cycle", device="cpu").tolist() == [0, 1, 2, 0, 1, 0]
    for sections, order in (([], "blocks"), ([-1, 2], "blocks"), ([0, 0], "blocks"), ([1, 1], "rows")):
        with pytest.raises(ValueError):
            rotary_pair_axes(sections, order, device="cpu")


def test_structs_match_the_header():
    assert C.sizeof(Pages) == 32 and C.sizeof(Recurrence) == 40 and C.sizeof(Rows) == 24
