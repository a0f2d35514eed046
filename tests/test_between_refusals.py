"""What the operators between the projections refuse, on the host before any GPU work (no GPU needed: the
pointers below are never dereferenced, each call returns its status first)."""
import ctypes as C

import pytest

from r9700training_amd import AttnShape, Heads, lib

OK, EINVAL, EUNSUPPORTED, EWORKSPACE = 0, 1, 2, 4
FAKE = 0x10000
BF16, F32 = 1, 0


def heads(n=4, d=64, data=FAKE, dtype=BF16, **kw):
    h = Heads(data, 100 * n * d, n * d, d, n, dtype)
    for k, v in kw.items():
        setattr(h, k, v)
    return h


def shape(**kw):
    s = AttnShape(batch=2, head_dim=64, q_len=10, kv_len=10, causal=1, scale=0.125)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def fwd(s, q=None, k=None, v=None, out=None, ws=FAKE, nws=1 << 40):
    q, k, v, out = q or heads(), k or heads(2), v or heads(2), out or heads()
    return lib().r97q_attn_fwd(s, q, k, v, out, FAKE, ws, nws, None)


def bwd(s, q=None, k=None, v=None, out=None, lse=FAKE, d_out=None, dq=None, dk=None, dv=None, ws=FAKE, nws=1 << 40):
    q, k, v, out = q or heads(), k or heads(2), v or heads(2), out or heads()
    return lib().r97q_attn_bwd(s, q, k, v, out, lse, d_out or heads(), dq or heads(), dk or heads(2), dv or heads(2),
                               ws, nws, None)


SHAPES = [
    (dict(head_dim=0), EINVAL), (dict(head_dim=-8), EINVAL), (dict(head_dim=12), EUNSUPPORTED),
    (dict(head_dim=264), EUNSUPPORTED), (dict(batch=-1), EINVAL), (dict(q_len=-1), EINVAL), (dict(kv_len=-5), EINVAL),
    (dict(batch=65536), EUNSUPPORTED), (dict(q_len=1 << 31), EUNSUPPORTED), (dict(q_len=1 << 30), EUNSUPPORTED),
    (dict(kv_len=1 << 31), EUNSUPPORTED), (dict(window=-1), EINVAL), (dict(window=4, causal=0), EINVAL),
    (dict(kv_starts=FAKE, kv_lens=FAKE), EINVAL), (dict(q_starts=FAKE, q_tokens=-1), EINVAL),
    (dict(kv_starts=FAKE, kv_tokens=-1), EINVAL), (dict(scale=float("nan")), EINVAL), (dict(scale=float("inf")), EINVAL),
]


@pytest.mark.parametrize("bad,code", SHAPES)
def test_attention_shapes(bad, code):
    assert fwd(shape(**bad)) == code and lib().r97q_last_error()
    assert bwd(shape(**bad)) == code and lib().r97q_last_error()
    assert lib().r97q_attn_fwd_workspace_bytes(shape(**bad), 4, 2) == -1
    assert lib().r97q_attn_bwd_workspace_bytes(shape(**bad), 4, 2) == -1


HEADS = [
    (dict(data=0), EINVAL), (dict(dtype=F32), EINVAL), (dict(dtype=7), EINVAL), (dict(data=FAKE + 2), EUNSUPPORTED),
    (dict(token_stride=260), EUNSUPPORTED), (dict(head_stride=65), EUNSUPPORTED), (dict(batch_stride=1001), EUNSUPPORTED),
    (dict(token_stride=-256), EINVAL), (dict(head_stride=-64), EINVAL), (dict(batch_stride=-2560), EINVAL),
]


@pytest.mark.parametrize("bad,code", HEADS)
def test_attention_tensors(bad, code):
    for which in ("q", "k", "v", "d_out"):
        t = heads(2 if which in "kv" else 4, **bad)
        if which != "d_out":
            assert fwd(shape(), **{which: t}) == code, which
        assert bwd(shape(), **{which: t}) == code, which
    if bad != dict(dtype=F32):  # outputs, and the forward's output in the backward, may be f32
        assert fwd(shape(), out=heads(**bad)) == code
        for which in ("out", "dq", "dk", "dv"):
            assert bwd(shape(), **{which: heads(2 if which in ("dk", "dv") else 4, **bad)}) == code, which


def test_attention_outputs_do_not_overlap_themselves():
    for zero in ("token_stride", "head_stride", "batch_stride"):
        assert fwd(shape(), out=heads(**{zero: 0})) == EINVAL, zero
        for which in ("dq", "dk", "dv"):
            assert bwd(shape(), **{which: heads(2 if which != "dq" else 4, **{zero: 0})}) == EINVAL, (which, zero)


def test_attention_heads_and_nulls():
    L = lib()
    assert fwd(shape(), k=heads(3), v=heads(3)) == EINVAL          # 4 query heads over 3
    assert fwd(shape(), v=heads(4)) == EINVAL                      # v's heads are k's
    assert fwd(shape(), out=heads(2)) == EINVAL
    assert fwd(shape(), q=heads(0)) == EINVAL
    assert L.r97q_attn_fwd(None, heads(), heads(), heads(), heads(), FAKE, None, 0, None) == EINVAL
    assert L.r97q_attn_fwd(shape(), None, heads(), heads(), heads(), FAKE, None, 0, None) == EINVAL
    assert bwd(shape(), lse=None) == EINVAL
    assert bwd(shape(), ws=None) == EWORKSPACE
    need = L.r97q_attn_bwd_workspace_bytes(shape(), 4, 2)
    assert need >= 4 * 2 * 4 * 10
    assert bwd(shape(), nws=need - 1) == EWORKSPACE
    # nothing to do: done
    assert fwd(shape(batch=0)) == OK and bwd(shape(batch=0)) == OK
    assert fwd(shape(q_len=0)) == OK


def rotary(q=None, qo=None, k="same", ko="same", tokens=5, dim=64, rot=64, pairs=0, freq=FAKE):
    k = heads(2) if k == "same" else k
    ko = heads(2) if ko == "same" else ko
    return lib().r97q_rotary(q or heads(), qo or heads(), k, ko, tokens, dim, rot, pairs, freq, None, 0, 1.0, 0, None)


@pytest.mark.parametrize("kw,code", [
    (dict(rot=0), EINVAL), (dict(rot=7), EINVAL), (dict(rot=66), EINVAL), (dict(dim=0), EINVAL), (dict(pairs=2), EINVAL),
    (dict(tokens=-1), EINVAL), (dict(tokens=1 << 31), EINVAL), (dict(freq=None), EINVAL), (dict(ko=None), EINVAL),
    (dict(k=None), EINVAL), (dict(q=heads(dtype=3)), EINVAL), (dict(k=heads(2, dtype=F32)), EINVAL),
    (dict(qo=heads(dtype=F32)), EINVAL), (dict(qo=heads(3)), EINVAL), (dict(q=heads(0)), EINVAL),
    (dict(qo=heads(token_stride=0)), EINVAL), (dict(ko=heads(2, head_stride=0)), EINVAL), (dict(q=heads(data=0)), EINVAL),
    (dict(q=heads(token_stride=-1)), EINVAL), (dict(dim=65, rot=64, pairs=1), EUNSUPPORTED),
    (dict(dim=16384, rot=8194), EUNSUPPORTED)])
def test_rotary(kw, code):
    assert rotary(**kw) == code and lib().r97q_last_error()


def test_rotary_nothing_to_do():
    assert rotary(tokens=0) == OK


@pytest.mark.parametrize("args,code", [
    ((0, 1e4, 0, 1, 0, 0, 0), EINVAL), ((7, 1e4, 0, 1, 0, 0, 0), EINVAL), ((8, 0.0, 0, 1, 0, 0, 0), EINVAL),
    ((8, 1e4, 3, 1, 0, 0, 0), EINVAL), ((8, 1e4, 1, 0.0, 0, 0, 0), EINVAL), ((8, 1e4, 2, 4.0, 0.0, 1, 32), EINVAL),
    ((8, 1e4, 2, 4.0, 4096, 32, 1), EINVAL)])
def test_rotary_frequencies(args, code):
    out = (C.c_double * 8)()
    rot, base, kind, factor, original, slow, fast = args
    assert lib().r97q_rotary_frequencies(rot, base, kind, factor, original, slow, fast, C.cast(out, C.c_void_p), None) == code
    assert lib().r97q_rotary_frequencies(8, 1e4, 0, 1, 0, 0, 0, None, None) == EINVAL


def norm(x=FAKE, res=FAKE, w=FAKE, dtype=BF16, rows=4, n=128, group=0, h=FAKE, codes=FAKE, scale=FAKE, y=None, rstd=FAKE):
    return lib().r97q_add_rmsnorm_i8g(x, res, w, dtype, rows, n, group, 1e-6, 0.0, h, codes, scale, y, rstd, None)


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), EINVAL), (dict(w=None), EINVAL), (dict(dtype=3), EINVAL), (dict(rows=-1), EINVAL), (dict(n=0), EINVAL),
    (dict(rows=1 << 31), EUNSUPPORTED), (dict(n=1 << 31), EUNSUPPORTED), (dict(codes=None), EINVAL), (dict(scale=None), EINVAL),
    (dict(h=None), EINVAL), (dict(res=None), EINVAL),
    (dict(res=None, h=None, codes=None, scale=None, rstd=None), EINVAL)])
def test_norm(kw, code):
    assert norm(**kw) == code and lib().r97q_last_error()


def test_norm_nothing_to_do():
    assert norm(rows=0) == OK


def norm_bwd(h=FAKE, w=FAKE, dtype=BF16, rows=4, n=128, group=0, rstd=FAKE, scale=FAKE, gc=FAKE, gy=None, gh=None, dx=FAKE,
             dw=FAKE, ws=FAKE, nws=1 << 40):
    return lib().r97q_add_rmsnorm_i8g_bwd(h, w, dtype, rows, n, group, 0.0, rstd, scale, gc, gy, gh, dx, dw, 0, ws, nws, None)


@pytest.mark.parametrize("kw,code", [
    (dict(h=None), EINVAL), (dict(w=None), EINVAL), (dict(dtype=2), EINVAL), (dict(rows=-1), EINVAL), (dict(n=0), EINVAL),
    (dict(rstd=None), EINVAL), (dict(dx=None), EINVAL), (dict(scale=None), EINVAL), (dict(ws=None), EWORKSPACE),
    (dict(nws=4 * 4 * 128 - 1), EWORKSPACE), (dict(n=1 << 31), EUNSUPPORTED)])
def test_norm_bwd(kw, code):
    assert norm_bwd(**kw) == code and lib().r97q_last_error()
    assert lib().r97q_add_rmsnorm_i8g_bwd_workspace_bytes(4, 128) >= 4 * 128 * 4
    assert lib().r97q_add_rmsnorm_i8g_bwd_workspace_bytes(-1, 128) == -1
    assert lib().r97q_add_rmsnorm_i8g_bwd_workspace_bytes(4, 0) == -1


def test_fronts_refuse_before_the_library():
    """The Python fronts' own checks, on CPU tensors: a message, not a launch."""
    import torch

    from r9700training_amd.attention import attention_fwd
    from r9700training_amd.norm import add_rmsnorm_i8g, add_rmsnorm_i8g_bwd
    from r9700training_amd.rotary import rotary as turn
    from r9700training_amd.rotary import rotary_frequencies

    x = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        attention_fwd(x, x, x)                                   # not on a device
    with pytest.raises(ValueError):
        attention_fwd(x, x, x[:, :2])                            # v has k's shape
    with pytest.raises(ValueError):
        attention_fwd(x[0], x[0], x[0])                          # packed without starts
    with pytest.raises(ValueError):
        attention_fwd(x[0], x, x, q_starts=torch.zeros(3, dtype=torch.int32))  # no max_q
    y = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        add_rmsnorm_i8g(y, None, y[0])
    with pytest.raises(ValueError):
        add_rmsnorm_i8g_bwd(y, y[0], torch.zeros(4))
    with pytest.raises(ValueError):
        turn(x[0], None, torch.zeros(32, dtype=torch.float64))
    with pytest.raises(ValueError):
        turn(x[0], None, torch.zeros(32), pairs="quarter")
    with pytest.raises(ValueError):
        rotary_frequencies(64, scaling="cubic", device="cpu")


def test_attention_limits_of_its_tiles():
    """Tokens so far apart that a tile passes 31 bits, workspaces off 16 bytes, and more heads than a grid holds."""
    far = dict(token_stride=(1 << 24) + 8)
    for which in ("q", "k", "v", "d_out"):
        t = heads(2 if which in "kv" else 4, **far)
        if which != "d_out":
            assert fwd(shape(), **{which: t}) == EUNSUPPORTED, which
        assert bwd(shape(), **{which: t}) == EUNSUPPORTED, which
    need = lib().r97q_attn_bwd_workspace_bytes(shape(), 4, 2)
    assert bwd(shape(), ws=FAKE + 8, nws=need + 64) == EINVAL
    long = shape(batch=1, q_len=1, kv_len=1 << 16)
    assert lib().r97q_attn_fwd_workspace_bytes(long, 4, 2) > 0
    assert fwd(long, ws=None) == EWORKSPACE and fwd(long, ws=FAKE + 4) == EINVAL
    assert lib().r97q_attn_fwd_workspace_bytes(shape(batch=65535), 256, 256) == -1


PACKED_LONG = [
    # batch, query tokens in all, q_heads, kv_heads, head_dim, kv_len: few rows and tiles of rows, cut along the keys
    (1, 1, 8, 2, 128, 32768),
    (4, 300, 8, 2, 128, 4096),
    (1, 40, 4, 4, 64, 8192),
]


@pytest.mark.parametrize("b,tokens,hq,hk,d,lk", PACKED_LONG)
def test_a_longest_length_of_nothing_still_needs_the_workspace(b, tokens, hq, hk, d, lk):
    """Packed queries whose longest length is given as 0 run like those of 1, with the same partial sums' room."""
    def packed(q_len):
        return shape(batch=b, head_dim=d, q_len=q_len, kv_len=lk, q_starts=FAKE, q_tokens=tokens)

    need = lib().r97q_attn_fwd_workspace_bytes(packed(1), hq, hk)
    assert need > 0 and lib().r97q_attn_fwd_workspace_bytes(packed(0), hq, hk) == need
    t = dict(q=heads(hq, d), k=heads(hk, d), v=heads(hk, d), out=heads(hq, d))
    for q_len in (0, 1):
        assert fwd(packed(q_len), ws=None, nws=0, **t) == EWORKSPACE
        assert fwd(packed(q_len), nws=need - 1, **t) == EWORKSPACE
    # no tokens: nothing runs
    none = shape(batch=b, head_dim=d, q_len=5, kv_len=lk, q_starts=FAKE, q_tokens=0)
    assert lib().r97q_attn_fwd_workspace_bytes(none, hq, hk) == 0 and fwd(none, ws=None, nws=0, **t) == OK


def test_fronts_refuse_a_workspace_off_the_card():
    """A workspace is an operand like the others: one in host memory, or with gaps, is refused with a message that names it.
    (The operands here are host tensors that say they are on a device: nothing gets as far as a launch.)"""
    import torch

    from r9700training_amd.attention import attention_bwd, attention_fwd
    from r9700training_amd.norm import add_rmsnorm_i8g_bwd

    class Card(torch.Tensor):
        is_cuda = True

    def card(*size, dtype=torch.bfloat16):
        return torch.zeros(size, dtype=dtype).as_subclass(Card)

    x, kv = card(1, 3, 4, 64), card(1, 50, 4, 64)
    lse = card(1, 4, 3, dtype=torch.float32)
    y, w, rs, dw = card(4, 64), card(64), card(4, dtype=torch.float32), card(64, dtype=torch.float32)
    bad = [torch.empty(1 << 20, dtype=torch.uint8), card(1 << 20, 2, dtype=torch.uint8)[:, :1]]
    for ws in bad:
        with pytest.raises(ValueError, match="workspace"):
            attention_fwd(x, kv, kv, out=x.clone(), lse=lse, workspace=ws)
        with pytest.raises(ValueError, match="workspace"):
            attention_bwd(x, kv, kv, x.clone(), lse, x.clone(), dq=x.clone(), dk=kv.clone(), dv=kv.clone(), workspace=ws)
        with pytest.raises(ValueError, match="workspace"):
            add_rmsnorm_i8g_bwd(y, w, rs, g_y=y.clone(), dx=y.clone(), dw=dw, workspace=ws)
