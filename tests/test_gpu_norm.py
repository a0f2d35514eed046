"""The residual's addition, the RMS norm and the 8-bit output, forward and adjoint, against float64: both types, odd and
wide rows, every kind of group, rows of zeros, tiny and huge values. Tolerances count f32 roundings: a sum over n
values in f32 is off by less than n roundings of its size."""
import pytest
import torch

import between_ref as R

pytestmark = pytest.mark.gpu
EPS = 1e-6


def rnd(seed, *shape, dtype=torch.bfloat16, std=1.0):
    return (std * torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")).to(dtype)


def forward(rows, n, group, dtype, residual=True, wadd=0.0, std=1.0, x=None):
    from r9700training_amd.norm import add_rmsnorm_i8g

    x = rnd(1, rows, n, dtype=dtype, std=std) if x is None else x
    r = rnd(2, rows, n, dtype=dtype, std=2 * std) if residual else None
    w = (1.0 + 0.2 * rnd(3, n, dtype=torch.float32)).to(dtype)
    codes, scale, h, y, rs = add_rmsnorm_i8g(x, r, w, group, eps=EPS, wadd=wadd, want_y=True)
    torch.cuda.synchronize()
    wh, wrs, wy = R.norm(x, r, w, EPS, wadd, dtype)
    assert torch.equal(h.double(), wh)
    rel = (n + 8) * R.U32  # the sum of squares and the few roundings after it
    assert bool(((rs.double() - wrs).abs() <= rel * wrs).all())
    y_tol = (rel + 4 * R.U32) * wy.abs()
    assert bool(((y.double() - wy).abs() <= y_tol + R.HALF[torch.bfloat16] * wy.abs()).all())
    want = R.group_scale(wy, group)
    assert bool(((scale.double() - want).abs() <= (rel + 6 * R.U32) * want).all())
    each = scale.double()[:, R.group_index(n, group, x.device)]
    # a code is the nearest to y / scale: half a step, y's error and the quotient's
    off = (codes.double() * each - wy).abs() - (0.5 * each + y_tol + 4 * R.U32 * wy.abs() + 1e-300)
    assert float(off.max()) <= 0.0, float(off.max())
    top = torch.zeros_like(scale, dtype=torch.int32)
    top.scatter_reduce_(1, R.group_index(n, group, x.device).expand(rows, n), codes.int().abs(), "amax")
    zero = R.group_scale(wy, group) == 1.0
    assert bool(((top == 127) | (zero & (top == 0)) | (want == 1.0)).all())
    return x, r, w, codes, scale, h, y, rs


SHAPES = [(1, 1, 0), (3, 7, 0), (5, 64, 0), (5, 64, 8), (4, 100, 32), (9, 128, 128), (7, 130, 128), (33, 512, 64), (65, 1000, 0),
          (17, 1024, 16), (5, 2040, 0), (21, 2048, 128), (5, 2056, 128), (3, 4096, 512), (6, 5120, 0), (6, 5120, 128),
          (2, 5120, 1024), (3, 6000, 48), (3, 8192, 128), (2, 8200, 128), (2, 12288, 0), (2, 17408, 256), (40, 256, 24),
          (3, 515, 5), (2, 5120, 5119)]


@pytest.mark.parametrize("rows,n,group", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_forward(rows, n, group, dtype):
    print(f"case norm forward {(rows, n, group, dtype)}", flush=True)
    forward(rows, n, group, dtype)
    forward(rows, n, group, dtype, residual=False, wadd=1.0)


@pytest.mark.parametrize("rows,n,group", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_backward(rows, n, group, dtype):
    from r9700training_amd.norm import add_rmsnorm_i8g_bwd

    print(f"case norm backward {(rows, n, group, dtype)}", flush=True)
    _, _, w, _, scale, h, _, rs = forward(rows, n, group, dtype, wadd=0.5)
    gc, gy, gh = rnd(4, rows, n, dtype=dtype, std=0.01), rnd(5, rows, n, dtype=dtype), rnd(6, rows, n, dtype=dtype)
    for use in ((gc, gy, gh), (gc, None, None), (None, gy, gh), (None, None, None)):
        dx, dw = add_rmsnorm_i8g_bwd(h, w, rs, group, scale=scale if use[0] is not None else None, g_codes=use[0], g_y=use[1],
                                     g_h=use[2], wadd=0.5)
        # from rstd as it is given
        wdx, wdw, e = R.norm_backward(h.double(), rs.double(), w, 0.5, scale, group, *use)
        we, x = ((w.double() + 0.5) * e).abs(), (h.double() * rs.double()[:, None]).abs()
        rel = (n + 16) * R.U32
        tol = rs.double()[:, None] * (8 * R.U32 * we + rel * x * (we * x).mean(1, keepdim=True)) + 8 * R.U32 * wdx.abs()
        tol = tol + R.HALF[dtype] * wdx.abs()
        assert bool(((dx.double() - wdx).abs() <= tol + 1e-30).all()), use
        assert bool(((dw.double() - wdw).abs() <= (rows + 8) * R.U32 * (e * x).abs().sum(0) + 1e-30).all()), use
    start = rnd(7, n, dtype=torch.float32)
    dw = start.clone()
    dx, dw = add_rmsnorm_i8g_bwd(h, w, rs, group, scale=scale, g_codes=gc, g_y=gy, g_h=gh, wadd=0.5, dw=dw, accumulate=True)
    dx2, dw2 = add_rmsnorm_i8g_bwd(h, w, rs, group, scale=scale, g_codes=gc, g_y=gy, g_h=gh, wadd=0.5)
    assert torch.equal(dw, start + dw2) and torch.equal(dx, dx2)
    dx3, none = add_rmsnorm_i8g_bwd(h, w, rs, group, scale=scale, g_codes=gc, g_y=gy, g_h=gh, wadd=0.5, want_dw=False)
    assert none is None and torch.equal(dx3, dx)
    for k in range(3):  # dx over a cotangent
        gs = [gc.clone(), gy.clone(), gh.clone()]
        dx4, _ = add_rmsnorm_i8g_bwd(h, w, rs, group, scale=scale, g_codes=gs[0], g_y=gs[1], g_h=gs[2], wadd=0.5, dx=gs[k])
        assert torch.equal(dx4, dx)


@pytest.mark.parametrize("rows", [1, 2, 511, 512, 513, 1500, 5000])
def test_many_rows(rows):
    """Row counts around the workgroups' shares, the gain's gradient summed over all of them, the same bits twice."""
    from r9700training_amd.norm import add_rmsnorm_i8g_bwd

    for n, group in ((256, 128), (4096, 0)):
        _, _, w, _, scale, h, _, rs = forward(rows, n, group, torch.bfloat16)
        gy = rnd(5, rows, n)
        dx, dw = add_rmsnorm_i8g_bwd(h, w, rs, group, g_y=gy)
        wdx, wdw, e = R.norm_backward(h.double(), rs.double(), w, 0.0, scale, group, None, gy, None)
        assert bool(((dw.double() - wdw).abs() <= (rows + 8) * R.U32 * (e * h.double() * rs.double()[:, None]).abs().sum(0)).all())
        again = add_rmsnorm_i8g_bwd(h, w, rs, group, g_y=gy)
        assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


@pytest.mark.parametrize("n,group", [(512, 128), (5120, 0), (333, 0)])
def test_zero_tiny_and_huge_rows(n, group):
    from r9700training_amd.norm import add_rmsnorm_i8g

    x = rnd(1, 6, n, dtype=torch.float32)
    x[0] = 0.0
    x[1] *= 1e-30
    x[2] *= 1e15
    x[3, :n // 2] = 0.0
    x[4] *= 1e-3
    forward(6, n, group, torch.float32, residual=False, x=x)
    # a gain of zeros: y is zero everywhere, the scales are 1
    codes, scale, h, y, rs = add_rmsnorm_i8g(x, None, torch.zeros(n, device="cuda"), group, eps=EPS, want_y=True)
    assert int(codes.abs().max()) == 0 and torch.equal(scale, torch.ones_like(scale)) and float(y.abs().max()) == 0.0
    # a tiny gain: amax / 127 is far below one, codes still span the range
    codes, scale, _, _, _ = add_rmsnorm_i8g(x, None, torch.full((n,), 1e-33, device="cuda"), group, eps=EPS)
    assert int(codes[4].abs().max()) == 127 and int(codes[2].abs().max()) == 127


def test_outputs_given_in_place_and_optional():
    from r9700training_amd.norm import add_rmsnorm_i8g

    for n, group in ((2048, 128), (5120, 0), (777, 32)):
        for dtype in (torch.bfloat16, torch.float32):
            x, r, w, codes, scale, h, y, rs = forward(19, n, group, dtype)
            for which in ("x", "r"):
                a, b = x.clone(), r.clone()
                got = add_rmsnorm_i8g(a, b, w, group, eps=EPS, want_y=True, h=a if which == "x" else b)
                for p, q in zip(got, (codes, scale, h, y, rs)):
                    assert torch.equal(p, q), which
            got = add_rmsnorm_i8g(x, r, w, group, eps=EPS, want_codes=False, want_y=True)
            assert got[0] is None and got[1] is None and torch.equal(got[3], y) and torch.equal(got[2], h)
            got = add_rmsnorm_i8g(x, r, w, group, eps=EPS)
            assert got[3] is None and torch.equal(got[0], codes)


def test_unaligned_rows():
    """Tensors off 16 bytes take the general kernels: the same values to their roundings."""
    from r9700training_amd.norm import add_rmsnorm_i8g, add_rmsnorm_i8g_bwd

    n, rows = 1024, 9
    for off in (1, 3):
        pad = rnd(1, rows * n + 8)
        x = pad[off:off + rows * n].view(rows, n)
        forward(rows, n, 128, torch.bfloat16, x=x)
        w = rnd(3, n)
        _, _, h, _, rs = add_rmsnorm_i8g(x, None, w, eps=EPS)
        gy = rnd(4, rows, n)
        dx, dw = add_rmsnorm_i8g_bwd(h, w, rs, g_y=gy)
        wdx, _, _ = R.norm_backward(x.double(), rs.double(), w, 0.0, None, 0, None, gy, None)
        assert float((dx.double() - wdx).norm() / wdx.norm()) <= 2 ** -8


def test_stream_and_graph():
    from r9700training_amd.norm import add_rmsnorm_i8g, add_rmsnorm_i8g_bwd

    x, r, w = rnd(1, 700, 1024), rnd(2, 700, 1024), rnd(3, 1024)
    gc = rnd(4, 700, 1024)

    def step(**kw):
        codes, scale, h, _, rs = add_rmsnorm_i8g(x, r, w, 128, eps=EPS, **kw)
        return (codes, scale, h, rs) + add_rmsnorm_i8g_bwd(h, w, rs, 128, scale=scale, g_codes=gc, **kw)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(stream=side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        x.copy_(rnd(10 + i, 700, 1024))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held)), i


def test_no_rows():
    from r9700training_amd.norm import add_rmsnorm_i8g, add_rmsnorm_i8g_bwd

    x, w = rnd(1, 0, 256), rnd(2, 256)
    codes, scale, h, y, rs = add_rmsnorm_i8g(x, None, w, 128)
    assert codes.shape == (0, 256) and scale.shape == (0, 2)
    dx, dw = add_rmsnorm_i8g_bwd(x, w, rs, 128, g_y=x)
    assert dx.shape == (0, 256) and float(dw.abs().max()) == 0.0


@pytest.mark.parametrize("rows,n,group", [(3, 100, 1), (4, 65, 64), (5, 200, 96), (2, 8191, 100), (3, 8192, 65), (2, 8193, 128), (6, 2049, 63),
                                          (7, 1, 0), (3, 513, 512), (2, 5119, 2), (300, 1001, 128), (2, 4100, 4096)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_column_at_a_time(rows, n, group, dtype):
    """Widths and groups off the 16-byte pieces: groups of one column, of just over a wave's, that end inside one."""
    from r9700training_amd.norm import add_rmsnorm_i8g_bwd

    print(f"case norm columns {(rows, n, group, dtype)}", flush=True)
    forward(rows, n, group, dtype, residual=False, wadd=1.0)
    _, _, w, _, scale, h, _, rs = forward(rows, n, group, dtype)
    gc, gh = rnd(4, rows, n, dtype=dtype, std=0.01), rnd(6, rows, n, dtype=dtype)
    dx, dw = add_rmsnorm_i8g_bwd(h, w, rs, group, scale=scale, g_codes=gc, g_h=gh)
    wdx, wdw, e = R.norm_backward(h.double(), rs.double(), w, 0.0, scale, group, gc, None, gh)
    we, x = (w.double() * e).abs(), (h.double() * rs.double()[:, None]).abs()
    tol = rs.double()[:, None] * (8 * R.U32 * we + (n + 16) * R.U32 * x * (we * x).mean(1, keepdim=True)) + 8 * R.U32 * wdx.abs()
    assert bool(((dx.double() - wdx).abs() <= tol + R.HALF[dtype] * wdx.abs() + 1e-30).all())
    assert bool(((dw.double() - wdw).abs() <= (rows + 8) * R.U32 * (e * x).abs().sum(0) + 1e-30).all())
    again = add_rmsnorm_i8g_bwd(h, w, rs, group, scale=scale, g_codes=gc, g_h=gh)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


def placed(t, by, guard):
    """t's values `by` values into a buffer that is otherwise full of `guard`."""
    whole = torch.full((t.numel() + 32,), guard, dtype=t.dtype, device="cuda")
    view = whole[by:by + t.numel()].view(t.shape)
    view.copy_(t)
    return whole, view


@pytest.mark.parametrize("rows,n,group", [(9, 1, 0), (6, 9, 0), (5, 18, 8), (7, 515, 128), (3, 1028, 64), (5, 1533, 0), (4, 2046, 512), (3, 2049, 128),
                                          (2, 7007, 40), (3, 5127, 0), (2, 16383, 128), (3, 2048, 96), (2, 16384, 1000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("by", [0, 1, 5])
def test_rows_that_begin_anywhere(rows, n, group, dtype, by):
    """Last pieces of one to eight columns, tensors off 16 bytes: the same results as from aligned ones, nothing beside them."""
    from r9700training_amd.norm import add_rmsnorm_i8g, add_rmsnorm_i8g_bwd

    print(f"case norm anywhere {(rows, n, group, dtype, by)}", flush=True)
    x, r, w, codes, scale, h, y, rs = forward(rows, n, group, dtype)
    gc, gy, gh = (rnd(4 + i, rows, n, dtype=dtype) for i in range(3))
    args = [placed(v, by, float("nan"))[1] for v in (x, r, w, gc, gy, gh)]
    outs = [placed(torch.zeros_like(v), by, 77) for v in (codes, h)]
    got = add_rmsnorm_i8g(args[0], args[1], args[2], group, eps=EPS, codes=outs[0][1], h=outs[1][1], want_y=True)
    for a, b in zip(got, (codes, scale, h, y, rs)):
        assert torch.equal(a, b)
    dx, dw = add_rmsnorm_i8g_bwd(h, w, rs, group, scale=scale, g_codes=gc, g_y=gy, g_h=gh)
    wdx, wdw, e = R.norm_backward(h.double(), rs.double(), w, 0.0, scale, group, gc, gy, gh)
    size = (gc.double().abs() / scale.double()[:, R.group_index(n, group, x.device)]) + gy.double().abs()
    we, hx = w.double().abs() * size, (h.double() * rs.double()[:, None]).abs()
    tol = rs.double()[:, None] * (8 * R.U32 * we + (n + 16) * R.U32 * hx * (we * hx).mean(1, keepdim=True)) + 8 * R.U32 * (wdx.abs() + gh.double().abs())
    assert bool(((dx.double() - wdx).abs() <= tol + R.HALF[dtype] * wdx.abs() + 1e-30).all())
    assert bool(((dw.double() - wdw).abs() <= (rows + 8) * R.U32 * (size * hx).sum(0) + 1e-30).all())
    whole, into = placed(torch.zeros_like(dx), by, 77)
    got = add_rmsnorm_i8g_bwd(placed(h, by, 77)[1], args[2], rs, group, scale=scale, g_codes=args[3], g_y=args[4], g_h=args[5], dx=into)
    assert torch.equal(into, dx) and torch.equal(got[1], dw)
    torch.cuda.synchronize()
    for one, part in outs + [(whole, into)]:
        assert bool((one[:by] == 77).all()) and bool((one[by + part.numel():] == 77).all())


@pytest.mark.parametrize("n", [512, 2056])
def test_workspace_off_16_bytes(n):
    from r9700training_amd.norm import add_rmsnorm_i8g_bwd

    h, gy = rnd(1, 700, n), rnd(2, 700, n)
    w, rs = rnd(3, n), 1.0 + rnd(4, 700, dtype=torch.float32).abs()
    dx, dw = add_rmsnorm_i8g_bwd(h, w, rs, g_y=gy)
    space = torch.empty(4 * 512 * n + 16, dtype=torch.uint8, device="cuda")
    for by in (4, 8):
        got = add_rmsnorm_i8g_bwd(h, w, rs, g_y=gy, workspace=space[by:])
        assert torch.equal(got[0], dx) and torch.equal(got[1], dw)


@pytest.mark.parametrize("rows,n,group", [(67_200_003, 8, 0), (16_800_005, 3, 1), (67_300_001, 2, 0)])
def test_more_rows_than_a_launch_takes(rows, n, group):
    """Rows on both sides of a launch's end have the bits they have in a call of their own, forward and back."""
    from r9700training_amd.norm import add_rmsnorm_i8g, add_rmsnorm_i8g_bwd

    print(f"case norm rows {(rows, n, group)}", flush=True)
    x, r, w, gy = rnd(1, rows, n), rnd(2, rows, n), rnd(3, n), rnd(4, rows, n)
    codes, scale, h, y, rs = add_rmsnorm_i8g(x, r, w, group, eps=EPS, want_y=True)
    dx, _ = add_rmsnorm_i8g_bwd(h, w, rs, group, g_y=gy, want_dw=False)
    ends = (0, 16_777_200, 16_777_216, 67_108_800, 67_108_860, rows - 40)
    for at in (i for i in ends if i + 40 <= rows):
        part = slice(at, at + 40)
        want = add_rmsnorm_i8g(x[part].contiguous(), r[part].contiguous(), w, group, eps=EPS, want_y=True)
        for a, b in zip((codes[part], scale[part], h[part], y[part], rs[part]), want):
            assert torch.equal(a, b), at
        back, _ = add_rmsnorm_i8g_bwd(h[part].contiguous(), w, rs[part].contiguous(), group, g_y=gy[part].contiguous(), want_dw=False)
        assert torch.equal(dx[part], back), at


ENDS = [(64, 0), (512, 128), (2048, 0), (5120, 0), (777, 32), (515, 5), (17408, 256), (17408, 0), (3, 1), (1, 0)]


@pytest.mark.parametrize("n,group", ENDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_squares_past_f32(n, group, dtype):
    """Finite rows whose sum of squares is none in f32: 1 / rms, codes and scales are those of any other row."""
    print(f"case norm range {(n, group, dtype)}", flush=True)
    size = torch.tensor([1.0, 1e17, 2e18, 1e19, 3e25, 1e33, 1e37], device="cuda")
    x = rnd(1, 7, n, dtype=torch.float32) * size[:, None]
    x[6, ::3] = 3e38
    forward(7, n, group, dtype, residual=False, x=x.to(dtype))


@pytest.mark.parametrize("n,group", ENDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_squares_below_f32(n, group, dtype):
    """With an eps of 0, or far below the rows' squares, tiny rows are normed like any other."""
    from r9700training_amd.norm import add_rmsnorm_i8g

    print(f"case norm small {(n, group, dtype)}", flush=True)
    size = torch.tensor([1.0, 1e-14, 1e-17, 1e-22, 1e-27, 1e-33, 1e-36], device="cuda")
    x = rnd(1, 7, n, dtype=torch.float32)
    x = ((x.abs() + 0.5) * x.sign() * size[:, None]).to(dtype)
    w = (1.0 + 0.2 * rnd(3, n, dtype=torch.float32)).to(dtype)
    for eps in (0.0, 1e-33):
        codes, scale, _, y, rs = add_rmsnorm_i8g(x, None, w, group, eps=eps, want_y=True)
        _, wrs, wy = R.norm(x, None, w, float(torch.tensor(eps)), 0.0, dtype)
        rel = (n + 8) * R.U32
        assert bool(((rs.double() - wrs).abs() <= rel * wrs).all()), eps
        y_tol = (rel + 4 * R.U32) * wy.abs()
        assert bool(((y.double() - wy).abs() <= y_tol + R.HALF[torch.bfloat16] * wy.abs()).all()), eps
        each = scale.double()[:, R.group_index(n, group, x.device)]
        assert bool(((codes.double() * each - wy).abs() <= 0.5 * each + y_tol + 8 * R.U32 * wy.abs() + 1e-300).all()), eps


@pytest.mark.parametrize("n,group", [(64, 0), (512, 128), (2048, 64), (5120, 0), (5120, 128), (5120, 1024), (777, 32), (2048, 96), (515, 5), (515, 70), (17408, 256),
                                     (17408, 0), (7, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nan_and_infinity_are_kept(n, group, dtype):
    """A group with a NaN or an infinity in y has it in its scale, so that what reads the codes has it too; other groups and
    rows are as they were."""
    from r9700training_amd.norm import add_rmsnorm_i8g

    print(f"case norm nan {(n, group, dtype)}", flush=True)
    inf, nan, c = float("inf"), float("nan"), n // 2
    x, r, w = rnd(1, 6, n, dtype=dtype), rnd(2, 6, n, dtype=dtype), rnd(3, n, dtype=dtype)
    clean = add_rmsnorm_i8g(x, r, w, group, eps=EPS, want_y=True)
    idx = R.group_index(n, group, x.device)
    other = torch.arange(int(idx[-1]) + 1, device="cuda") != idx[c]
    a, b = x.clone(), r.clone()
    a[1, c], b[2, c], a[3, c], a[4, c] = nan, nan, inf, -inf
    codes, scale, h, y, rs = add_rmsnorm_i8g(a, b, w, group, eps=EPS, want_y=True)
    for i in (0, 5):
        for got, was in zip((codes, scale, h, y, rs), clean):
            assert torch.equal(got[i], was[i])
    for i in (1, 2):  # nothing of the row is a number
        assert bool(rs[i].isnan()) and bool(y[i].isnan().all()) and bool(scale[i].isnan().all())
    for i in (3, 4):  # 1 / rms is zero: zeros, and a NaN where the infinity is
        assert float(rs[i]) == 0.0 and bool(y[i, c].isnan()) and int(y[i].isnan().sum()) == 1
        assert bool(scale[i, idx[c]].isnan()) and bool((scale[i][other] == 1.0).all()) and bool((codes[i, idx != idx[c]] == 0).all())
    for bad in (nan, inf):
        v = w.clone()
        v[c] = bad
        codes, scale, h, y, rs = add_rmsnorm_i8g(x, r, v, group, eps=EPS, want_y=True)
        at = scale[:, idx[c]]
        assert bool(at.isnan().all() if bad != bad else (at == inf).all())
        assert torch.equal(scale[:, other], clean[1][:, other]) and torch.equal(codes[:, idx != idx[c]], clean[0][:, idx != idx[c]])


def test_a_nan_reaches_the_projection():
    """The codes' product has the NaN of its activation's row, and only that row."""
    from r9700training_amd.norm import add_rmsnorm_i8g
    from r9700training_amd.qlinear import gemm_nt_q_fwd

    x, w = rnd(1, 70, 512), rnd(2, 512)
    b = torch.randint(-127, 128, (256, 512), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda", dtype=torch.int8)
    bs = torch.full((256, 4), 0.01, device="cuda").to(torch.bfloat16).view(torch.int16)
    was = gemm_nt_q_fwd(b, bs, *add_rmsnorm_i8g(x, None, w, 128)[:2], y_dtype=torch.float32)
    x[33, 5] = float("nan")
    got = gemm_nt_q_fwd(b, bs, *add_rmsnorm_i8g(x, None, w, 128)[:2], y_dtype=torch.float32)
    keep = torch.arange(70, device="cuda") != 33
    assert bool(got[33].isnan().all()) and torch.equal(got[keep], was[keep])


@pytest.mark.parametrize("rows,n,group", [(3, 17408, 256), (3, 17408, 0), (2, 9001, 100), (5, 16386, 0), (4, 77, 1), (2, 20000, 20000 - 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("by", [0, 1, 3])
def test_general_kernels_anywhere_and_in_place(rows, n, group, dtype, by):
    """Rows past the registers, groups of one column: the kernels that read a row again for each stage, with tensors off 16
    bytes and h over x or the residual."""
    from r9700training_amd.norm import add_rmsnorm_i8g, add_rmsnorm_i8g_bwd

    print(f"case norm general {(rows, n, group, dtype, by)}", flush=True)
    x, r, w, codes, scale, h, y, rs = forward(rows, n, group, dtype)
    for which in (0, 1):
        (wx, px), (wr, pr) = placed(x, by, 77), placed(r, by, 77)
        wc, pc = placed(torch.zeros_like(codes), by, 77)
        got = add_rmsnorm_i8g(px, pr, placed(w, by, 77)[1], group, eps=EPS, want_y=True, codes=pc, h=(px, pr)[which])
        for a, b in zip(got, (codes, scale, h, y, rs)):
            assert torch.equal(a, b), which
        torch.cuda.synchronize()
        for one in (wx, wr, wc):
            assert bool((one[:by] == 77).all()) and bool((one[by + x.numel():] == 77).all())
    gc, gy, gh = (rnd(4 + i, rows, n, dtype=dtype, std=0.05) for i in range(3))
    dx, dw = add_rmsnorm_i8g_bwd(h, w, rs, group, scale=scale, g_codes=gc, g_y=gy, g_h=gh)
    wdx, wdw, e = R.norm_backward(h.double(), rs.double(), w, 0.0, scale, group, gc, gy, gh)
    size = gc.double().abs() / scale.double()[:, R.group_index(n, group, x.device)] + gy.double().abs()
    we, hx = w.double().abs() * size, (h.double() * rs.double()[:, None]).abs()
    tol = rs.double()[:, None] * (8 * R.U32 * we + (n + 16) * R.U32 * hx * (we * hx).mean(1, keepdim=True)) + 8 * R.U32 * (wdx.abs() + gh.double().abs())
    assert bool(((dx.double() - wdx).abs() <= tol + R.HALF[dtype] * wdx.abs() + 1e-30).all())
    assert bool(((dw.double() - wdw).abs() <= (rows + 8) * R.U32 * (size * hx).sum(0) + 1e-30).all())
    for k in range(3):  # dx over a cotangent
        parts = [placed(t, by, 77) for t in (gc, gy, gh)]
        got = add_rmsnorm_i8g_bwd(placed(h, by, 77)[1], w, rs, group, scale=scale, g_codes=parts[0][1], g_y=parts[1][1], g_h=parts[2][1], dx=parts[k][1])
        assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
        assert all(bool((one[:by] == 77).all()) and bool((one[by + x.numel():] == 77).all()) for one, _ in parts)


@pytest.mark.parametrize("rows,n,group", [(1100, 40, 1), (513, 17408, 256)])
def test_general_kernels_many_rows(rows, n, group):
    """More rows than the gain's partial sums: a workgroup adds its second row to its first, in the same order each time."""
    from r9700training_amd.norm import add_rmsnorm_i8g_bwd

    print(f"case norm general rows {(rows, n, group)}", flush=True)
    _, _, w, _, scale, h, _, rs = forward(rows, n, group, torch.bfloat16)
    gy = rnd(5, rows, n)
    dx, dw = add_rmsnorm_i8g_bwd(h, w, rs, group, g_y=gy)
    wdx, wdw, e = R.norm_backward(h.double(), rs.double(), w, 0.0, scale, group, None, gy, None)
    hx = (h.double() * rs.double()[:, None]).abs()
    assert bool(((dw.double() - wdw).abs() <= (rows + 8) * R.U32 * (e.abs() * hx).sum(0)).all())
    we = (w.double() * e).abs()
    tol = rs.double()[:, None] * (8 * R.U32 * we + (n + 16) * R.U32 * hx * (we * hx).mean(1, keepdim=True)) + 8 * R.U32 * wdx.abs()
    assert bool(((dx.double() - wdx).abs() <= tol + R.HALF[torch.bfloat16] * wdx.abs() + 1e-30).all())
    again = add_rmsnorm_i8g_bwd(h, w, rs, group, g_y=gy)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])
