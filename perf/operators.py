"""The operators between a layer's projections: rotary positions, attention forward and backward, and the
RMS norm with the residual's addition and an 8-bit output.

    listed()            the cases that stand for the ranges
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program holds before the call, on the card
    run(state)          one pass: the plain form where `own` is false, the package's kernels where it is true
    work(case)          the bytes and operations the pass cannot do without
    exact(case, seed)   the same outputs in float64, from the operators' definitions

Widths are those of the benchmark workloads and of the published real-model projections (1024-, 2048-,
4096-, 5120- and 6144-wide activations as heads of 64, 128 and 256), 2048-token sequences eight at a time,
and the odd and ragged lengths between them.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SCORES = 8 * 32 * 2048 * 2048                  # the most scores that a listed case has
PRODUCTS = 10 * 8 * 16 * 2048 * 2049 // 2 * 256  # the largest listed case's operations


def listed():
    return [
        # a serving loop's step: one token's 24 query and 4 key heads of 256 turned in a quarter of the head,
        # far into a long context
        dict(name="rotary_token", op="rotary", tokens=1, q_heads=24, kv_heads=4, dim=256, rot=64, pairs="half",
             dtype="bf16", start=100000, scaling="linear", inverse=False),
        # the backward of a training batch's rotation: neighbouring pairs, frequencies ramped for a long context
        dict(name="rotary_back", op="rotary", tokens=16384, q_heads=32, kv_heads=8, dim=128, rot=128,
             pairs="interleaved", dtype="bf16", start=0, scaling="ramp", inverse=True),
        # the norm before the coded projections of one token, one scale a token
        dict(name="norm_token", op="norm", rows=1, n=5120, group=0, dtype="bf16", back=False, residual=True, y=True),
        # the norm before the coded projections of a training batch, a scale every 128 columns
        dict(name="norm_step", op="norm", rows=16384, n=2048, group=128, dtype="bf16", back=False, residual=True,
             y=False),
        # its backward at the real model's width, with the gain's gradient
        dict(name="norm_back", op="norm", rows=4096, n=5120, group=128, dtype="f32", back=True, residual=True, y=False),
        # one new token against a long cache: 24 query heads share 4 key heads
        dict(name="attn_token", op="attn", form="dense", batch=1, q_len=1, kv_len=32768, q_heads=24, kv_heads=4,
             dim=256, causal=True, window=0, back=False),
        # a serving batch: 16 sequences of different lengths in one cache, one new token each
        dict(name="attn_batch", op="attn", form="cache", batch=16, q_len=1, kv_len=4096, q_heads=32, kv_heads=8,
             dim=128, causal=True, window=0, back=False),
        # sequences of odd lengths packed into one batch, sliding window, a head for every query head
        dict(name="attn_packed", op="attn", form="packed", batch=7, q_len=1500, kv_len=1500, q_heads=8, kv_heads=8,
             dim=64, causal=True, window=500, back=False),
        # the forward of a training batch
        dict(name="attn_step", op="attn", form="dense", batch=8, q_len=2048, kv_len=2048, q_heads=32, kv_heads=8,
             dim=128, causal=True, window=0, back=False),
        # the smallest training step: 128 tokens of a 1024-wide layer
        dict(name="attn_small_back", op="attn", form="dense", batch=1, q_len=128, kv_len=128, q_heads=16, kv_heads=4,
             dim=64, causal=True, window=0, back=True),
        # the backward of packed odd lengths
        dict(name="attn_packed_back", op="attn", form="packed", batch=5, q_len=1300, kv_len=1300, q_heads=16,
             kv_heads=4, dim=128, causal=True, window=0, back=True),
        # the backward of a training batch with the real model's heads of 256
        dict(name="attn_step_back", op="attn", form="dense", batch=8, q_len=2048, kv_len=2048, q_heads=16, kv_heads=4,
             dim=256, causal=True, window=0, back=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * math.exp(rng.random() * math.log(hi / lo)))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "norm", "attn", "attn", "attn", "attn_back", "attn_back"])
    if op == "rotary":
        dim = rng.choice([64, 96, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        q_heads = kv_heads * rng.choice([1, 2, 4, 6])
        most = max(2, 16384 * 40 * 128 // (dim * (q_heads + kv_heads)) // 2)
        return dict(op="rotary", tokens=_log(rng, 1, min(16384, most)), q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                    rot=rng.choice([dim, dim // 2, dim // 4]), pairs=rng.choice(["half", "interleaved"]),
                    dtype=rng.choice(["bf16", "f32"]), start=rng.choice([0, rng.randrange(1, 200000)]),
                    scaling=rng.choice(["none", "linear", "ramp"]), inverse=rng.random() < 0.5)
    if op == "norm":
        n = _log(rng, 64, 8192) if rng.random() < 0.3 else 128 * _log(rng, 4, 64)
        back = rng.random() < 0.5
        return dict(op="norm", rows=_log(rng, 1, min(16384, 16384 * 2048 // n // 2)), n=n,
                    group=rng.choice([0, 0, 64, 128, 128]), dtype=rng.choice(["bf16", "bf16", "f32"]), back=back,
                    residual=rng.random() < 0.8, y=not back and rng.random() < 0.5)
    back = op == "attn_back"
    dim = rng.choice([64, 64, 80, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 4, 6])
    form = rng.choice(["dense", "packed"] if back else ["token", "dense", "cache", "packed"])
    causal = rng.random() < 0.8
    window = rng.choice([0, 0, _log(rng, 16, 1024)]) if causal else 0
    while True:
        if form in ("token", "cache"):
            batch, q_len, kv_len = _log(rng, 1, 32), rng.choice([1, 1, 1, 2, 5]), _log(rng, 1, 32768)
        elif form == "dense":
            batch, q_len = _log(rng, 1, 8), _log(rng, 16, 4096)
            kv_len = rng.choice([q_len, q_len, q_len, _log(rng, 1, 4096)])
        else:
            batch, q_len = _log(rng, 1, 12), _log(rng, 16, 2500)
            kv_len = q_len
        across = batch * batch if form == "packed" else batch  # the plain form has every sequence against every other
        pairs = across * q_heads * q_len * kv_len
        if pairs <= SCORES // 2 and (10 if back else 4) * pairs * dim <= PRODUCTS \
                and batch * kv_len * kv_heads * dim <= 32768 * 4 * 256 * 2:
            return dict(op="attn", form="dense" if form == "token" else form, batch=batch, q_len=q_len, kv_len=kv_len,
                        q_heads=q_heads, kv_heads=kv_heads, dim=dim, causal=causal, window=window, back=back)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, shape, dtype, std=1.0):
    return (std * torch.randn(shape, generator=g, device=DEV)).to(dtype)


def _lengths(c, seed):
    """The packed form's lengths and the cache form's lengths in use, from one token to the longest: the same
    ones for every seed, in another order."""
    longest = c["q_len"] if c["form"] == "packed" else c["kv_len"]
    g = torch.Generator().manual_seed(1000 * c["batch"] + longest)
    n = 1 + (torch.rand(c["batch"], generator=g) * (longest - 1)).round().long()
    n[0] = longest
    return n[torch.randperm(c["batch"], generator=torch.Generator().manual_seed(int(seed)))]


def _frequencies(c):
    """(f64 inverse frequencies [rot / 2], the factor on the rotated values) as a program makes them once: base
    10000, all stretched 4 times ("linear"), or stretched 8 times where a turn is long and not where it is
    short, with a ramp between ("ramp")."""
    half = c["rot"] // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    if c["scaling"] == "linear":
        return f / 4.0, 1.0
    if c["scaling"] == "ramp":
        turns = 4096.0 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return f * keep + f / 8.0 * (1.0 - keep), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def prepare(c, seed):
    g = _gen(seed)
    s = dict(c)
    if c["op"] == "rotary":
        dt = DTYPES[c["dtype"]]
        f, m = _frequencies(c)
        s.update(q=_randn(g, (c["tokens"], c["q_heads"], c["dim"]), dt), k=_randn(g, (c["tokens"], c["kv_heads"], c["dim"]), dt),
                 inv_freq=f.to(DEV), mscale=m,
                 positions=torch.arange(c["start"], c["start"] + c["tokens"], dtype=torch.int32, device=DEV))
        s.update(q_out=torch.empty_like(s["q"]), k_out=torch.empty_like(s["k"]))
        return s
    if c["op"] == "norm":
        dt = DTYPES[c["dtype"]]
        rows, n = c["rows"], c["n"]
        width = n if c["group"] <= 0 or c["group"] > n else c["group"]
        # a residual stream: a few columns much larger than the rest
        big = torch.where(torch.rand(n, generator=g, device=DEV) < 0.01, 20.0, 1.0)
        s.update(x=_randn(g, (rows, n), dt), weight=(1.0 + 0.1 * torch.randn(n, generator=g, device=DEV)).to(dt),
                 residual=(2.0 * big * torch.randn((rows, n), generator=g, device=DEV)).to(dt) if c["residual"] else None,
                 width=width)
        if c["back"]:
            h = s["x"].float() + (s["residual"].float() if c["residual"] else 0.0)
            s["h"] = h.to(dt)
            rs, y = _norm(s["h"], s["weight"])
            s["rstd"] = rs
            s["scale"] = _quantise(y, width)[1]
            s.update(g_codes=_randn(g, (rows, n), dt, 0.01), g_y=_randn(g, (rows, n), dt), g_h=_randn(g, (rows, n), dt))
        else:
            s.update(h_out=torch.empty((rows, n), dtype=dt, device=DEV) if c["residual"] else None,
                     y_out=torch.empty((rows, n), dtype=torch.bfloat16, device=DEV) if c["y"] else None,
                     values=torch.empty((rows, n), dtype=torch.bfloat16, device=DEV),
                     codes=torch.empty((rows, n), dtype=torch.int8, device=DEV),
                     scale_out=torch.empty((rows, (n + width - 1) // width), dtype=torch.float32, device=DEV),
                     rstd_out=torch.empty(rows, dtype=torch.float32, device=DEV))
        return s
    b, lq, lk, hq, hk, d = (c[x] for x in ("batch", "q_len", "kv_len", "q_heads", "kv_heads", "dim"))
    s["sm_scale"] = 1.0 / math.sqrt(d)
    if c["form"] == "packed":
        n = _lengths(c, seed)
        s["starts"] = torch.cat([torch.zeros(1, dtype=torch.long), n.cumsum(0)]).to(torch.int32).to(DEV)
        t = int(n.sum())
        qs, ks = (t, hq, d), (t, hk, d)
    else:
        qs, ks = (b, lq, hq, d), (b, lk, hk, d)
        if c["form"] == "cache":
            s["lengths"] = _lengths(c, seed).to(torch.int32).to(DEV)
    s.update(q=_randn(g, qs, torch.bfloat16), k=_randn(g, ks, torch.bfloat16), v=_randn(g, ks, torch.bfloat16))
    lse = (hq, qs[0]) if c["form"] == "packed" else (b, hq, lq)
    if c["back"]:
        out, s["lse"] = _attention(s)
        s["out"] = out.to(torch.bfloat16)
        s["d_out"] = _randn(g, qs, torch.bfloat16)
    else:
        s.update(out=torch.empty(qs, dtype=torch.bfloat16, device=DEV), lse=torch.empty(lse, dtype=torch.float32, device=DEV))
    return s


# ------------------------------------------------------------------ the plain forms
def _rotary(x, s):
    """f32 [tokens, heads, dim]; the angles in f64, since a far position times a frequency loses its turn in f32."""
    half = s["rot"] // 2
    a = s["positions"].double()[:, None] * s["inv_freq"]
    a = -a if s["inverse"] else a
    cos, sin = (torch.cos(a) * s["mscale"]).float()[:, None, :], (torch.sin(a) * s["mscale"]).float()[:, None, :]
    x = x.float()
    r, rest = x[..., :2 * half], x[..., 2 * half:]
    if s["pairs"] == "half":
        u, v = r[..., :half], r[..., half:]
        r = torch.cat([u * cos - v * sin, u * sin + v * cos], -1)
    else:
        u, v = r[..., 0::2], r[..., 1::2]
        r = torch.stack([u * cos - v * sin, u * sin + v * cos], -1).flatten(-2)
    return torch.cat([r, rest], -1)


def _norm(h, weight):
    """(1 / rms f32 [rows], y f64): in f64, since a code next to a border goes by the last bits."""
    h = h.double()
    rs = 1.0 / torch.sqrt((h * h).mean(1) + EPS)
    return rs.float(), h * rs[:, None] * weight.double()


def _groups(y, width):
    pad = -y.shape[1] % width
    return torch.nn.functional.pad(y, (0, pad)).view(y.shape[0], -1, width)


def _quantise(y, width):
    """(the codes' values, f32 scales [rows, groups]) of y f64."""
    g = _groups(y, width)
    amax = g.abs().amax(-1)
    scale = torch.where(amax > 0, amax / 127.0, torch.ones_like(amax)).float()
    codes = torch.round(g / scale.double()[..., None]).clamp(-127, 127)
    return (codes * scale.double()[..., None]).flatten(1)[:, :y.shape[1]], scale


def _visible(s):
    """True where a query may look at a key: [tokens, tokens] for packed sequences, else [batch or 1, 1, q_len, kv_len]."""
    if s["form"] == "packed":
        t = s["q"].shape[0]
        at = torch.arange(t, device=DEV)
        seq = torch.bucketize(at, s["starts"][1:].long(), right=True)
        see = seq[:, None] == seq[None, :]
        far = at[:, None] - at[None, :]
    else:
        lq, lk = s["q"].shape[1], s["k"].shape[1]
        j = torch.arange(lk, device=DEV)
        n = s["lengths"].long()[:, None, None, None] if s["form"] == "cache" else torch.full((1, 1, 1, 1), lk, device=DEV)
        see = j < n
        far = torch.arange(lq, device=DEV)[:, None] + (n - lq) - j
    if s["causal"]:
        see = see & (far >= 0)
    if s["window"]:
        see = see & (far < s["window"])
    return see


def _heads(x, s, repeat=1):
    """f32 [batch, heads, tokens, dim] (packed: one batch), each key head once for every query head that shares it."""
    x = x.float()
    x = x[None] if s["form"] == "packed" else x
    return x.transpose(1, 2).repeat_interleave(repeat, 1)


def _tokens(x, s):
    x = x.transpose(1, 2)
    return x[0] if s["form"] == "packed" else x


def _scores(s):
    r = s["q_heads"] // s["kv_heads"]
    return (_heads(s["q"], s) @ _heads(s["k"], s, r).transpose(2, 3).contiguous() * s["sm_scale"]).masked_fill_(~_visible(s), -math.inf)


def _attention(s):
    """(out f32, log-sum-exp f32); a query that sees nothing gives zeros and minus infinity."""
    x = _scores(s)
    m = x.amax(-1, keepdim=True) if x.shape[-1] else x.new_full(x.shape[:-1] + (1,), -math.inf)
    p = torch.exp(x.sub_(torch.where(m == -math.inf, 0.0, m)))
    total = p.sum(-1, keepdim=True)
    o = (p @ _heads(s["v"], s, s["q_heads"] // s["kv_heads"])) / torch.where(total > 0, total, 1.0)
    lse = (m + torch.log(total))[..., 0]
    return _tokens(o, s), lse[0] if s["form"] == "packed" else lse


def _attention_back(s):
    """f32 (dq, dk, dv): the probabilities again from the scores and the log-sum-exp."""
    r = s["q_heads"] // s["kv_heads"]
    lse = s["lse"][None] if s["form"] == "packed" else s["lse"]
    p = torch.exp(_scores(s).sub_(torch.where(lse == -math.inf, 0.0, lse)[..., None]))
    do = _heads(s["d_out"], s)
    delta = (do * _heads(s["out"], s)).sum(-1, keepdim=True)
    dv = p.transpose(2, 3).contiguous() @ do
    ds = (do @ _heads(s["v"], s, r).transpose(2, 3).contiguous()).sub_(delta).mul_(p)
    dq = ds @ _heads(s["k"], s, r) * s["sm_scale"]
    dk = ds.transpose(2, 3).contiguous() @ _heads(s["q"], s) * s["sm_scale"]
    shared = lambda x: x.unflatten(1, (s["kv_heads"], r)).sum(2)  # noqa: E731
    return _tokens(dq, s), _tokens(shared(dk), s), _tokens(shared(dv), s)


# ------------------------------------------------------------------ one pass
def run(s):
    if s["op"] == "rotary":
        if own:
            from r9700training_amd.rotary import rotary

            return rotary(s["q"], s["k"], s["inv_freq"], s["positions"], pairs=s["pairs"], mscale=s["mscale"],
                          inverse=s["inverse"], q_out=s["q_out"], k_out=s["k_out"])
        return _rotary(s["q"], s).to(s["q"].dtype), _rotary(s["k"], s).to(s["k"].dtype)
    if s["op"] == "norm":
        return _run_norm_back(s) if s["back"] else _run_norm(s)
    if own:
        from r9700training_amd.attention import attention_bwd, attention_fwd

        kw = dict(causal=s["causal"], window=s["window"], scale=s["sm_scale"])
        if s["form"] == "packed":
            kw.update(q_starts=s["starts"], kv_starts=s["starts"], max_q=s["q_len"], max_kv=s["kv_len"])
        if s["form"] == "cache":
            kw.update(kv_lens=s["lengths"])
        if s["back"]:
            return attention_bwd(s["q"], s["k"], s["v"], s["out"], s["lse"], s["d_out"], **kw)
        return attention_fwd(s["q"], s["k"], s["v"], out=s["out"], lse=s["lse"], **kw)
    if s["back"]:
        return tuple(x.to(torch.bfloat16) for x in _attention_back(s))
    out, lse = _attention(s)
    return out.to(torch.bfloat16), lse


def _run_norm(s):
    """(h, the codes' values bf16, scales, 1 / rms, and y bf16 where it is asked for)"""
    if own:
        from r9700training_amd.norm import add_rmsnorm_i8g

        codes, scale, h, y, rs = add_rmsnorm_i8g(s["x"], s["residual"], s["weight"], s["group"], eps=EPS, codes=s["codes"],
                                                 scale=s["scale_out"], h=s["h_out"], y=s["y_out"], rstd=s["rstd_out"],
                                                 want_y=s["y"])
        return (h, _values(codes, scale, s), scale, rs) + ((y,) if s["y"] else ())
    h = s["x"].float() + s["residual"].float() if s["residual"] is not None else s["x"].float()
    h = h.to(s["x"].dtype)  # the stream's own type: the norm is of what the next layer reads
    rs, y = _norm(h, s["weight"])
    values, scale = _quantise(y, s["width"])
    return (h, values.to(torch.bfloat16), scale, rs) + ((y.to(torch.bfloat16),) if s["y"] else ())


def _values(codes, scale, s):
    """What the codes stand for, bf16."""
    rows, n, width = s["rows"], s["n"], s["width"]
    if n % width:
        return (_groups(codes, width) * scale[..., None]).flatten(1)[:, :n].to(torch.bfloat16)
    torch.mul(codes.view(rows, -1, width), scale[..., None], out=s["values"].view(rows, -1, width))
    return s["values"]


def _run_norm_back(s):
    """(dx in the stream's type, dw f32)"""
    if own:
        from r9700training_amd.norm import add_rmsnorm_i8g_bwd

        return add_rmsnorm_i8g_bwd(s["h"], s["weight"], s["rstd"], s["group"], scale=s["scale"], g_codes=s["g_codes"],
                                   g_y=s["g_y"], g_h=s["g_h"])
    h, rs = s["h"].float(), s["rstd"][:, None]
    e = (_groups(s["g_codes"].float(), s["width"]) / s["scale"][..., None]).flatten(1)[:, :h.shape[1]] + s["g_y"].float()
    x = h * rs
    we = s["weight"].float() * e
    dx = rs * (we - x * (we * x).mean(1, keepdim=True)) + s["g_h"].float()
    return dx.to(s["h"].dtype), (e * x).double().sum(0).float()


# ------------------------------------------------------------------ what a pass cannot do without
def _pairs(c):
    """(query-key pairs that are looked at, for one head; key tokens that are; query tokens)"""
    if c["form"] == "packed":
        each = [(x, x) for x in _lengths(c, 0).tolist()]
    elif c["form"] == "cache":
        each = [(c["q_len"], x) for x in _lengths(c, 0).tolist()]
    else:
        each = [(c["q_len"], c["kv_len"])] * c["batch"]
    pairs = keys = 0
    for lq, lk in each:
        if not c["causal"]:
            pairs, keys = pairs + lq * lk, keys + lk
            continue
        hi = torch.arange(lq) + 1 + lk - lq            # one past the last key of each query
        lo = (hi - c["window"]).clamp(min=0) if c["window"] else torch.zeros_like(hi)
        pairs += int((hi.clamp(min=0, max=lk) - lo).clamp(min=0).sum())
        keys += min(lk, max(0, lk - int(lo[0])))
    return pairs, keys, sum(x for x, _ in each)


def work(c):
    if c["op"] == "rotary":
        size = 2 if c["dtype"] == "bf16" else 4
        n = c["tokens"] * (c["q_heads"] + c["kv_heads"])
        return {"bytes": 2 * n * c["dim"] * size + 4 * c["tokens"] + 4 * c["rot"], "flops": 3 * n * c["rot"]}
    if c["op"] == "norm":
        size, n = (2 if c["dtype"] == "bf16" else 4), c["rows"] * c["n"]
        groups = c["rows"] * (1 if c["group"] <= 0 or c["group"] > c["n"] else -(-c["n"] // c["group"]))
        if c["back"]:
            return {"bytes": 5 * n * size + 4 * groups + 4 * c["rows"] + c["n"] * (size + 4), "flops": 12 * n}
        return {"bytes": n * (size * (3 if c["residual"] else 2) + 1 + (2 if c["y"] else 0)) + 4 * groups + 4 * c["rows"] + c["n"] * size, "flops": 7 * n}
    pairs, keys, rows = _pairs(c)
    q, kv = 2 * rows * c["q_heads"] * c["dim"], 2 * keys * c["kv_heads"] * c["dim"]
    if c["back"]:
        return {"bytes": 4 * q + 4 * kv + 4 * rows * c["q_heads"], "flops": 10 * pairs * c["q_heads"] * c["dim"]}
    return {"bytes": 2 * q + 2 * kv + 4 * rows * c["q_heads"], "flops": 4 * pairs * c["q_heads"] * c["dim"]}


# ------------------------------------------------------------------ 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rotary":
        sign = -1.0 if c["inverse"] else 1.0
        turn = torch.polar(torch.full((c["tokens"], c["rot"] // 2), s["mscale"], dtype=torch.float64, device=DEV),
                           sign * torch.outer(s["positions"].double(), s["inv_freq"]))
        outs = []
        for x in (s["q"].double(), s["k"].double()):
            first, second = ((slice(0, c["rot"] // 2), slice(c["rot"] // 2, c["rot"])) if c["pairs"] == "half"
                             else (slice(0, c["rot"], 2), slice(1, c["rot"], 2)))
            z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn[:, None]
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            outs.append(y)
        return tuple(outs)
    if c["op"] == "norm":
        w = s["weight"].double()
        rows, n, width = c["rows"], c["n"], s["width"]
        column = torch.arange(n, device=DEV) // width
        if not c["back"]:
            h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
            h = h.to(s["x"].dtype).double()
            rs = torch.rsqrt(h.square().sum(1) / n + EPS)
            y = w * (h * rs[:, None])
            top = torch.zeros((rows, int(column[-1]) + 1), dtype=torch.float64, device=DEV)
            top.scatter_reduce_(1, column.expand(rows, n), y.abs(), "amax")
            scale = torch.where(top == 0, 1.0, top / 127)
            each = scale[:, column]
            return (h, torch.round(y / each) * each, scale, rs) + ((y,) if c["y"] else ())
        h = s["h"].double()
        rs = torch.rsqrt(h.square().sum(1) / n + EPS)[:, None]
        e = s["g_codes"].double() / s["scale"].double()[:, column] + s["g_y"].double()
        # d y_j / d h_i = w_j rs (delta_ij - h_i h_j rs^2 / n)
        dot = (e * w * h).sum(1, keepdim=True)
        return rs * e * w - h * rs ** 3 * dot / n + s["g_h"].double(), (e * h * rs).sum(0)
    lengths = None
    if c["form"] == "packed":
        at = s["starts"].tolist()
        each = [(slice(at[i], at[i + 1]), slice(at[i], at[i + 1]), i) for i in range(c["batch"])]
        get = lambda x, i, rows: x[rows]  # noqa: E731
    else:
        lengths = s["lengths"].tolist() if c["form"] == "cache" else [c["kv_len"]] * c["batch"]
        each = [(slice(0, c["q_len"]), slice(0, lengths[i]), i) for i in range(c["batch"])]
        get = lambda x, i, rows: x[i, rows]  # noqa: E731
    share = c["q_heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device=DEV)
    dq, dk, dv = (torch.zeros(s[x].shape, dtype=torch.float64, device=DEV) for x in ("q", "k", "v"))
    for qr, kr, i in each:
        lq, lk = qr.stop - qr.start, kr.stop - kr.start
        back = torch.arange(lq, device=DEV)[:, None] + lk - lq - torch.arange(lk, device=DEV)[None, :]
        hide = torch.zeros((lq, lk), dtype=torch.bool, device=DEV)
        if c["causal"]:
            hide |= back < 0
        if c["window"]:
            hide |= back >= c["window"]
        for h in range(c["q_heads"]):
            q, k, v = get(s["q"], i, qr)[:, h].double(), get(s["k"], i, kr)[:, h // share].double(), get(s["v"], i, kr)[:, h // share].double()
            x = torch.mm(q, k.t()) * s["sm_scale"]
            x[hide] = -math.inf
            total = torch.logsumexp(x, 1) if lk else torch.full((lq,), -math.inf, dtype=torch.float64, device=DEV)
            p = torch.exp(x - torch.where(torch.isinf(total), torch.zeros_like(total), total)[:, None])
            p[hide] = 0.0
            if not c["back"]:
                get(out, i, qr)[:, h] = torch.mm(p, v)
                if c["form"] == "packed":
                    lse[h, qr] = total
                else:
                    lse[i, h] = total
                continue
            do = get(s["d_out"], i, qr)[:, h].double()
            dp = torch.mm(do, v.t())
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) * s["sm_scale"]
            get(dq, i, qr)[:, h] = torch.mm(ds, k)
            get(dk, i, kr)[:, h // share] += torch.mm(ds.t(), q)
            get(dv, i, kr)[:, h // share] += torch.mm(p.t(), do)
    return (dq, dk, dv) if c["back"] else (out, lse)
