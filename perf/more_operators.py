"""The operators that continue a sequence from what is kept of it: rotary positions with several axes, the write of
new keys and values into a paged cache, attention of new tokens over that cache, and a gated linear recurrence,
forward and backward.

    listed()            the cases that stand for the ranges
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program holds before the call, on the card
    run(state)          one pass: the plain form where `own` is false, the package's kernels where it is true
    work(case)          the bytes and operations the pass cannot do without
    exact(case, seed)   the same outputs in float64, from the operators' definitions

Widths are those of the benchmark workloads and of the published real-model projections (1024-, 2048-, 4096-, 5120-
and 6144-wide activations, heads of 64, 128 and 256), 2048-token sequences eight at a time, and the odd and ragged
lengths between them.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
CHUNK = 128                                    # tokens between two states that the recurrence's forward keeps
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SCORES = 16 * 2048 * 16384                     # the most scores that a listed case has
PRODUCTS = 4 * SCORES * 256                    # the largest listed case's operations
VALUES = 8 * 2048 * 2048                       # the most values of a listed recurrence


def listed():
    return [
        # a serving loop's step: one token's 24 query and 4 key heads of 256 turned in a quarter of the head, after a
        # video in its context
        dict(name="axes_token", op="rotary", tokens=1, q_heads=24, kv_heads=4, dim=256, rot=64, axes=3, order="cycle",
             pairs="half", dtype="bf16", start=100000, inverse=False),
        # the backward of a training batch's rotation over text and images
        dict(name="axes_back", op="rotary", tokens=16384, q_heads=32, kv_heads=8, dim=128, rot=128, axes=3, order="blocks",
             pairs="half", dtype="bf16", start=0, inverse=True),
        # a serving batch's step: one new token of each of 16 sequences
        dict(name="write_token", op="write", form="dense", batch=16, q_len=1, kv_len=1024, kv_heads=8, dim=128, page=16,
             order="slots"),
        # a prompt's chunks: ragged pieces of four prompts
        dict(name="write_chunk", op="write", form="packed", batch=4, q_len=2048, kv_len=4096, kv_heads=8, dim=128, page=64,
             order="heads"),
        # a serving batch: 16 sequences of different lengths, one new token each, small pages
        dict(name="paged_batch", op="paged", form="dense", batch=16, q_len=1, kv_len=4096, q_heads=32, kv_heads=8, dim=128,
             page=16, window=0, order="slots"),
        # one new token against a long cache: 24 query heads share 4 key heads
        dict(name="paged_token", op="paged", form="dense", batch=1, q_len=1, kv_len=32768, q_heads=24, kv_heads=4, dim=256,
             page=64, window=0, order="heads"),
        # ragged chunks of four prompts in one call, a sliding window
        dict(name="paged_ragged", op="paged", form="packed", batch=4, q_len=500, kv_len=5000, q_heads=16, kv_heads=4, dim=64,
             page=32, window=1000, order="slots"),
        # a long prompt's last chunk
        dict(name="paged_chunk", op="paged", form="dense", batch=1, q_len=2048, kv_len=16384, q_heads=16, kv_heads=4, dim=128,
             page=64, window=0, order="slots"),
        # a serving batch's step: one token of 32 sequences from their kept states
        dict(name="scan_token", op="scan", form="dense", batch=32, length=1, width=4096, dtype="bf16", gated=True, back=False),
        # the forward of a training batch
        dict(name="scan_step", op="scan", form="dense", batch=8, length=2048, width=2048, dtype="bf16", gated=True, back=False),
        # the backward of packed odd lengths, without a gate on the input
        dict(name="scan_packed_back", op="scan", form="packed", batch=5, length=1300, width=1024, dtype="f32", gated=False,
             back=True),
        # the backward of one long sequence
        dict(name="scan_long_back", op="scan", form="dense", batch=1, length=16384, width=2048, dtype="bf16", gated=True,
             back=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * math.exp(rng.random() * math.log(hi / lo)))))


def draw(rng):
    op = rng.choice(["rotary", "write", "paged", "paged", "paged", "scan", "scan", "scan_back", "scan_back"])
    if op == "rotary":
        dim = rng.choice([64, 80, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        q_heads = kv_heads * rng.choice([1, 2, 4, 6])
        most = max(2, 16384 * 40 * 128 // (dim * (q_heads + kv_heads)) // 2)
        return dict(op="rotary", tokens=_log(rng, 1, min(16384, most)), q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                    rot=rng.choice([dim, dim // 2, dim // 4]), axes=rng.choice([2, 3]), order=rng.choice(["blocks", "cycle"]),
                    pairs=rng.choice(["half", "interleaved"]), dtype=rng.choice(["bf16", "f32"]),
                    start=rng.choice([0, rng.randrange(1, 200000)]), inverse=rng.random() < 0.5)
    if op in ("scan", "scan_back"):
        width = _log(rng, 64, 4096) if rng.random() < 0.3 else 64 * _log(rng, 2, 64)
        batch = _log(rng, 1, 32)
        most = VALUES // 2 // (width * batch)
        return dict(op="scan", form=rng.choice(["dense", "packed"]), batch=batch,
                    length=_log(rng, 1, max(2, min(16384, most))), width=width, dtype=rng.choice(["bf16", "bf16", "f32"]),
                    gated=rng.random() < 0.7, back=op == "scan_back")
    page = rng.choice([16, 16, 32, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    order = rng.choice(["slots", "heads"])
    if op == "write":
        form = rng.choice(["dense", "packed"])
        batch, dim = _log(rng, 1, 32), rng.choice([64, 80, 128, 256])
        q_len = rng.choice([1, _log(rng, 2, 2048)])
        kv_len = max(q_len, min(8192, _log(rng, 1, max(2, 16384 * 8 * 128 // (batch * kv_heads * dim)))))
        while batch * q_len * kv_heads * dim > 4 * 2048 * 8 * 128 or batch * kv_len * kv_heads * dim > 16384 * 8 * 256:
            q_len, kv_len = max(1, q_len // 2), max(1, q_len // 2, kv_len // 2)
        return dict(op="write", form=form, batch=batch, q_len=q_len, kv_len=kv_len, kv_heads=kv_heads, dim=dim, page=page,
                    order=order)
    dim = rng.choice([64, 64, 80, 128, 128, 256])
    q_heads = kv_heads * rng.choice([1, 2, 4, 6])
    while True:
        form = rng.choice(["dense", "packed"])
        token = form == "dense" and rng.random() < 0.6
        batch = _log(rng, 1, 32) if token else _log(rng, 1, 8)
        q_len = rng.choice([1, 1, 1, 2, 5]) if token else _log(rng, 16, 2048)
        kv_len = max(q_len, _log(rng, 16, 32768 if token else 16384))
        window = rng.choice([0, 0, _log(rng, 16, 2048)])
        scores = batch * q_heads * q_len * kv_len
        if scores <= SCORES // 2 and 4 * scores * dim <= PRODUCTS // 2 and batch * kv_len * kv_heads * dim <= 32768 * 4 * 256 * 2:
            return dict(op="paged", form=form, batch=batch, q_len=q_len, kv_len=kv_len, q_heads=q_heads, kv_heads=kv_heads,
                        dim=dim, page=page, window=window, order=order)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, shape, dtype, std=1.0):
    return (std * torch.randn(shape, generator=g, device=DEV)).to(dtype)


def _order(n, seed):
    return torch.randperm(n, generator=torch.Generator().manual_seed(int(seed)))


def _spread(n, longest, salt):
    """n lengths from one to the longest, the longest among them: the same ones for every seed."""
    g = torch.Generator().manual_seed(1000 * n + longest + salt)
    x = 1 + (torch.rand(n, generator=g) * (longest - 1)).round().long()
    x[0] = longest
    return x


def _lengths(c, seed):
    """(new tokens, tokens in the cache with them) of each sequence: the same pairs for every seed, in another order."""
    new = _spread(c["batch"], c["q_len"], 1) if c["form"] == "packed" else torch.full((c["batch"],), c["q_len"])
    held = torch.maximum(_spread(c["batch"], c["kv_len"], 2), new)
    p = _order(c["batch"], seed)
    return new[p], held[p]


def _starts(n):
    return torch.cat([torch.zeros(1, dtype=torch.long), n.cumsum(0)]).to(torch.int32).to(DEV)


def _sections(half, axes):
    """Pairs of each axis, the first (time) taking what does not divide."""
    each = half // (axes + 1) if axes == 3 else half // 2
    return [half - (axes - 1) * each] + [each] * (axes - 1)


def _pair_axis(c):
    """The axis of each pair: a block of pairs for each, or in turn as long as an axis has pairs left."""
    half = c["rot"] // 2
    left, axis = _sections(half, c["axes"]), []
    if c["order"] == "blocks":
        return [a for a, n in enumerate(left) for _ in range(n)]
    while len(axis) < half:
        for a in range(c["axes"]):
            if left[a]:
                left[a] -= 1
                axis.append(a)
    return axis


def _positions(c, g):
    """int32 [axes, tokens]: text, whose axes all count on, and between it pictures of 24 x 32 patches, whose tokens
    share a time and lie at their row and column."""
    t = torch.arange(c["tokens"], device=DEV)
    period, rows, cols = 1000, 24, 32
    at, run = t % period, t // period
    shift = int(torch.randint(0, 100, (1,), generator=g, device=DEV))
    base = c["start"] + shift + run * (period - rows * cols + cols)
    image = at < rows * cols
    text = base + cols + at - rows * cols
    axes = [torch.where(image, base, text), torch.where(image, base + at // cols, text),
            torch.where(image, base + at % cols, text)]
    return torch.stack(axes[3 - c["axes"]:]).to(torch.int32)


def _pools(c, g, pages):
    """Two pools of pages as a cache keeps them, [pages, slots, heads, dim] or (order "heads") the same view of
    [pages, heads, slots, dim]."""
    shape = (pages, c["page"], c["kv_heads"], c["dim"]) if c["order"] == "slots" else (pages, c["kv_heads"], c["page"], c["dim"])
    k, v = _randn(g, shape, torch.bfloat16), _randn(g, shape, torch.bfloat16)
    return (k, v) if c["order"] == "slots" else (k.transpose(1, 2), v.transpose(1, 2))


def _rates(g, n):
    """The channels' decay rates, from a memory of thousands of tokens to none."""
    return torch.exp(math.log(1e-3) + torch.rand(n, generator=g, device=DEV) * math.log(8e3))


def prepare(c, seed):
    g = _gen(seed)
    s = dict(c)
    if c["op"] == "rotary":
        dt, half = DTYPES[c["dtype"]], c["rot"] // 2
        s.update(q=_randn(g, (c["tokens"], c["q_heads"], c["dim"]), dt), k=_randn(g, (c["tokens"], c["kv_heads"], c["dim"]), dt),
                 inv_freq=(10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).to(DEV),
                 pair_axis=torch.tensor(_pair_axis(c), dtype=torch.int32, device=DEV), positions=_positions(c, g))
        s.update(q_out=torch.empty_like(s["q"]), k_out=torch.empty_like(s["k"]))
        return s
    if c["op"] == "scan":
        return _prepare_scan(c, s, g, seed)
    new, held = _lengths(c, seed)
    need = (held + c["page"] - 1) // c["page"]
    most = int(need.max())
    pages = int(need.sum()) + 3
    # pages lie in the pool as they were taken and given back, in no order; entries past a sequence's pages are -1
    table = torch.full((c["batch"], most), -1, dtype=torch.int32)
    table[torch.arange(most) < need[:, None]] = _order(pages, seed)[:int(need.sum())].to(torch.int32)
    s["table"], s["lengths"] = table.to(DEV), held.to(torch.int32).to(DEV)
    s["k_pages"], s["v_pages"] = _pools(c, g, pages)
    if c["form"] == "packed":
        s["starts"] = _starts(new)
    lead = (int(new.sum()),) if c["form"] == "packed" else (c["batch"], c["q_len"])
    if c["op"] == "write":
        # the projection's output holds k and v side by side
        kv = _randn(g, lead + (2, c["kv_heads"], c["dim"]), torch.bfloat16)
        s.update(k=kv.select(-3, 0), v=kv.select(-3, 1))
        return s
    shape = lead + (c["q_heads"], c["dim"])
    s.update(q=_randn(g, shape, torch.bfloat16), out=torch.empty(shape, dtype=torch.bfloat16, device=DEV),
             lse=torch.empty((c["q_heads"], lead[0]) if c["form"] == "packed" else (c["batch"], c["q_heads"], c["q_len"]),
                             dtype=torch.float32, device=DEV), sm_scale=1.0 / math.sqrt(c["dim"]))
    return s


def _scan_lengths(c, seed):
    if c["form"] == "dense":
        return torch.full((c["batch"],), c["length"])
    return _spread(c["batch"], c["length"], 3)[_order(c["batch"], seed)]


def _prepare_scan(c, s, g, seed):
    dt, n = DTYPES[c["dtype"]], _scan_lengths(c, seed)
    s["starts"] = _starts(n)
    lead = (int(n.sum()),) if c["form"] == "packed" else (c["batch"], c["length"])
    shape = lead + (c["width"],)
    s.update(x=_randn(g, shape, dt), gate=_randn(g, shape, dt, 2.0), input_gate=_randn(g, shape, dt) if c["gated"] else None,
             rate=_rates(g, c["width"]), h0=_randn(g, (c["batch"], c["width"]), torch.float32, 0.5))
    if not c["back"]:
        s.update(h=torch.empty(shape, dtype=dt, device=DEV), last=torch.empty_like(s["h0"]))
        return s
    s.update(d_h=_randn(g, shape, dt), d_last=_randn(g, (c["batch"], c["width"]), torch.float32))
    # what the forward kept: the state before each sequence's tokens 0, 128, 256, ..
    before = _before(s, _states(s))
    if c["form"] == "dense":
        s["states"] = before.view(c["batch"], c["length"], -1)[:, ::CHUNK].contiguous()
    else:
        start, at, rows = s["starts"].long(), torch.arange(before.shape[0], device=DEV), before.shape[0] // CHUNK + c["batch"]
        seq = torch.bucketize(at, start[1:], right=True)
        at = at - start[seq]
        keep = at % CHUNK == 0
        s["states"] = torch.zeros((rows, c["width"]), dtype=torch.float32, device=DEV)
        s["states"][(start[seq] // CHUNK + seq + at // CHUNK)[keep]] = before[keep]
    return s


# ------------------------------------------------------------------ the plain forms
def _rotary(x, s):
    """f32 [tokens, heads, dim]; the angles in f64, since a far position times a frequency loses its turn in f32."""
    half = s["rot"] // 2
    a = s["positions"].double()[s["pair_axis"].long()].T * s["inv_freq"]
    a = -a if s["inverse"] else a
    cos, sin = torch.cos(a).float()[:, None, :], torch.sin(a).float()[:, None, :]
    x = x.float()
    r, rest = x[..., :2 * half], x[..., 2 * half:]
    if s["pairs"] == "half":
        u, v = r[..., :half], r[..., half:]
        r = torch.cat([u * cos - v * sin, u * sin + v * cos], -1)
    else:
        u, v = r[..., 0::2], r[..., 1::2]
        r = torch.stack([u * cos - v * sin, u * sin + v * cos], -1).flatten(-2)
    return torch.cat([r, rest], -1)


def _new(s):
    """(sequence, position in the cache) of every new token, in order."""
    held = s["lengths"].long()
    if s["form"] == "dense":
        seq = torch.arange(s["batch"], device=DEV).repeat_interleave(s["q_len"])
        return seq, held[seq] - s["q_len"] + torch.arange(s["q_len"], device=DEV).repeat(s["batch"])
    start = s["starts"].long()
    at = torch.arange(s["tokens_in_all"], device=DEV)
    seq = torch.bucketize(at, start[1:], right=True)
    return seq, held[seq] + at - start[seq + 1]


def _write(s):
    s["tokens_in_all"] = s["k"].shape[0]
    seq, at = _new(s)
    page, slot = s["table"][seq, at // s["page"]].long(), at % s["page"]
    s["k_pages"][page, slot] = s["k"].reshape((-1,) + s["k"].shape[-2:])
    s["v_pages"][page, slot] = s["v"].reshape((-1,) + s["v"].shape[-2:])
    return s["k_pages"], s["v_pages"]


def _gather(pages, s):
    """f32 [batch, query heads, tokens, dim]: a sequence's pages in a row, each key head once for every query head."""
    x = pages[s["table"].clamp(min=0).long()].flatten(1, 2)[:, :s["kv_len"]].float()
    return x.transpose(1, 2).repeat_interleave(s["q_heads"] // s["kv_heads"], 1)


def _paged(s):
    """(out f32, log-sum-exp f32); a query that sees nothing gives zeros and minus infinity."""
    q, packed = s["q"].float(), s["form"] == "packed"
    if packed:  # ragged chunks as a batch of the longest one's length, ending together
        s["tokens_in_all"] = q.shape[0]
        seq, at = _new(s)
        row = at - s["lengths"].long()[seq] + s["q_len"]
        q = q.new_zeros((s["batch"], s["q_len"]) + q.shape[1:]).index_put((seq, row), q)
    x = q.transpose(1, 2) @ _gather(s["k_pages"], s).transpose(2, 3).contiguous() * s["sm_scale"]
    held = s["lengths"].long()[:, None, None, None]
    key = torch.arange(x.shape[-1], device=DEV)
    far = torch.arange(s["q_len"], device=DEV)[:, None] + held - s["q_len"] - key
    see = (far >= 0) & (key < held)
    if s["window"]:
        see = see & (far < s["window"])
    x = x.masked_fill_(~see, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x.sub_(torch.where(m == -math.inf, 0.0, m)))
    total = p.sum(-1, keepdim=True)
    o = ((p @ _gather(s["v_pages"], s)) / torch.where(total > 0, total, 1.0)).transpose(1, 2)
    lse = (m + torch.log(total))[..., 0]
    return (o[seq, row], lse[seq, :, row].T.contiguous()) if packed else (o, lse)


def _scan(a, u, longest):
    """h of h[t] = a[t] h[t - 1] + u[t] along the first axis, spans of 1, 2, 4, .. tokens joined two by two. a is zero where
    a sequence begins, so nothing passes from one to the next."""
    span = 1
    while span < longest:
        u = torch.cat([u[:span], u[span:] + a[span:] * u[:-span]])
        a = torch.cat([a[:span], a[span:] * a[:-span]])
        span *= 2
    return u


def _flat(x):
    return x.reshape(-1, x.shape[-1]).float()


def _ends(s):
    """Indices of the sequences' first and last tokens among all tokens."""
    start = s["starts"].long()
    return start[:-1], start[1:] - 1


def _parts(s):
    """f32 (sigmoid of the gate, decay a, the input's factor, the gated input), tokens in a row. The decay by its
    distance from one: thousands of decays next to one are multiplied, and an error with a sign would add up."""
    sg = torch.sigmoid(_flat(s["gate"]))
    la = -s["rate"] * sg
    w = _flat(s["x"]) * torch.sigmoid(_flat(s["input_gate"])) if s["gated"] else _flat(s["x"])
    return sg, 1.0 + torch.expm1(la), torch.sqrt(-torch.expm1(2.0 * la)), w


def _states(s):
    """f32 [tokens, width]: every token's state."""
    _, a, b, w = _parts(s)
    first, u = _ends(s)[0], b * w
    u[first] += a[first] * s["h0"]
    a[first] = 0.0
    return _scan(a, u, s["length"])


def _before(s, h):
    """Each token's state before it."""
    h = torch.roll(h, 1, 0)
    h[_ends(s)[0]] = s["h0"]
    return h


def _scan_back(s):
    """f32 (dx, dgate, dinput_gate, drate, dh0)"""
    sg, a, b, w = _parts(s)
    before = _before(s, _states(s))
    first, last = _ends(s)
    e = _flat(s["d_h"])
    e = e.index_add(0, last, s["d_last"])
    turn = torch.roll(a, -1, 0)
    turn[last] = 0.0
    lam = _scan(turn.flip(0), e.flip(0), s["length"]).flip(0)
    dla = lam * a * (before - a * w / b)
    dw = lam * b
    drate = -(sg * dla).double().sum(0).float()
    dgate = -s["rate"] * sg * (1.0 - sg) * dla
    dh0 = a[first] * lam[first]
    if not s["gated"]:
        return dw, dgate, drate, dh0
    si = torch.sigmoid(_flat(s["input_gate"]))
    return dw * si, dgate, dw * _flat(s["x"]) * si * (1.0 - si), drate, dh0


# ------------------------------------------------------------------ one pass
def run(s):
    if s["op"] == "rotary":
        if own:
            from r9700training_amd.rotary import rotary_axes

            return rotary_axes(s["q"], s["k"], s["inv_freq"], s["positions"], s["pair_axis"], pairs=s["pairs"],
                               inverse=s["inverse"], q_out=s["q_out"], k_out=s["k_out"])
        return _rotary(s["q"], s).to(s["q"].dtype), _rotary(s["k"], s).to(s["k"].dtype)
    if s["op"] == "scan":
        return _run_scan_back(s) if s["back"] else _run_scan(s)
    packed = dict(q_starts=s["starts"], max_q=s["q_len"]) if s["form"] == "packed" else {}
    if s["op"] == "write":
        if own:
            from r9700training_amd.paged import paged_write

            paged_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], **packed)
            return s["k_pages"], s["v_pages"]
        return _write(s)
    if own:
        from r9700training_amd.paged import paged_attention_fwd

        return paged_attention_fwd(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], window=s["window"],
                                   scale=s["sm_scale"], max_kv=s["kv_len"], out=s["out"], lse=s["lse"], **packed)
    out, lse = _paged(s)
    return out.to(torch.bfloat16), lse


def _run_scan(s):
    """(h in the inputs' type, the last states f32)"""
    packed = s["form"] == "packed"
    if own:
        from r9700training_amd.recurrence import recurrence_fwd

        return recurrence_fwd(s["x"], s["gate"], s["rate"], s["input_gate"], h0=s["h0"], out=s["h"], last=s["last"],
                              **(dict(starts=s["starts"], max_len=s["length"]) if packed else {}))[:2]
    h = _states(s)
    return h.to(s["x"].dtype).view(s["x"].shape), h[_ends(s)[1]]


def _run_scan_back(s):
    """(dx, dgate, dinput_gate where there is one, in the inputs' type; drate and dh0 f32)"""
    if own:
        from r9700training_amd.recurrence import recurrence_bwd

        grads = recurrence_bwd(s["x"], s["gate"], s["rate"], s["states"], s["d_h"], s["input_gate"], d_last=s["d_last"],
                               **(dict(starts=s["starts"], max_len=s["length"]) if s["form"] == "packed" else {}))
        return tuple(x for x in grads if x is not None)
    grads = _scan_back(s)
    return tuple(x.to(s["x"].dtype).view(s["x"].shape) for x in grads[:-2]) + grads[-2:]


# ------------------------------------------------------------------ what a pass cannot do without
def work(c):
    if c["op"] == "rotary":
        size, n = (2 if c["dtype"] == "bf16" else 4), c["tokens"] * (c["q_heads"] + c["kv_heads"])
        return {"bytes": 2 * n * c["dim"] * size + 4 * c["axes"] * c["tokens"] + 6 * c["rot"], "flops": 3 * n * c["rot"]}
    if c["op"] == "scan":
        size, tokens = (2 if c["dtype"] == "bf16" else 4), int(_scan_lengths(c, 0).sum())
        n, ends, inputs = tokens * c["width"], 4 * c["batch"] * c["width"], 3 if c["gated"] else 2
        if not c["back"]:
            return {"bytes": n * size * (inputs + 1) + 2 * ends + 4 * c["width"], "flops": 20 * n}
        kept = 4 * c["width"] * int(((_scan_lengths(c, 0) + CHUNK - 1) // CHUNK).sum())
        return {"bytes": n * size * (2 * inputs + 1) + kept + 2 * ends + 8 * c["width"], "flops": 45 * n}
    new, held = _lengths(c, 0)
    row = 2 * c["kv_heads"] * c["dim"]
    if c["op"] == "write":
        return {"bytes": 4 * row * int(new.sum()) + 8 * c["batch"], "flops": 0}
    pairs = keys = 0
    for n, m in zip(new.tolist(), held.tolist()):
        hi = torch.arange(n) + 1 + m - n               # one past the last key of each query
        lo = (hi - c["window"]).clamp(min=0) if c["window"] else torch.zeros_like(hi)
        pairs, keys = pairs + int((hi - lo).sum()), keys + m - int(lo[0])
    rows = int(new.sum()) * c["q_heads"]
    return {"bytes": 4 * rows * c["dim"] + 2 * row * keys + 4 * rows + 4 * keys // c["page"], "flops": 4 * pairs * c["q_heads"] * c["dim"]}


# ------------------------------------------------------------------ 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rotary":
        angle = torch.stack([s["positions"][a].double() * s["inv_freq"][i] for i, a in enumerate(_pair_axis(c))], 1)
        turn = torch.polar(torch.ones_like(angle), -angle if c["inverse"] else angle)
        first, second = ((slice(0, c["rot"] // 2), slice(c["rot"] // 2, c["rot"])) if c["pairs"] == "half"
                         else (slice(0, c["rot"], 2), slice(1, c["rot"], 2)))
        outs = []
        for x in (s["q"].double(), s["k"].double()):
            z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn[:, None]
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            outs.append(y)
        return tuple(outs)
    if c["op"] == "scan":
        return _exact_scan(c, s)
    held = s["lengths"].tolist()
    table = s["table"].tolist()
    start = s["starts"].tolist() if c["form"] == "packed" else None
    share = c.get("q_heads", 1) // c["kv_heads"]
    if c["op"] == "write":
        k, v = s["k_pages"].double(), s["v_pages"].double()
        for b, m in enumerate(held):
            new_k, new_v = ((x[start[b]:start[b + 1]] if start else x[b]).double() for x in (s["k"], s["v"]))
            at = m - new_k.shape[0]
            done = 0
            while done < new_k.shape[0]:
                slot = (at + done) % c["page"]
                n = min(c["page"] - slot, new_k.shape[0] - done)
                page = table[b][(at + done) // c["page"]]
                k[page, slot:slot + n], v[page, slot:slot + n] = new_k[done:done + n], new_v[done:done + n]
                done += n
        return k, v
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device=DEV)
    for b, m in enumerate(held):
        ids = s["table"][b, :(m + c["page"] - 1) // c["page"]].long()
        k, v = s["k_pages"][ids].flatten(0, 1)[:m].double(), s["v_pages"][ids].flatten(0, 1)[:m].double()
        q, to = (s["q"][start[b]:start[b + 1]], out[start[b]:start[b + 1]]) if start else (s["q"][b], out[b])
        n = q.shape[0]
        behind = torch.arange(m - n, m, device=DEV)[:, None] - torch.arange(m, device=DEV)[None, :]
        hide = behind < 0
        if c["window"]:
            hide |= behind >= c["window"]
        for h in range(c["q_heads"]):
            x = torch.mm(q[:, h].double(), k[:, h // share].t().contiguous()) * s["sm_scale"]
            x[hide] = -math.inf
            total = torch.logsumexp(x, 1)
            to[:, h] = torch.mm(torch.exp(x - total[:, None]), v[:, h // share].contiguous())
            if start:
                lse[h, start[b]:start[b + 1]] = total
            else:
                lse[b, h] = total
    return out, lse


def _exact_scan(c, s):
    """Token by token, all sequences side by side; a sequence that is over rests."""
    n = (s["starts"][1:] - s["starts"][:-1]).tolist()
    longest, width = max(n), c["width"]

    def side(x):  # f64 [longest, batch, width], ragged sequences filled up with zeros
        x = x.double()
        if c["form"] == "dense":
            return x.transpose(0, 1).contiguous()
        return torch.nn.utils.rnn.pad_sequence(list(x.split(n)))

    def row(x):
        if c["form"] == "dense":
            return x.transpose(0, 1).contiguous()
        return torch.cat([x[:m, b] for b, m in enumerate(n)])

    alive = (torch.arange(longest)[:, None] < torch.tensor(n)[None, :]).to(DEV)[..., None]
    x, gate, rate = side(s["x"]), side(s["gate"]), s["rate"].double()
    open_ = 1.0 / (1.0 + torch.exp(-gate))
    decay = torch.where(alive, torch.exp(-open_ * rate), 1.0)
    less = -torch.expm1(-2.0 * open_ * rate)         # 1 - decay^2
    room = torch.sqrt(less)
    enter = 1.0 / (1.0 + torch.exp(-side(s["input_gate"]))) if c["gated"] else torch.ones_like(x)
    add = torch.where(alive, room * enter * x, 0.0)
    h, before, after = s["h0"].double(), [], []
    for t in range(longest):
        before.append(h)
        h = decay[t] * h + add[t]
        after.append(h)
    if not c["back"]:
        return row(torch.stack(after)), h
    d_h, lam = side(s["d_h"]), s["d_last"].double()
    full = [None] * longest
    for t in range(longest - 1, -1, -1):
        full[t] = lam + d_h[t]                         # a resting sequence's cotangent is zero and its decay one
        lam = decay[t] * full[t]
    full, before = torch.stack(full), torch.stack(before)
    d_decay = torch.where(alive, full * (before - decay * enter * x / room), 0.0)
    d_open = -rate * decay * d_decay
    grads = [full * room * enter, d_open * open_ * (1.0 - open_)]
    if c["gated"]:
        grads.append(full * room * x * enter * (1.0 - enter))
    return tuple(row(y) for y in grads) + (-(open_ * decay * d_decay).sum((0, 1)), lam)
