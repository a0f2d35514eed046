"""The operators that continue a sequence, together as a serving loop of a hybrid model runs them: ragged chunks of several
prompts, then a token of each at a time, through the recurrence (from its kept states), rotary positions with three axes, the
paged cache's write and attention over it; every stage against float64 from its own inputs over the whole sequences."""
import math

import pytest
import torch

import between_ref as A
import recurrence_ref as R
from test_gpu_paged import close as close_attention

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def rnd(g, *shape, std=1.0):
    return (std * torch.randn(shape, generator=g, device="cuda")).to(BF)


@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128)])
def test_prompts_in_chunks_and_tokens(page, dim):
    from r9700training_amd.paged import paged_attention_fwd, paged_write
    from r9700training_amd.recurrence import recurrence_fwd
    from r9700training_amd.rotary import rotary_axes, rotary_frequencies, rotary_pair_axes

    heads, kv_heads, batch = 6, 2, 3
    width = (heads + 2 * kv_heads) * dim
    # new tokens of each prompt in each call
    calls = [[300, 0, 41], [17, 130, 0], [1, 1, 1], [1, 1, 1], [260, 1, 5]]
    total = [sum(c[b] for c in calls) for b in range(batch)]
    g = torch.Generator(device="cuda").manual_seed(5)
    x, gate, gi = ([rnd(g, n, width, std=s) for n in total] for s in (1.0, 2.0, 1.0))
    rate = torch.exp(torch.linspace(math.log(1e-3), math.log(8.0), width, device="cuda"))
    where = [torch.stack([torch.arange(n) // 5, torch.arange(n) % 7, torch.arange(n)]).to(torch.int32).cuda() for n in total]
    freq, _ = rotary_frequencies(dim)
    axis = rotary_pair_axes([dim // 2 - 2 * (dim // 6), dim // 6, dim // 6], "cycle")
    need = [-(-n // page) for n in total]
    table = torch.full((batch, max(need)), -1, dtype=torch.int32)
    ids = torch.randperm(sum(need), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    for b in range(batch):
        table[b, :need[b]] = ids[sum(need[:b]):sum(need[:b + 1])]
    table = table.cuda()
    kp, vp = (torch.full((sum(need), page, kv_heads, dim), math.nan, dtype=BF, device="cuda") for _ in range(2))
    state = torch.zeros((batch, width), device="cuda")
    held = [0] * batch
    mixed, turned, out = [[[] for _ in range(batch)] for _ in range(3)]
    for new in calls:
        starts = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
        part = lambda t: torch.cat([t[b][held[b]:held[b] + new[b]] for b in range(batch)])  # noqa: E731
        h, _, _ = recurrence_fwd(part(x), part(gate), rate, part(gi), h0=state, last=state, starts=starts, max_len=max(new))
        q, k, v = (t.unflatten(1, (-1, dim)) for t in h.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
        pos = torch.cat([where[b][:, held[b]:held[b] + new[b]] for b in range(batch)], 1)
        q, k = rotary_axes(q, k, freq, pos, axis)
        held = [a + n for a, n in zip(held, new)]
        lens = torch.tensor(held, dtype=torch.int32, device="cuda")
        kw = dict(q_starts=starts, max_q=max(new))
        paged_write(k, v, kp, vp, table, lens, **kw)
        o, _ = paged_attention_fwd(q, kp, vp, table, lens, **kw)
        for b, (a, e) in enumerate(zip(starts.tolist(), starts.tolist()[1:])):
            mixed[b].append(h[a:e])
            turned[b].append((q[a:e], k[a:e]))
            out[b].append(o[a:e])
    for b in range(batch):
        h = torch.cat(mixed[b])
        ref = R.forward(x[b].double(), gate[b].double(), rate.double(), gi[b].double(), torch.zeros(width, dtype=torch.float64, device="cuda"))
        value, err = ref["h"]
        tol = err * (1 + len(calls)) + A.HALF[BF] * (value.abs() + err)  # each call joins anew
        assert float(((h.double() - value).abs() - tol).max()) <= 0
        q, k = torch.cat([t for t, _ in turned[b]]), torch.cat([t for _, t in turned[b]])
        angles = where[b].double()[axis.long()].T * freq
        for src, got in ((h[:, :heads * dim], q), (h[:, heads * dim:(heads + kv_heads) * dim], k)):
            src = src.unflatten(1, (-1, dim)).double()
            want = A.rotary(src, angles, dim, "half", 1.0, False)
            size = src.abs() + torch.cat([src[..., dim // 2:], src[..., :dim // 2]], -1).abs()
            assert float(((got.double() - want).abs() - A.HALF[BF] * want.abs() - 2 * 12 * A.U32 * size).max()) <= 0
        v = h[:, (heads + kv_heads) * dim:].unflatten(1, (-1, dim))
        ref = A.reference([(q.double(), k.double(), v.double(), None)], heads, kv_heads, True, 0, 1.0 / math.sqrt(dim), A.HALF[BF])
        close_attention(torch.cat(out[b]), *ref[0]["out"], f"sequence {b}")
