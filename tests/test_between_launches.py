"""The launches of the operators between the projections, on the host: no grid passes what the runtime takes (2^32 work items
a dimension), however many sequences, heads and rows there are, and all rows are covered. The library runs in a process of
its own with tests/launch_hook.c in the place of the runtime's launch: no kernel runs, and no pointer is read."""
import json
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HOOK = os.path.join(ROOT, "tests", "launch_hook.c")
FAKE = 1 << 20

CHILD = r"""
import ctypes as C, json, sys
hook = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
sys.path.insert(0, sys.argv[2])
from r9700training_amd import AttnShape, Heads, lib
FAKE = 1 << 20

def heads(n, d, dtype=1, data=FAKE, gap=0):
    return Heads(data, 0, n * d + gap, d, n, dtype)

def attn(back, batch, hq, hk, d, q_tokens, kv_tokens, max_q, max_kv, causal=1, window=0):
    s = AttnShape(batch=batch, head_dim=d, q_len=max_q, kv_len=max_kv, q_starts=FAKE, kv_starts=FAKE, q_tokens=q_tokens,
                  kv_tokens=kv_tokens, causal=causal, window=window, scale=0.1)
    q, k = heads(hq, d), heads(hk, d)
    if back:
        need = lib().r97q_attn_bwd_workspace_bytes(s, hq, hk)
        return lib().r97q_attn_bwd(s, q, k, k, q, FAKE, q, q, k, k, FAKE, max(need, 1), None)
    need = lib().r97q_attn_fwd_workspace_bytes(s, hq, hk)
    return lib().r97q_attn_fwd(s, q, k, k, q, FAKE, FAKE, max(need, 0), None)

def norm(rows, n, group, dtype=1, codes=FAKE, data=FAKE):
    return lib().r97q_add_rmsnorm_i8g(data, data, FAKE, dtype, rows, n, group, 1e-6, 0.0, data, codes, codes, None, FAKE, None)

def norm_bwd(rows, n, group, dw, dtype=1):
    return lib().r97q_add_rmsnorm_i8g_bwd(FAKE, FAKE, dtype, rows, n, group, 0.0, FAKE, FAKE, FAKE, None, None, FAKE,
                                          FAKE if dw else None, 0, FAKE, 1 << 60, None)

def rotary(tokens, hq, dim, rot, dtype=1, data=FAKE, pairs=0):
    q = heads(hq, dim, dtype, data)
    return lib().r97q_rotary(q, heads(hq, dim, dtype, data + (1 << 40)), None, None, tokens, dim, rot, pairs, FAKE, None, 0, 1.0, 0, None)

for line in sys.stdin:
    what, args = json.loads(line)
    hook.hook_clear()
    rc = globals()[what](**args)
    out, one = [], (C.c_int64 * 30)()
    for i in range(min(hook.hook_count(), 4096)):
        hook.hook_launch(i, one)
        out.append(list(one))
    print(json.dumps([rc, hook.hook_count(), out, lib().r97q_last_error().decode()]), flush=True)
"""


@pytest.fixture(scope="session")
def hook(tmp_path_factory):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    so = str(tmp_path_factory.mktemp("hook") / "launch_hook.so")
    subprocess.run([cc, "-O1", "-Wall", "-shared", "-fPIC", "-o", so, HOOK], check=True)
    p = subprocess.Popen([sys.executable, "-c", CHILD, so, ROOT], stdin=subprocess.PIPE, stdout=subprocess.PIPE, text=True)
    yield p
    p.stdin.close()
    p.wait(timeout=60)


def launches(hook, what, **args):
    """The call's launches: [(grid, workgroup, words)], all of them accepted."""
    hook.stdin.write(json.dumps([what, args]) + "\n")
    hook.stdin.flush()
    rc, count, got, error = json.loads(hook.stdout.readline())
    assert rc == 0, (what, args, error)
    assert count == len(got)
    return [(tuple(x[:3]), tuple(x[3:6]), x[6:]) for x in got]


ATTENTION = [
    # many sequences with one long one among them: batch, q_heads, kv_heads, head_dim, q_tokens, kv_tokens, max_q, max_kv
    (1024, 32, 8, 64, 200000, 200000, 131072, 131072),
    (1024, 32, 8, 128, 200000, 200000, 131072, 131072),
    (1024, 32, 8, 256, 200000, 200000, 131072, 131072),
    # as many heads as are served, next to no tokens: neither cuts nor the join may pass the limit
    (65535, 128, 128, 64, 3, 3, 1, 1),
    (65535, 128, 128, 128, 40, 70000000, 1, 70000000),
    (65535, 128, 64, 256, 40, 70000000, 40, 70000000),
    (65535, 96, 2, 64, 500, 200000000, 500, 5000000),
    (65535, 128, 1, 256, 1, 9000000000, 1, 200000),
]


@pytest.mark.parametrize("b,hq,hk,d,qt,kt,mq,mk", ATTENTION)
@pytest.mark.parametrize("back", [False, True])
def test_attention_grids(hook, b, hq, hk, d, qt, kt, mq, mk, back):
    got = launches(hook, "attn", back=back, batch=b, hq=hq, hk=hk, d=d, q_tokens=qt, kv_tokens=kt, max_q=mq, max_kv=mk)
    assert got


NORM_MOST = 2 ** 31 - 1


@pytest.mark.parametrize("rows,n,group,size", [
    (NORM_MOST, 64, 0, 2), (NORM_MOST, 64, 8, 4), (NORM_MOST, 2056, 128, 2), (NORM_MOST, 16384, 0, 2), (NORM_MOST, 3, 2, 2),
    (NORM_MOST, 5, 3, 4), (NORM_MOST, 3, 1, 2), (NORM_MOST, 17408, 256, 2), (70_000_001, 60, 0, 2), (5, 64, 0, 2)])
def test_norm_grids(hook, rows, n, group, size):
    """The forward's launches take every row once, in order, each where the rows before it end."""
    got = launches(hook, "norm", rows=rows, n=n, group=group, dtype=1 if size == 2 else 0)
    groups = 1 if group <= 0 else -(-n // group)
    done = 0
    for grid, block, w in got:
        x, res, _, here, width, _, ngroups = w[:7]
        h, codes, scale, y, rstd = w[8:13]
        assert (width, ngroups, y) == (n, groups, 0)
        assert x == res == h == FAKE + done * n * size and codes == FAKE + done * n
        assert scale == FAKE + 4 * done * groups and rstd == FAKE + 4 * done
        # a row a workgroup, or one for each of its four waves
        assert here > 0 and here <= grid[0] * (4 if block[0] == 256 and grid[0] < here else 1)
        done += here
    assert done == rows and (rows > 10 ** 6 or len(got) == 1)


@pytest.mark.parametrize("rows,n,group", [(NORM_MOST, 64, 0), (NORM_MOST, 2056, 128), (NORM_MOST, 3, 2), (NORM_MOST, 3, 1)])
def test_norm_backward_grids(hook, rows, n, group):
    """The adjoint's workgroups walk the rows: one launch, and with the gain's gradient one more."""
    assert len(launches(hook, "norm_bwd", rows=rows, n=n, group=group, dw=False)) == 1
    assert len(launches(hook, "norm_bwd", rows=rows, n=n, group=group, dw=True)) == 2


@pytest.mark.parametrize("n", [2 ** 27, 2 ** 28 + 7, NORM_MOST])
def test_norm_gain_grids(hook, n):
    """Every column's partial sums are added, 32 columns a workgroup, each launch from where the one before it ends."""
    got = launches(hook, "norm_bwd", rows=2, n=n, group=0, dw=True)[1:]
    done = 0
    for grid, block, w in got:
        assert block[0] == 1024 and w[0] == FAKE + 4 * done
        done += 32 * grid[0]
    assert n <= done < n + 32


@pytest.mark.parametrize("tokens,heads,dim,rot,data,pairs", [
    (2 ** 31 - 1, 1, 64, 64, FAKE, 0), (16_777_300, 1, 2052, 2052, FAKE + 2, 0), (20_000_000, 1, 2100, 4, FAKE + 2, 0), (17_000_000, 32, 128, 128, FAKE, 1),
    (2 ** 31 - 1, 1, 8, 8, FAKE + 2, 1), (300, 4, 64, 64, FAKE, 0), (1, 28, 256, 64, FAKE, 0)])
def test_rotary_grids(hook, tokens, heads, dim, rot, data, pairs):
    """One launch; its workgroups hold all tokens, and a workgroup's table of sines its tokens' pairs."""
    (grid, _, w), = launches(hook, "rotary", tokens=tokens, hq=heads, dim=dim, rot=rot, data=data, pairs=pairs)
    each, half = w[14] & 0xFFFFFFFF, w[14] >> 32
    assert w[13] == tokens and half == rot // 2
    blocks = grid[0] * grid[2]
    assert each * half <= 4096 and (blocks - grid[2]) * each < tokens <= blocks * each
    assert grid[2] == 1 or tokens > 10 ** 6
