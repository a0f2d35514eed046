"""The launches of the operators that continue a sequence, on the host: no grid passes what the runtime takes (2^32 work items a
dimension), and ranges cover the tokens. The library runs in a process of its own with tests/launch_hook.c in the place of the
runtime's launch: no kernel runs, and no pointer is read."""
import json
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HOOK = os.path.join(ROOT, "tests", "launch_hook.c")

CHILD = r"""
import ctypes as C, json, sys
hook = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
sys.path.insert(0, sys.argv[2])
from r9700training_amd import AttnShape, Heads, Pages, Recurrence, Rows, lib
FAKE = 1 << 20

def heads(n, d, page=1):
    return Heads(FAKE, page * n * d, n * d, d, n, 1)

def paged(batch, hq, hk, d, q_len, kv_len, page, max_pages, pages, packed=0, window=0):
    s = AttnShape(batch=batch, head_dim=d, q_len=q_len, kv_len=kv_len, kv_lens=FAKE, causal=1, window=window, scale=0.1)
    if packed:
        s.q_starts, s.q_tokens = FAKE, packed
    p = Pages(FAKE, max_pages, pages, page, max_pages)
    need = lib().r97q_paged_attn_fwd_workspace_bytes(s, p, hq, hk)
    return lib().r97q_paged_attn_fwd(s, p, heads(hq, d), heads(hk, d, page), heads(hk, d, page), heads(hq, d), FAKE, FAKE, max(need, 0), None)

def write(batch, hk, d, q_len, page, max_pages, pages, packed=0):
    s = AttnShape(batch=batch, head_dim=d, q_len=q_len, kv_len=1, kv_lens=FAKE, causal=1, scale=0.1)
    if packed:
        s.q_starts, s.q_tokens = FAKE, packed
    p = Pages(FAKE, max_pages, pages, page, max_pages)
    return lib().r97q_paged_write(s, p, heads(hk, d), heads(hk, d), heads(hk, d, page), heads(hk, d, page), None)

def scan(back, batch, channels, length, dtype=1, packed=0, off=0):
    s = Recurrence(batch, channels, length, FAKE if packed else None, packed, dtype)
    r = Rows(FAKE + off, length * channels, channels)
    outs = [Rows(i * FAKE + off, length * channels, channels) for i in (2, 3, 4)]
    if back:
        return lib().r97q_recurrence_bwd(s, r, r, r, FAKE, FAKE, r, None, *outs, FAKE, FAKE, FAKE, max(lib().r97q_recurrence_bwd_workspace_bytes(s), 0), None)
    return lib().r97q_recurrence_fwd(s, r, r, r, FAKE, FAKE, r, FAKE, FAKE, FAKE, max(lib().r97q_recurrence_fwd_workspace_bytes(s), 0), None)

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


@pytest.fixture(scope="module")
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
    """The call's launches, [(grid, workgroup)], all of them accepted."""
    hook.stdin.write(json.dumps([what, args]) + "\n")
    hook.stdin.flush()
    rc, count, got, error = json.loads(hook.stdout.readline())
    assert rc == 0, (what, args, error)
    assert count == len(got)
    return [(tuple(x[:3]), tuple(x[3:6])) for x in got]


@pytest.mark.parametrize("b,hq,hk,d,q,kv,page,most,pages", [
    (65535, 128, 128, 64, 1, 1, 8, 1, 70000), (65535, 128, 64, 256, 3, 40, 16, 3, 200000), (1, 8, 8, 128, 1, 0x7FFFFF00, 1 << 20, 2047, 4000),
    (1, 24, 4, 256, 1, 200000, 64, 4000, 5000), (1, 1, 1, 64, 1 << 24, 1 << 24, 64, 1 << 18, 1 << 18), (7, 16, 4, 128, 2048, 16384, 16, 1024, 9000)])
def test_paged_grids(hook, b, hq, hk, d, q, kv, page, most, pages):
    got = launches(hook, "paged", batch=b, hq=hq, hk=hk, d=d, q_len=q, kv_len=kv, page=page, max_pages=most, pages=pages)
    assert got
    # packed, and planned for a length that is too small or too large
    for length in (0, 1, q):
        for kv_len in (0, 1, 0x7FFFFF00):
            assert launches(hook, "paged", batch=b, hq=hq, hk=hk, d=d, q_len=length, kv_len=kv_len, page=page, max_pages=most, pages=pages,
                            packed=b + q)


@pytest.mark.parametrize("b,hk,d,q,packed", [(65535, 128, 256, 1, 0), (1, 1, 8, 0x7FFFFF00, 0), (4, 8, 128, 0, 5000), (65535, 8, 128, 1 << 20, 1 << 30)])
def test_write_grids(hook, b, hk, d, q, packed):
    (grid, block), = launches(hook, "write", batch=b, hk=hk, d=d, q_len=q, page=16, max_pages=100, pages=1000, packed=packed)
    assert grid[1] == b and block == (256, 1, 1)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("batch,channels,length", [
    (1, 64, 2 ** 31 - 1), (65535, 64, 1), (65535, 4096, 300), (1, 2 ** 27, 1), (2, 2 ** 27, 700), (1, 1, 5000), (3, 100, 16384), (300, 1024, 64), (1, 64, 0)])
def test_recurrence_grids(hook, back, batch, channels, length):
    """One launch over the tokens, with ranges one before it for the spans of all but one, and in the backward one that adds the
    rate's gradients where there is more than one sequence or range."""
    for off in (0, 2):  # pieces of 16 bytes, and single values
        got = launches(hook, "scan", back=back, batch=batch, channels=channels, length=length, off=off)
        adds = back and got[-1][1][0] == 1024
        main = got[-2] if adds else got[-1]
        few, slabs = main[1][0] == 64, -(-channels // 64)
        cut = len(got) == 2 + adds
        if few:
            assert main[0][1] == batch
        elif main[0][1:] == (1, 1) and slabs >= 4 and main[0][0] % 8 == 0 and main[0][0] != slabs:
            # dealt by XCD: all workgroups, and up to seven too many
            ranges = main[0][0] // (slabs * batch)
            assert 0 <= main[0][0] - slabs * ranges * batch < 8 and ranges <= 257
            assert not cut or got[0][0][0] >= slabs * (ranges - 1) * batch
        else:
            ranges = main[0][1]
            assert main[0] == (slabs, ranges, batch) and ranges <= 257
            x, y, z = got[0][0]  # a range's spans
            assert not cut or ((x, z) == (slabs, batch) and y > 0 and y % (ranges - 1) == 0)
        assert len(got) == 1 + cut + adds and (not back or adds == (batch > 1 or cut))
    packed = launches(hook, "scan", back=back, batch=batch, channels=channels, length=0, packed=min(batch * max(length, 1), 2 ** 31 - 1))
    assert packed
