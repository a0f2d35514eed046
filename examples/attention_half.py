"""The attention half of a decoder layer on the card, as a program would run it: the norm with the residual's addition
gives 8-bit codes, the coded projection reads them, q and k are turned, attention runs, and the output projection
with its adapter closes it; then the whole way back. And the same layer a token at a time over a cache.

    python examples/attention_half.py [--tokens 2048] [--batch 1]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from r9700training_amd.attention import attention_bwd, attention_fwd  # noqa: E402
from r9700training_amd.norm import add_rmsnorm_i8g, add_rmsnorm_i8g_bwd  # noqa: E402
from r9700training_amd.qlinear import QWeight, gemm_nt_q_dx, gemm_nt_q_fwd, qlinear_lora_bwd, qlinear_lora_fwd  # noqa: E402
from r9700training_amd.rotary import rotary, rotary_frequencies  # noqa: E402

GROUP = 128  # columns a scale of the coded trunk


class AttentionHalf:
    """Frozen coded weights (codes int8 and a bf16 scale every 128 columns) and the trained parts: the norm's gain and the
    output projection's adapter."""

    def __init__(self, width: int, heads: int, kv_heads: int, head_dim: int, rank: int = 16, seed: int = 0):
        self.width, self.heads, self.kv_heads, self.dim = width, heads, kv_heads, head_dim
        g = torch.Generator(device="cuda").manual_seed(seed)

        def coded(n, k):
            codes = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
            scale = (torch.rand((n, k // GROUP), generator=g, device="cuda") + 0.5) / (73.0 * k ** 0.5)
            return codes, scale.to(torch.bfloat16).view(torch.int16)

        self.qkv = coded((heads + 2 * kv_heads) * head_dim, width)
        self.out = coded(width, heads * head_dim)
        self.w_qkv, self.w_out = QWeight.from_decoded(*self.qkv), QWeight.from_decoded(*self.out)
        self.gain = (1.0 + 0.1 * torch.randn(width, generator=g, device="cuda")).to(torch.bfloat16)
        self.A = (0.05 * torch.randn((rank, heads * head_dim), generator=g, device="cuda")).to(torch.bfloat16)
        self.B = (0.05 * torch.randn((width, rank), generator=g, device="cuda")).to(torch.bfloat16)
        self.inv_freq, self.mscale = rotary_frequencies(head_dim, scaling="linear", factor=2.0)

    def split(self, y):
        """q, k, v [tokens, heads, head_dim] as views of the projection's output (or of its gradient)."""
        hq, hk, d = self.heads, self.kv_heads, self.dim
        return (y[:, :hq * d].unflatten(1, (hq, d)), y[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d)),
                y[:, (hq + hk) * d:].unflatten(1, (hk, d)))

    def project(self, x, residual, positions):
        """(codes, scale, h, rstd, y): y holds q and k turned in place, and v."""
        codes, scale, h, _, rstd = add_rmsnorm_i8g(x, residual, self.gain, GROUP)
        y = gemm_nt_q_fwd(*self.qkv, codes, scale, y_dtype=torch.bfloat16)
        q, k, _ = self.split(y)
        rotary(q, k, self.inv_freq, positions, mscale=self.mscale, q_out=q, k_out=k)
        return codes, scale, h, rstd, y

    def forward(self, x, residual, starts, longest):
        """x, residual bf16 [tokens, width], sequences packed at `starts`. (z, h, what the way back needs)"""
        positions = torch.arange(x.shape[0], dtype=torch.int32, device=x.device)
        positions -= torch.repeat_interleave(starts[:-1], starts.diff(), output_size=x.shape[0])
        codes, scale, h, rstd, y = self.project(x, residual, positions)
        q, k, v = self.split(y)
        o, lse = attention_fwd(q, k, v, q_starts=starts, kv_starts=starts, max_q=longest, max_kv=longest)
        z, t = qlinear_lora_fwd(self.w_out, o.flatten(1), self.A, self.B, 1.0)
        return z, h, dict(scale=scale, h=h, rstd=rstd, y=y, o=o, lse=lse, t=t, positions=positions, starts=starts, longest=longest)

    def backward(self, s, dz, dh):
        """dz, dh: the cotangents of z and of the residual stream h. (dx, which is the residual's too, and the trained
        parts' gradients)"""
        do, dA, dB = qlinear_lora_bwd(self.w_out, s["o"].flatten(1), dz, self.A, self.B, s["t"], 1.0)
        q, k, v = self.split(s["y"])
        dy = torch.empty_like(s["y"])
        dq, dk, dv = self.split(dy)  # the gradients go straight into the projection's cotangent
        attention_bwd(q, k, v, s["o"], s["lse"], do.view_as(s["o"]), q_starts=s["starts"], kv_starts=s["starts"],
                      max_q=s["longest"], max_kv=s["longest"], dq=dq, dk=dk, dv=dv)
        rotary(dq, dk, self.inv_freq, s["positions"], mscale=self.mscale, inverse=True, q_out=dq, k_out=dk)
        g_codes = gemm_nt_q_dx(self.w_qkv, dy, s["scale"], da_dtype=torch.bfloat16)
        dx, dgain = add_rmsnorm_i8g_bwd(s["h"], self.gain, s["rstd"], GROUP, scale=s["scale"], g_codes=g_codes, g_h=dh)
        return dict(dx=dx, dgain=dgain, dA=dA, dB=dB, dy=dy, do=do, g_codes=g_codes)

    def cache(self, batch, room):
        """Keys, values [batch, room, kv_heads, head_dim] and how much of them is in use."""
        shape = (batch, room, self.kv_heads, self.dim)
        return dict(k=torch.zeros(shape, dtype=torch.bfloat16, device="cuda"), v=torch.zeros(shape, dtype=torch.bfloat16, device="cuda"),
                    lens=torch.zeros(batch, dtype=torch.int32, device="cuda"))

    def token(self, x, residual, cache):
        """One token a sequence: x, residual bf16 [batch, width]. (z, h); the cache grows by one."""
        _, _, h, _, y = self.project(x, residual, cache["lens"])
        q, k, v = self.split(y)
        at = cache["lens"].long()
        row = torch.arange(at.shape[0], device=at.device)
        cache["k"][row, at], cache["v"][row, at] = k, v
        cache["lens"] += 1
        o, _ = attention_fwd(q[:, None], cache["k"], cache["v"], kv_lens=cache["lens"])
        z, _ = qlinear_lora_fwd(self.w_out, o.flatten(1), self.A, self.B, 1.0)
        return z, h


def main() -> None:
    p = argparse.ArgumentParser()
    p.add_argument("--tokens", type=int, default=2048)
    p.add_argument("--batch", type=int, default=1)
    a = p.parse_args()
    layer = AttentionHalf(2048, 16, 4, 128)
    starts = torch.arange(a.batch + 1, dtype=torch.int32, device="cuda") * a.tokens
    n = a.batch * a.tokens
    x, r, dz, dh = (torch.randn((n, 2048), device="cuda").to(torch.bfloat16) for _ in range(4))

    def step():
        _, _, s = layer.forward(x, r, starts, a.tokens)
        return layer.backward(s, dz, dh)

    step()
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    for _ in range(10):
        step()
    t1.record()
    torch.cuda.synchronize()
    print(f"forward and backward of {a.batch} x {a.tokens} tokens: {t0.elapsed_time(t1) / 10:.3f} ms")
    cache = layer.cache(a.batch, a.tokens + 1)
    at = torch.arange(a.batch, device="cuda") * a.tokens
    whole, _, _ = layer.forward(x, r, starts, a.tokens)
    few = min(a.tokens, 64)
    for i in range(few):
        z, _ = layer.token(x[at + i], r[at + i], cache)
    off = float((z.float() - whole[at + few - 1].float()).norm() / z.float().norm())
    print(f"token by token, {few} of them, the last one's output differs from the whole sequence's by {off:.2e}")


if __name__ == "__main__":
    main()
