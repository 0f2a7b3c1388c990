"""The paged cache's operators in float64 and plain loops, for the tests."""
from __future__ import annotations

import math

import torch

BF = torch.bfloat16
E4 = torch.float8_e4m3fn


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def starts_of(lens, device):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return ints(out, device)


def attend(q, k, v, scale, visible=None):
    """softmax(q k^T scale) v in float64 -> (out, weight of |v|, lse); rows that see no key are zero, lse -inf.
    q [R, D], k, v [M, D]; visible bool [R, M]."""
    s = (q.double() @ k.double().t().contiguous()) * scale
    if visible is not None:
        s = s.masked_fill(~visible, -math.inf)
    if s.shape[1] == 0:
        z = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
        return z, z, torch.full((q.shape[0],), -math.inf, dtype=torch.float64, device=q.device)
    lse = torch.logsumexp(s, -1)
    p = torch.where((lse == -math.inf)[:, None], torch.zeros_like(s), torch.softmax(s, -1))
    # a key without weight has no part, whatever its value
    vd = v.double()
    if visible is not None:
        vd = torch.where(visible.any(0)[:, None], vd, torch.zeros_like(vd))
    return p @ vd, p @ vd.abs(), lse


def prompt_reference(q, k, v, rows, keys, causal, scale=None):
    """Packed prompts with ``rows`` and ``keys`` each: (out, weight of |v|) [Tq, H, D] and lse [H, Tq]."""
    T, H, D = q.shape
    G = H // k.shape[1]
    out = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    lse = torch.full((H, T), -math.inf, dtype=torch.float64, device=q.device)
    r = m = 0
    for n, length in zip(rows, keys):
        vis = None
        if causal:
            i = torch.arange(n, device=q.device)[:, None] + length - n
            vis = torch.arange(length, device=q.device)[None] <= i
        for h in range(H):
            o, a, ls = attend(q[r:r + n, h], k[m:m + length, h // G], v[m:m + length, h // G],
                              scale or 1 / math.sqrt(D), vis)
            out[r:r + n, h], mag[r:r + n, h], lse[h, r:r + n] = o, a, ls
        r, m = r + n, m + length
    return out, mag, lse


def assert_attention_close(got, out, mag, what="", weight=2 ** -8):
    """|error| <= ``weight`` (P to bf16, half a step of each weight; two bf16 parts: 2^-16) + 2^-8 (the result to
    bf16) of the weighted magnitudes, and 2^-12 for the float32 scores (128 products, exp2 of a sum whose
    magnitude stays below 2^7)."""
    err = (got.double() - out).abs()
    bound = mag * (weight + 2 ** -8 + 2 ** -12) + 1e-30
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: error {worst:.2f} of its bound"


def assert_lse_close(got, ref, what=""):
    """lse from float32 scores below 2^7 in base 2 (a few roundings of 2^-24 * 2^7 each) and a sum of rounded exps."""
    assert torch.equal(got == -math.inf, ref == -math.inf), what
    fin = ref != -math.inf
    err = (got.double()[fin] - ref[fin]).abs()
    assert err.numel() == 0 or err.max().item() <= 2e-4, f"{what}: lse off by {err.max().item()}"


class Cache:
    """Pools [blocks, block, heads, D] (views; ``layout`` "heads": a head's tokens together in memory, "tokens": a
    token's heads together) and tables of requests with ``lens`` tokens of random values."""

    def __init__(self, lens, Hk, D, block, kv, device, seed=0, layout="heads", spare=3, width=None):
        g = torch.Generator().manual_seed(seed)
        held = [-(-n // block) for n in lens]
        self.n = sum(held) + spare
        self.lens, self.block, self.kv = list(lens), block, kv
        perm = torch.randperm(self.n, generator=g)
        width = width or max(1, max(held, default=1))
        tables = torch.full((len(lens), width), -7, dtype=torch.int32)
        at = 0
        for b, h in enumerate(held):
            tables[b, :h] = perm[at:at + h].int()
            at += h
        self.tables, self.free = tables.to(device), perm[at:].int().to(device)
        shape = (self.n, Hk, block, D) if layout == "heads" else (self.n, block, Hk, D)
        view = (lambda t: t.permute(0, 2, 1, 3)) if layout == "heads" else (lambda t: t)
        self.k_scales = self.v_scales = None
        if kv == "bf16":
            self.k, self.v = (view(torch.randn(shape, generator=g).to(BF).to(device)) for _ in range(2))
        else:
            self.k, self.v = (view((torch.randn(shape, generator=g) * 120).clamp(-448, 448).to(E4).to(device))
                              for _ in range(2))
            sc = [(torch.rand(self.n, Hk, block, generator=g) + 0.5) / 120 for _ in range(2)]
            self.k_scales, self.v_scales = (s.to(device).permute(0, 2, 1) for s in sc)
        self.lens_t = ints(list(lens), device)

    def dense(self, b, n=None):
        """Request b's K and V [n, heads, D] in float64; entries outside the pool are left out."""
        n = self.lens[b] if n is None else n
        row = self.tables[b].tolist()
        at = [(row[p // self.block], p % self.block) for p in range(n)]
        at = [(i, o) for i, o in at if 0 <= i < self.n]
        i = torch.tensor([a for a, _ in at], dtype=torch.long, device=self.k.device)
        o = torch.tensor([a for _, a in at], dtype=torch.long, device=self.k.device)
        out = []
        for pool, scales in ((self.k, self.k_scales), (self.v, self.v_scales)):
            x = pool.view(torch.uint8)[i, o].view(E4).double() if self.kv == "fp8" else pool[i, o].double()
            out.append(x * scales[i, o].double()[..., None] if scales is not None else x)
        return out

    def reference(self, q, scale=None):
        B, H, D = q.shape
        out = torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
        mag = torch.zeros_like(out)
        lse = torch.full((B, H), -math.inf, dtype=torch.float64, device=q.device)
        for b in range(B):
            k, v = self.dense(b)
            G = H // k.shape[1]
            for h in range(H):
                o, a, ls = attend(q[b, h][None], k[:, h // G], v[:, h // G], scale or 1 / math.sqrt(D))
                out[b, h], mag[b, h], lse[b, h] = o[0], a[0], ls[0]
        return out, mag, lse


def grow_reference(tables, lens, new, free, top, block, tokens):
    """The allocation request by request -> (tables, slots, positions, starts, lens, top)."""
    tables = [list(r) for r in tables]
    slots, positions, starts, out = [], [], [0], []
    for b, (p, n) in enumerate(zip(lens, new)):
        for j in range(-(-p // block), -(-(p + n) // block)):
            top -= 1
            tables[b][j] = free[top]
        slots += [tables[b][x // block] * block + x % block for x in range(p, p + n)]
        positions += range(p, p + n)
        starts.append(starts[-1] + n)
        out.append(p + n)
    behind = tokens - len(slots)
    return tables, slots + [-1] * behind, positions + [0] * behind, starts, out, top
