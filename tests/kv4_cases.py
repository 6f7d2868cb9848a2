"""Requests, caches and expected results shared by the tests of the key/value cache in 4 bits."""
from __future__ import annotations

import torch

from oracle import kv4_oracle as orc


def half_step(dtype) -> float:
    """Largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


class Requests:
    """A batch of requests whose keys and values stand in a cache: the rows as they were written (CPU), the block table in
    any order of blocks, everything else of the cache filled with ``junk`` bytes (255: NaN scales, codes of 6)."""

    def __init__(self, device, lens, new, Hq, Hkv, D, bs=64, dtype=torch.bfloat16, seed=0, pad=0, junk=255, extra=2, amp=1.0):
        from gemma_triton_flash_attn_amd import kv4

        g = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.Hq, self.Hkv, self.D, self.bs, self.dtype = lens, new, Hq, Hkv, D, bs, dtype
        need = [-(-n // bs) for n in lens]
        blocks = sum(need) + 3
        order = torch.randperm(blocks, generator=g).tolist()
        width = max(max(need), 1) + extra
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for c in range(n):
                table[b, c] = order.pop()
        self.table = table.to(device)
        self.cache = kv4.allocate(blocks, Hkv, D, bs, dtype, device)
        self.cache.codes.fill_(junk)
        self.cache.scales.fill_(junk)
        self.k = [(torch.randn(Hkv, n, D, generator=g) * amp).to(dtype) for n in lens]
        self.v = [torch.randn(Hkv, n, D, generator=g).to(dtype) for n in lens]
        T = sum(new)
        self.T = T + pad
        self.q = torch.randn(1, Hq, self.T, D, generator=g).to(dtype)
        self.cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=device)
        self.lens_dev = torch.tensor(lens, dtype=torch.int32, device=device)
        self.device = device

    def slots(self, b):
        j = torch.arange(self.lens[b])
        t = self.table.cpu()[b].long()
        return t[j // self.bs] * self.bs + j % self.bs

    def store(self):
        from gemma_triton_flash_attn_amd import kv4

        for b, n in enumerate(self.lens):
            if n:
                kv4.write(self.cache, self.k[b][None].to(self.device), self.v[b][None].to(self.device),
                          self.slots(b).to(self.device))
        return self

    def attend(self, **kw):
        from gemma_triton_flash_attn_amd import kv4

        return kv4.attention(self.q.to(self.device), self.cache, self.table, self.lens_dev, self.cu, **kw)

    def expected(self, causal=True, window=0, scale=None, softcap=0.0, held=None):
        """(o, bound): float64 (Hq, T, D); ``bound`` is what the kernel's roundings can add up to, element by element."""
        o = torch.zeros(self.Hq, self.T, self.D, dtype=torch.float64)
        bound = torch.zeros_like(o)
        t = 0
        sc = self.D ** -0.5 if scale is None else scale
        for b, (n, m) in enumerate(zip(self.lens, self.new)):
            if m:
                k, v = orc.rounded(self.k[b]), orc.rounded(self.v[b])
                q = self.q[0, :, t:t + m]
                ob, w = orc.attend(q, k, v, n, causal, window, sc, softcap, None if held is None else held[b])
                o[:, t:t + m] = ob
                # p and o are each rounded to the type once, and the row sum is that of the rounded p: with p_j (1 + e_j),
                # |e_j| <= u, the numerator moves by at most u sum p |v| (the weight), the sum by at most u of itself, the
                # quotient so by at most u (weight + |o|) to first order, and its rounding adds u |o|. A p below the
                # type's normal range is off by half its smallest step instead. Scores are 32-bit sums of D products,
                # each rounding at most 2^-24 of the sum of magnitudes so far; a shift of a score by x moves p and
                # the row sum by x each; exp2 and tanh are good to 2^-22 (tanh times the cap).
                u = half_step(self.dtype)
                top = lambda x: torch.nan_to_num(x.double(), 0.0, 0.0, 0.0).abs()  # noqa: E731
                mag = float((top(q).amax((0, 1)) * top(k).amax((0, 1))).sum() * sc) if n else 0.0
                shift = self.D * 2.0 ** -24 * mag + 2.0 ** -21 + softcap * 2.0 ** -22
                tiny = n * torch.finfo(self.dtype).smallest_normal * u * (float(top(v).max()) if n else 0.0)
                bound[:, t:t + m] = (u + 2 * shift) * w + 2 * u * ob.abs() + 4 * u * u * w + tiny + 1e-30
            t += m
        return o, bound


def check(got, want, bound):
    got = got[0].double().cpu()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    off = torch.where(nan, torch.zeros_like(want), (got - want).abs() - bound * 1.001)
    assert float(off.max()) <= 0, f"off by {float((got - want).abs()[~nan].max()):.3g}, past the bound by {float(off.max()):.3g}"
