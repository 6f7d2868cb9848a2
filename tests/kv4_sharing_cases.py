"""Pools, tables and requests with something in common, shared by the tests of the cache's pages, prefixes and drafts."""
from __future__ import annotations

import torch

from kv4_cases import Requests

LAYERS = [(1, 256), (2, 64), (1, 512), (3, 128)]  # KV heads, head dim


class Pool:
    """Caches of random bytes, a block table over them with blocks that several rows hold, and a free list."""

    def __init__(self, device, lens, bs=64, spare=6, layers=LAYERS[:2], common=0, seed=0, extra=2, missing=0.0, width=None, gap=0):
        from gemma_triton_flash_attn_amd import kv4

        g = torch.Generator().manual_seed(seed)
        self.bs, self.lens, self.device = bs, list(lens), device
        need = [-(-max(n, 0) // bs) for n in lens]
        width = max(max(need), 1) + extra if width is None else width
        names, nxt = [], 0
        first = list(range(min(common, max(need))))
        nxt = len(first)
        for n in need:
            row = first[:n]
            row += range(nxt, nxt + n - len(row))
            nxt = max(nxt, row[-1] + 1 if row else 0)
            names.append(row[:width])
        self.live = nxt
        self.blocks = max(1, nxt + spare)
        order = torch.randperm(self.blocks, generator=g).tolist()
        t = torch.randint(-3, self.blocks + 5, (len(lens), width + gap), generator=g, dtype=torch.int32)  # junk where nothing is held
        for b, row in enumerate(names):
            for c, x in enumerate(row):
                t[b, c] = order[x]
                if float(torch.rand((), generator=g)) < missing:
                    t[b, c] = -1 if c % 2 else self.blocks + 7
        self.table = t.to(device)[:, :width]
        self.free = torch.tensor(order, dtype=torch.int32, device=device)
        self.used = torch.tensor([nxt], dtype=torch.int32, device=device)
        self.lens_dev = torch.tensor(self.lens, dtype=torch.int32, device=device)
        self.caches = [kv4.allocate(self.blocks, h, d, bs, torch.bfloat16, device) for h, d in layers]
        for c in self.caches:
            c.codes.random_(0, 256)
            c.scales.random_(0, 256)
        self.before = [(c.codes.clone(), c.scales.clone()) for c in self.caches]

    def lists(self):
        return self.table.tolist(), self.lens, self.free.tolist(), int(self.used)

    def check_bytes(self, pairs):
        """Every cache is what it was, but for the destinations of the pairs."""
        for c, (codes, scales) in zip(self.caches, self.before):
            if pairs:
                src, dst = torch.tensor(pairs, device=self.device).t()
                codes[dst], scales[dst] = codes[src].clone(), scales[src].clone()
            assert torch.equal(c.codes, codes) and torch.equal(c.scales, scales)


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


class Answers(Requests):
    """Requests of which neighbours begin with the same blocks: ``groups`` lists (requests, common tokens)."""

    def __init__(self, device, lens, new, Hq, Hkv, D, groups, **kw):
        super().__init__(device, lens, new, Hq, Hkv, D, **kw)
        t, b = self.table.cpu(), 0
        for n, common in groups:
            for i in range(b + 1, b + n):
                t[i, : common // self.bs] = t[b, : common // self.bs]
                whole = min(common // self.bs * self.bs, lens[i], lens[b])
                self.k[i][:, :whole] = self.k[b][:, :whole]
                self.v[i][:, :whole] = self.v[b][:, :whole]
            b += n
        assert b == len(lens)
        self.table = t.to(device)

    def share(self, least=64):
        from gemma_triton_flash_attn_amd import kv4

        return kv4.share(self.table, self.lens_dev, self.cu, block_size=self.bs, least=least)
