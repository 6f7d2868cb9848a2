"""The operators of requests with something in common as a server runs them together: prompts, answers forked from them, drafted
tokens attended, verified and taken back, beams, requests that leave, a compacted pool. Every output against the tokens' own history."""
from __future__ import annotations

import random

import pytest
import torch

from kv4_cases import check, half_step
from oracle import kv4_oracle as orc

pytestmark = pytest.mark.gpu

LAYERS = [(8, 2, 128), (8, 1, 256)]  # query heads, KV heads, head dim


class Server:
    """Requests over one pool. Keys and values are functions of (layer, token history), so that what is read back tells whose
    blocks were read: every request keeps the rows of its tokens."""

    def __init__(self, device, blocks=160, bs=32, width=24, dtype=torch.bfloat16):
        from gemma_triton_flash_attn_amd import kv4

        self.g = torch.Generator().manual_seed(blocks)
        self.device, self.bs, self.dtype, self.blocks, self.width = device, bs, dtype, blocks, width
        self.caches = [kv4.allocate(blocks, hkv, D, bs, dtype, device) for _, hkv, D in LAYERS]
        for c in self.caches:
            c.codes.fill_(255)
            c.scales.fill_(255)
        self.free = torch.randperm(blocks, generator=self.g).to(torch.int32).to(device)
        self.used = self.ints([0])
        self.table = torch.full((0, width), -1, dtype=torch.int32, device=device)
        self.lens = self.ints([])
        self.rows = []  # of each request: per layer (k, v), (Hkv, tokens, D)

    def ints(self, v):
        return torch.tensor(v, dtype=torch.int32, device=self.device)

    def randn(self, *s):
        return torch.randn(*s, generator=self.g).to(self.dtype)

    def join(self, n):
        """New, empty requests."""
        self.table = torch.cat([self.table, torch.full((n, self.width), -1, dtype=torch.int32, device=self.device)])
        self.lens = torch.cat([self.lens, self.ints([0] * n)])
        self.rows += [[(torch.zeros(hkv, 0, D, dtype=self.dtype),) * 2 for _, hkv, D in LAYERS] for _ in range(n)]

    def step(self, new, shared=True, pad=2, least=32):
        """New tokens for each request through all layers, checked; returns the plan."""
        from gemma_triton_flash_attn_amd import kv4

        T = sum(new) + pad
        p = kv4.plan(self.lens, self.ints(new), self.table, self.free, self.used, block_size=self.bs, tokens=T)
        s = kv4.share(self.table, p.lens, p.cu, block_size=self.bs, least=least) if shared else None
        for i, (cache, (hq, hkv, D)) in enumerate(zip(self.caches, LAYERS)):
            q, k, v = (self.randn(1, h, T, D) for h in (hq, hkv, hkv))
            kv4.write(cache, k.to(self.device), v.to(self.device), p.slots)
            o = kv4.attention(q.to(self.device), cache, self.table, p.lens, p.cu, max_new=max(max(new), 1), shared=s, apart=True)
            t = 0
            for b, n in enumerate(new):
                kb, vb = self.rows[b][i]
                kb, vb = torch.cat([kb, k[0, :, t:t + n]], 1), torch.cat([vb, v[0, :, t:t + n]], 1)
                self.rows[b][i] = (kb, vb)
                if n:
                    kk, vv = orc.rounded(kb), orc.rounded(vb)
                    want, w = orc.attend(q[0, :, t:t + n], kk, vv, kk.shape[1])
                    # one rounding of p, in the sum too, one of o, 32-bit score sums (kv4_cases.Requests.expected)
                    u = half_step(self.dtype)
                    mag = float((q.double().abs().amax((0, 1, 2)) * kk.abs().amax((0, 1))).sum() * D ** -0.5)
                    bound = (u + 2 * (D * 2.0 ** -24 * mag + 2.0 ** -21)) * w + 2 * u * want.abs() + 4 * u * u * w + 1e-30
                    check(o[:, :, t:t + n], want, bound)
                t += n
            assert not o[:, :, t:].any()
        self.lens, self.used = p.lens, p.used
        assert self.lens.tolist() == [r[0][0].shape[1] for r in self.rows]
        return p

    def fork(self, parents=None, keep=None):
        from gemma_triton_flash_attn_amd import kv4

        f = kv4.fork(self.caches, self.table, self.lens, self.free, self.used, parents=None if parents is None else self.ints(parents),
                     keep=keep)
        parents = range(len(self.rows)) if parents is None else parents
        self.table, self.lens, self.used = f.table, f.lens, f.used
        n = f.lens.tolist()
        self.rows = [[(k[:, :m].clone(), v[:, :m].clone()) for k, v in self.rows[p]] for p, m in zip(parents, n)]
        self.pool()

    def compact(self):
        from gemma_triton_flash_attn_amd import kv4

        self.table, self.used = kv4.compact(self.caches, self.table, self.lens, self.free)
        assert int(self.table.max()) < int(self.used)
        self.pool()

    def pool(self):
        """No block is lost or handed out twice: what requests hold and what is free are the pool."""
        held = {x for row, n in zip(self.table.tolist(), self.lens.tolist()) for x in row[: -(-n // self.bs)]}
        used = int(self.used)
        assert len(held) == used and sorted(held | set(self.free.tolist()[used:])) == list(range(self.blocks))


def test_answers_drafts_and_beams(device):
    from gemma_triton_flash_attn_amd import kv4

    r = random.Random(0)
    s = Server(device)
    s.join(3)
    s.step([150, 64, 33])                                # three prompts
    s.fork([0] * 6 + [1] * 3 + [2])                      # answers to them
    for _ in range(2):
        s.step([1] * 10)
    for turn in range(4):                                # drafted tokens, some of them not accepted
        new = [r.choice([1, 3, 5]) for _ in range(10)]
        p = s.step(new)
        T, V = p.slots.shape[0], 50
        target, draft = (torch.softmax(torch.randn(T, V, generator=s.g), -1).to(device) for _ in range(2))
        tokens = torch.multinomial(draft.cpu(), 1, generator=s.g)[:, 0].to(device)
        v = kv4.verify(target, draft, tokens, torch.rand(T, generator=s.g).to(device), torch.rand(10, generator=s.g).to(device), p.lens, p.cu)
        assert (v.lens >= p.lens - p.cu.diff() + 1).all()
        s.fork(keep=v.lens)
    s.fork([1, 1, 4, 0, 0, 0, 8, 9, 9, 9])               # beams: some dropped, some go on twice
    s.step([1] * 10)
    s.fork([6, 7, 8, 9, 0, 1])                           # requests leave, others change places
    s.compact()
    s.join(1)
    s.step([1, 1, 2, 1, 1, 0, 90], shared=False)         # a prompt joins
    s.step([1] * 7)
    s.fork([-1] * 7)                                     # all leave
    assert s.used.tolist() == [0]


def test_a_captured_turn(device):
    """One turn (plan, write, share, attention, verify, fork) captured and replayed with everything in place, against eager turns."""
    from gemma_triton_flash_attn_amd import kv4

    def build():
        s = Server(device, blocks=90)
        s.join(2)
        s.step([100, 40])
        s.fork([0, 0, 0, 1, 1])
        return s

    R, T, V = 5, 11, 40
    g = torch.Generator().manual_seed(1)
    draws = []
    for _ in range(4):
        new = [1, 2, 3, 3, 2]
        random.Random(len(draws)).shuffle(new)
        draws.append(dict(new=torch.tensor(new, dtype=torch.int32), q=[torch.randn(1, hq, T, D, generator=g) for hq, _, D in LAYERS],
                          k=[torch.randn(1, h, T, D, generator=g) for _, h, D in LAYERS], target=torch.rand(T, V, generator=g),
                          draft=torch.rand(T, V, generator=g), tokens=torch.randint(0, V, (T,), generator=g),
                          accept=torch.rand(T, generator=g), sample=torch.rand(R, generator=g)))

    def turn(s, x):
        p = kv4.plan(s.lens, x["new"], s.table, s.free, s.used, block_size=s.bs, tokens=T)
        shared = kv4.share(s.table, p.lens, p.cu, block_size=s.bs, least=32)
        outs = []
        for cache, q, k in zip(s.caches, x["q"], x["k"]):
            kv4.write(cache, k, k, p.slots)
            outs.append(kv4.attention(q, cache, s.table, p.lens, p.cu, max_new=3, shared=shared, apart=True))
        v = kv4.verify(x["target"], x["draft"], x["tokens"], x["accept"], x["sample"], p.lens, p.cu)
        f = kv4.fork(s.caches, s.table, p.lens, s.free, p.used, keep=v.lens)
        s.table.copy_(f.table)
        s.lens.copy_(f.lens)
        s.used.copy_(f.used)
        return outs + [v.tokens, v.accepted]

    def on_device(x):
        half = lambda t: t.to(device, torch.bfloat16)  # noqa: E731
        return {k: [half(t) for t in v] if isinstance(v, list) else v.to(device) for k, v in x.items()}

    eager, s = build(), build()
    for c, d in zip(eager.caches, s.caches):
        d.codes.copy_(c.codes)
        d.scales.copy_(c.scales)
    for a, b in ((s.table, eager.table), (s.lens, eager.lens), (s.used, eager.used), (s.free, eager.free)):
        a.copy_(b)
    x = on_device(draws[0])
    keep = [t.clone() for t in (s.table, s.lens, s.used, s.free)] + [t.clone() for c in s.caches for t in (c.codes, c.scales)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        turn(s, x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = turn(s, x)
    for a, b in zip([s.table, s.lens, s.used, s.free] + [t for c in s.caches for t in (c.codes, c.scales)], keep):
        a.copy_(b)
    for d in draws:
        y = on_device(d)
        for k, v in y.items():
            for a, b in zip(x[k], v) if isinstance(v, list) else ((x[k], v),):
                a.copy_(b)
        graph.replay()
        seen = [t.clone() for t in got]
        want = turn(eager, y)
        assert all(torch.equal(a, b) for a, b in zip(seen, want))
        assert torch.equal(s.table, eager.table) and torch.equal(s.lens, eager.lens) and torch.equal(s.free, eager.free)
