"""The cache operators as a server runs them: prompts in parts and single tokens through several layers, captured and replayed
steps, other streams, torch.compile."""
from __future__ import annotations

import pytest
import torch

from kv4_cases import Requests, check, half_step
from oracle import kv4_oracle as orc

pytestmark = pytest.mark.gpu


class Server:
    """Requests that take blocks from one pool; every token's q, k and v are drawn once and kept for the oracle."""

    def __init__(self, device, B, layers, blocks=64, bs=32, width=12, dtype=torch.bfloat16):
        from gemma_triton_flash_attn_amd import kv4

        self.g = torch.Generator().manual_seed(B)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
        self.device, self.B, self.layers, self.bs, self.dtype = device, B, layers, bs, dtype
        self.table = torch.full((B, width), -1, dtype=torch.int32, device=device)
        self.free = torch.randperm(blocks, generator=self.g).to(torch.int32).to(device)
        self.used, self.lens = ints([0]), ints([0] * B)
        self.caches = [kv4.allocate(blocks, hkv, D, bs, dtype, device) for _, hkv, D, _ in layers]
        for c in self.caches:
            c.codes.fill_(255)
            c.scales.fill_(255)
        self.k = [[torch.zeros(hkv, 0, D, dtype=dtype) for _ in range(B)] for _, hkv, D, _ in layers]
        self.v = [[torch.zeros(hkv, 0, D, dtype=dtype) for _ in range(B)] for _, hkv, D, _ in layers]

    def rows(self, T):
        """q, k, v of a step, one (1, H, T, D) triple per layer."""
        return [tuple(torch.randn(1, h, T, D, generator=self.g).to(self.dtype) for h in (hq, hkv, hkv))
                for hq, hkv, D, _ in self.layers]

    def step(self, new, rows, T):
        from gemma_triton_flash_attn_amd import kv4

        fresh = torch.tensor(new, dtype=torch.int32, device=self.device)
        p = kv4.plan(self.lens, fresh, self.table, self.free, self.used, block_size=self.bs, tokens=T)
        outs = []
        for cache, (q, k, v), (_, _, _, window) in zip(self.caches, rows, self.layers):
            q, k, v = (x.to(self.device) for x in (q, k, v))
            kv4.write(cache, k, v, p.slots)
            outs.append(kv4.attention(q, cache, self.table, p.lens, p.cu, max_new=max(max(new), 1), slide_size=window))
        self.lens, self.used = p.lens, p.used
        return outs

    def check(self, new, rows, outs):
        for i, ((q, k, v), o, (_, _, D, window)) in enumerate(zip(rows, outs, self.layers)):
            t = 0
            for b, n in enumerate(new):
                self.k[i][b] = torch.cat([self.k[i][b], k[0, :, t:t + n]], 1)
                self.v[i][b] = torch.cat([self.v[i][b], v[0, :, t:t + n]], 1)
                if n:
                    kk, vv = orc.rounded(self.k[i][b]), orc.rounded(self.v[i][b])
                    want, w = orc.attend(q[0, :, t:t + n], kk, vv, kk.shape[1], True, window)
                    # one rounding of p, in the sum too, one of o, 32-bit score sums (kv4_cases.Requests.expected)
                    u = half_step(self.dtype)
                    mag = float((q.double().abs().amax((0, 1, 2)) * kk.abs().amax((0, 1))).sum() * D ** -0.5)
                    bound = (u + 2 * (D * 2.0 ** -24 * mag + 2.0 ** -21)) * w + 2 * u * want.abs() + 4 * u * u * w + 1e-30
                    check(o[:, :, t:t + n], want, bound)
                t += n
            assert not o[:, :, t:].any()


LAYERS = [(8, 1, 256, 40), (8, 1, 512, 0), (4, 2, 128, 0)]


def test_prompts_and_tokens(device):
    """Four requests: a long prompt in parts, short ones, single tokens in between, one that joins late; padded steps."""
    s = Server(device, 4, LAYERS)
    for new in ([100, 7, 0, 33], [90, 1, 64, 1], [1, 1, 1, 1], [1, 0, 1, 1], [40, 1, 1, 1], [1, 1, 1, 1]):
        T = sum(new) + 5
        rows = s.rows(T)
        s.check(new, rows, s.step(new, rows, T))
    assert s.lens.tolist() == [233, 11, 68, 38]


def test_a_captured_step(device):
    """One graph of a decoding step (plan, write, attention) replayed while lengths grow in device memory, another over the same
    caches and tables, eager work in between: the results of eager steps, bit for bit."""
    from gemma_triton_flash_attn_amd import kv4

    def build(graph):
        s = Server(device, 3, LAYERS)
        new0 = [50, 3, 31]
        s.step(new0, s.rows(sum(new0)), sum(new0))
        q, k, v = ([torch.zeros(1, h, 4, D, dtype=s.dtype, device=device) for h, D in hd]
                   for hd in ([(hq, D) for hq, _, D, _ in LAYERS], [(hk, D) for _, hk, D, _ in LAYERS], [(hk, D) for _, hk, D, _ in LAYERS]))
        fresh = torch.zeros(3, dtype=torch.int32, device=device)
        outs = [torch.zeros_like(x) for x in q]

        def body(layers):
            p = kv4.plan(s.lens, fresh, s.table, s.free, s.used, block_size=s.bs, tokens=4)
            for i in layers:
                kv4.write(s.caches[i], k[i], v[i], p.slots)
                outs[i].copy_(kv4.attention(q[i], s.caches[i], s.table, p.lens, p.cu, max_new=1, slide_size=LAYERS[i][3]))
            return p

        def last(layers):
            p = body(layers)
            s.lens.copy_(p.lens)
            s.used.copy_(p.used)

        keep = (s.lens.clone(), s.used.clone())
        runs = [lambda: body([0]), lambda: last([1, 2])]
        if graph:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):  # warm-up, with nothing new
                for r in runs:
                    r()
            torch.cuda.current_stream().wait_stream(side)
            graphs = []
            for r in runs:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    r()
                graphs.append(g)
            runs = [g.replay for g in graphs]
            s.lens.copy_(keep[0])
            s.used.copy_(keep[1])
        seen = []
        gen = torch.Generator().manual_seed(9)
        for step in range(5):
            fresh.copy_(torch.tensor([1, step % 2, 1], dtype=torch.int32))
            for group in (q, k, v):
                for x in group:
                    x.copy_(torch.randn(x.shape, generator=gen))
            for r in runs:
                r()
            noise = torch.randn(1 << 20, device=device).sum()
            seen.append([o.clone() for o in outs])
            assert torch.isfinite(noise)
            torch.cuda.synchronize()
        return seen, s.lens.tolist(), s.table.tolist()

    eager, graph = build(False), build(True)
    assert eager[1:] == graph[1:]
    assert all(torch.equal(a, b) for x, y in zip(eager[0], graph[0]) for a, b in zip(x, y))


def test_other_streams(device):
    """Calls on a stream of their own, two at once over the same cache: the results of the default stream."""
    r = Requests(device, [700, 90, 333], [1, 1, 1], 8, 2, 256).store()
    big = Requests(device, [700, 300], [200, 300], 8, 2, 256, seed=1).store()
    want, want_big = r.attend(), big.attend()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (a, b):
        s.wait_stream(torch.cuda.current_stream())
    got, got_big = [], []
    for _ in range(4):
        with torch.cuda.stream(a):
            got.append(r.attend())
            got_big.append(big.attend())
        with torch.cuda.stream(b):
            got_big.append(big.attend())
            got.append(r.attend())
    for s in (a, b):
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, want) for x in got) and all(torch.equal(x, want_big) for x in got_big)


def test_compiled_step(device):
    """A step under torch.compile, one graph: the eager results."""
    from gemma_triton_flash_attn_amd import kv4

    def step(q, k, v, codes, scales, lens, new, table, free, used):
        cache = kv4.Cache(codes, scales, torch.bfloat16)
        p = kv4.plan(lens, new, table, free, used, block_size=32, tokens=6)
        kv4.write(cache, k * 2, v, p.slots)
        o = kv4.attention(q, cache, table, p.lens, p.cu, max_new=4, slide_size=20)
        back, _ = kv4.read(cache, p.slots)
        return o * 0.5, back, p.lens, p.used

    g = torch.Generator().manual_seed(3)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731

    def inputs():
        g.manual_seed(3)
        q, k, v = (torch.randn(1, h, 6, 128, generator=g).to(device, torch.bfloat16) for h in (4, 2, 2))
        c = kv4.allocate(8, 2, 128, 32, torch.bfloat16, device)
        c.codes.zero_()
        c.scales.fill_(127)
        return [q, k, v, c.codes, c.scales, ints([40, 31]), ints([4, 1]), ints([[5, 1, -1], [0, -1, -1]]), ints([2, 3, 4]), ints([0])]

    a, b = inputs(), inputs()
    want = step(*a)
    got = torch.compile(step, fullgraph=True, dynamic=False)(*b)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    assert all(torch.equal(a[i], b[i]) for i in (3, 4, 7))  # the cache and the table, written in place


def test_registered_ops(device):
    """torch.library's own checks of the ops, and the same results under a dispatch mode."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from gemma_triton_flash_attn_amd import kv4

    r = Requests(device, [50, 90], [2, 1], 4, 2, 64, pad=1).store()
    args = (r.q.to(device), r.cache.codes, r.cache.scales, True, r.table, r.lens_dev, r.cu, 2, True, 0, 0.125, 0.0)
    torch.library.opcheck(torch.ops.gfa.kv4_attention, args)
    slots = r.slots(0).to(device)
    torch.library.opcheck(torch.ops.gfa.kv4_read, (r.cache.codes, r.cache.scales, True, slots))

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    want = r.attend()
    with Seen() as seen:
        got = kv4.attention(args[0], r.cache, r.table, r.lens_dev, r.cu)
    assert torch.equal(got, want) and any("kv4_attention" in n for n in seen.names)


def test_no_gradient(device):
    from gemma_triton_flash_attn_amd import kv4

    r = Requests(device, [50], [1], 4, 2, 64).store()
    q = r.q.to(device).requires_grad_(True)
    with pytest.raises(NotImplementedError):
        kv4.attention(q, r.cache, r.table, r.lens_dev)
    with torch.no_grad():
        o = kv4.attention(q, r.cache, r.table, r.lens_dev)
    assert not o.requires_grad and torch.equal(o, r.attend())


def test_the_prompt_through_the_forward_kernel(device):
    """A first prompt's attention over the values the cache keeps, by the framework's prompt kernel on kv4.read's rows, and over
    the cache: the same within their roundings."""
    import gemma_triton_flash_attn_amd as gfa

    r = Requests(device, [300], [300], 8, 2, 256).store()
    k, v = gfa.kv4.read(r.cache, r.slots(0).to(device))
    o = gfa.attention_flash_gqa(r.q.to(device), k, v, causal=True, slide_size=100)
    want, bound = r.expected(window=100)
    check(r.attend(slide_size=100), want, bound)
    check(o, want, bound)


def test_inference_mode(device):
    r = Requests(device, [50, 90], [2, 1], 4, 2, 64, pad=1).store()
    want = r.attend()
    with torch.inference_mode():
        assert torch.equal(r.attend(), want)
        s = Server(device, 2, LAYERS)
        rows = s.rows(45)
        outs = s.step([40, 3], rows, 45)
        assert s.lens.is_inference() and outs[0].is_inference()
    s.check([40, 3], rows, outs)
