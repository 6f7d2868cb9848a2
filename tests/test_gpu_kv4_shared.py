"""What requests have in common, and attention that computes it once: against the definition, and against the plain call."""
from __future__ import annotations

import random

import pytest
import torch

from kv4_cases import check
from kv4_sharing_cases import Answers, ints
from oracle import kv4_sharing_oracle as orc

pytestmark = pytest.mark.gpu


# ---- share ----

def same_as_defined(table, lens, cu, bs, least, device):
    from gemma_triton_flash_attn_amd import kv4

    t = table if isinstance(table, torch.Tensor) else ints(table, device)
    got = kv4.share(t, ints(lens, device), ints(cu, device), block_size=bs, least=least)
    want = orc.share(t.tolist(), lens, cu, bs, least)
    assert [x.tolist() for x in got] == [list(x) for x in want]
    return want


def test_share_by_hand(device):
    table = [[5, 6, 7, 1], [5, 6, 7, 2], [5, 6, 8, 3], [9, 6, 7, 1], [9, 4, 0, 0]]
    want = same_as_defined(table, [256, 250, 200, 130, 70], [0, 1, 3, 4, 5, 6], 64, 64, device)
    assert want == ([128, 128, 128, 64, 64], [0, 4, 4, 4, 6, 6], [128, 0, 0, 64, 0])
    # a longer least keeps the third apart; the first two share what is full ahead of their new tokens
    want = same_as_defined(table, [256, 250, 200, 130, 70], [0, 1, 3, 4, 5, 6], 64, 129, device)
    assert want == ([192, 192, 0, 0, 0], [0, 3, 3, 4, 5, 6], [192, 0, 0, 0, 0])


@pytest.mark.parametrize("seed", range(12))
def test_share_any(seed, device):
    r = random.Random(seed)
    R, M, bs = r.choice([1, 2, 33, 300]), r.choice([1, 7, 130, 400]), r.choice([32, 64, 1024])
    rows = [[r.randint(-1, 9) for _ in range(M)]]
    for _ in range(R - 1):
        n = r.choice([0, 1, M // 2, M, M])
        rows.append(rows[-1][:n] + [r.randint(-1, 9) for _ in range(M - n)])
    lens = [r.choice([0, 5, M * bs, r.randint(0, M * bs), M * bs + 70]) for _ in range(R)]
    cu = [r.choice([0, 4])]
    for n in lens:
        cu.append(cu[-1] + r.choice([0, 1, 1, 8, min(n, 100)]))
    wide = torch.cat([ints(rows, device), torch.full((R, 3), 7, dtype=torch.int32, device=device)], 1)[:, :M]
    same_as_defined(wide, lens, cu, bs, r.choice([1, bs, 4 * bs, 1 << 40]) if seed else 1, device)


def test_share_many(device):
    """As many requests as a call takes, in groups of 1 to 1500."""
    r = random.Random(3)
    rows, n = [], 0
    while len(rows) < 4096:
        for _ in range(r.choice([1, 2, 30, 1500])):
            rows.append([n, n + 1, r.randint(0, 3)])
        n += 2
    rows = rows[:4096]
    same_as_defined(rows, [r.randint(90, 96) for _ in rows], list(range(4097)), 32, 64, device)


# ---- attention ----

CASES = {
    # groups (requests, common tokens), own tokens of a request (least, most), new tokens, Hq, Hkv, D, bs, dtype
    "d512_few": ([(4, 700)], (1, 90), 1, 8, 1, 512, 64, torch.bfloat16),
    "d512_many": ([(20, 900)], (1, 90), 1, 16, 2, 512, 64, torch.bfloat16),
    "d256_few": ([(2, 1300), (1, 0)], (1, 40), 1, 8, 4, 256, 128, torch.float16),
    "d256_many": ([(30, 640), (3, 2000), (2, 64)], (1, 200), 1, 16, 4, 256, 64, torch.bfloat16),
    "d128_many": ([(40, 2100), (1, 77), (17, 333)], (1, 70), 1, 32, 8, 128, 32, torch.bfloat16),
    "d128_drafts": ([(9, 1500), (1, 10), (2, 700)], (8, 300), 5, 16, 8, 128, 64, torch.float16),
    "d64_many": ([(70, 1111)], (1, 33), 1, 8, 2, 64, 32, torch.bfloat16),
    "d64_drafts": ([(5, 4000), (70, 512)], (3, 50), 3, 15, 5, 64, 64, torch.float16),
    "d512_drafts": ([(7, 1000), (2, 320)], (4, 100), 4, 8, 1, 512, 64, torch.float16),
    "long": ([(3, 20000)], (1, 3000), 1, 8, 2, 128, 256, torch.bfloat16),
}


def answers(name, device, seed=0, pad=0, **kw):
    groups, (lo, hi), new, Hq, Hkv, D, bs, dtype = CASES[name]
    r = random.Random(name)
    lens = [c // bs * bs + r.randint(max(lo, new), hi) for n, c in groups for _ in range(n)]
    return Answers(device, lens, [new] * len(lens), Hq, Hkv, D, groups, bs=bs, dtype=dtype, seed=seed, pad=pad, **kw).store()


def run(a, shared, **kw):
    """With every group's prefix taken apart, whatever that saves, unless kw has it otherwise."""
    return a.attend(**{**dict(max_new=max(a.new), shared=shared, apart=True), **kw})


@pytest.mark.parametrize("name", list(CASES))
def test_against_the_definition(name, device):
    a = answers(name, device, pad=3)
    s = a.share()
    assert int(s.lens.max()) >= 64 and int(s.skip.max()) == int(s.lens.max())
    o = run(a, s)
    want, bound = a.expected()
    check(o, want, bound)
    assert not o[:, :, -3:].any()
    assert torch.equal(o, run(a, s))  # the order of sums is fixed


@pytest.mark.parametrize("name", ["d512_many", "d128_drafts", "d64_drafts", "d256_few"])
def test_masks_and_caps(name, device):
    """Cross attention, soft-capping, a scale; with a window the plain path, bit for bit."""
    a = answers(name, device, seed=1)
    s = a.share()
    for kw in (dict(causal=False), dict(softcap=20.0), dict(scale=0.3, softcap=5.0, causal=False)):
        o = run(a, s, **kw)
        want, bound = a.expected(causal=kw.get("causal", True), softcap=kw.get("softcap", 0.0), scale=kw.get("scale"))
        check(o, want, bound)
    assert torch.equal(run(a, s, slide_size=100), run(a, None, slide_size=100))


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("rows", [16, 17, 32, 33, 64, 65, 128, 129, 260])
def test_rows_of_a_group(D, rows, device):
    """Every form a prefix's rows can take: a row block of 16 and several, half a workgroup whose waves share the keys, whole ones.
    Prefixes of one tile, of an odd number, of one that is split; two groups of different rows side by side, and a request alone."""
    G, Hkv, bs = {17: 1, 33: 3, 65: 5, 129: 3}.get(rows, 4), 4, 32 if rows % 2 else 64
    n = rows // G
    for tiles in (2, 5, 37) if n <= 17 else (2, 11):
        common = -(-tiles * 32 // bs) * bs
        lens = [common + 1 + i % 9 for i in range(n)] + [common + 3, common + 40, 7]
        a = Answers(device, lens, [1] * len(lens), G * Hkv, Hkv, D, [(n, common), (2, common), (1, 0)], bs=bs, seed=rows,
                    dtype=torch.float16 if rows in (33, 129) else torch.bfloat16).store()
        s = a.share(least=32)
        assert s.skip.tolist() == [common] * (n + 2) + [0]
        check(run(a, s), *a.expected())
        if rows in (33, 65):
            check(run(a, s, softcap=10.0), *a.expected(softcap=10.0))


# Requests of a group, by the kernel that takes its prefix: 12 rows the split kernel's, 48 the chunk kernel's with shared keys, 160 its own.
SIZES = [3, 12, 40]


def test_mixed_counts(device):
    """Requests with no new tokens, one, several: in a group, and between groups; max_new unknown or wrong; an empty request."""
    lens, new = [400, 410, 390, 0, 5, 850, 860, 849], [1, 0, 6, 0, 2, 3, 1, 2]
    a = Answers(device, lens, new, 8, 2, 128, [(3, 384), (2, 0), (3, 832)], bs=32, pad=2).store()
    want, bound = a.expected()
    s = a.share()
    assert s.skip.tolist() == [384, 384, 384, 0, 0, 832, 832, 832]
    for kw in (dict(max_new=6), dict(), dict(max_new=1)):
        check(a.attend(shared=s, apart=True, **kw), want, bound)
    q = a.q.to(device)
    assert torch.equal(q.cpu(), a.q)


def test_many_rows_take_the_plain_path(device):
    """A prompt's chunk of each of two answers: bit for bit the call without shared."""
    a = Answers(device, [700, 710], [100, 60], 8, 2, 128, [(2, 512)], bs=64).store()
    assert a.share().lens.tolist() == [512, 0]
    assert torch.equal(run(a, a.share()), run(a, None))


def test_nothing_in_common(device):
    """No group: sums are joined all the same, within the same bound."""
    a = Answers(device, [300, 1000, 64, 1], [1, 1, 1, 1], 8, 2, 128, [(4, 0)], bs=64).store()
    s = a.share()
    assert not s.skip.any() and not s.lens.any()
    check(run(a, s), *a.expected())


@pytest.mark.parametrize("D,Hkv", [(512, 1), (512, 4), (256, 4), (128, 8), (64, 16)])
def test_where_it_pays(D, Hkv, device):
    """The call's own choice, on either side of the line: many requests over a long prefix, few over a short one. In tables too narrow
    to gain anything it is the plain call, bit for bit."""
    a = Answers(device, [2100 + i for i in range(48)] + [90, 70], [1] * 50, 4 * Hkv, Hkv, D, [(48, 2048), (2, 64)], bs=64).store()
    s = a.share()
    assert s.lens.tolist()[0] == 2048 and s.lens.tolist()[48] == 64
    want = a.expected()
    for kw in (dict(), dict(apart=True), dict(apart=False)):
        check(run(a, s, **kw), *want)
    b = Answers(device, [150, 140, 400], [1, 2, 1], 4 * Hkv, Hkv, D, [(2, 128), (1, 0)], bs=64).store()
    s = b.share()
    assert s.lens.tolist() == [128, 0, 0]
    check(run(b, s), *b.expected())
    assert torch.equal(run(b, s, apart=False), run(b, None))


@pytest.mark.parametrize("D,Hkv", [(512, 2), (128, 8)])
def test_captured_where_it_pays(D, Hkv, device):
    """The choice is the replay's, not the capture's: lengths on both sides of the line, two graphs at once on two streams."""
    from gemma_triton_flash_attn_amd import kv4

    a = Answers(device, [2100 + i for i in range(48)], [1] * 48, 4 * Hkv, Hkv, D, [(48, 2048)], bs=64, junk=0).store()
    q, lens = a.q.to(device), [a.lens_dev.clone(), a.lens_dev.clone()]

    def step(n):
        return kv4.attention(q, a.cache, a.table, n, a.cu, max_new=1, shared=kv4.share(a.table, n, a.cu, block_size=64))

    step(lens[0])
    torch.cuda.synchronize()
    graphs, got = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, n in zip(graphs, lens):
        with torch.cuda.graph(graph):
            got.append(step(n))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for cut in (0, 2040, 1500, 600, 0):
        lens[0].copy_(a.lens_dev - cut)
        lens[1].copy_(a.lens_dev - (2040 - cut))
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for n, o in zip(lens, got):
            assert torch.equal(o, step(n))
    check(got[0], *a.expected())


@pytest.mark.parametrize("n", [64, 65, 128, 256, 257, 700])
def test_many_requests(n, device):
    """More requests than a wave looks through at once: dealt to four, several rounds each; groups that lie across the deal, requests
    without tokens, tokens of no request ahead and behind."""
    r = random.Random(n)
    groups, left = [], n
    while left:
        k = min(left, r.choice([1, 2, 3, 40, 150]))
        groups.append((k, r.choice([64, 128, 320]) if k > 1 else 0))
        left -= k
    lens = [c + r.randint(4, 70) for k, c in groups for _ in range(k)]
    new = [r.choice([0, 1, 1, 2, 3]) for _ in lens]
    a = Answers(device, lens, new, 4, 2, 64, groups, bs=64, pad=5, seed=n).store()
    s = a.share(least=64)
    want = a.expected()
    for kw in (dict(), dict(apart=False), dict(max_new=1)):
        check(run(a, s, **kw), *want)


@pytest.mark.parametrize("n,Hkv,D", [(500, 2, 512), (450, 4, 256), (400, 8, 128), (900, 2, 64)])
def test_more_items_than_workgroups(n, Hkv, D, device):
    """A workgroup takes several items in turn, prefixes of many rows and of few and requests behind them; rows of no request after all."""
    groups = [(n // 2, 192), (3, 128), (n - n // 2 - 3, 64)]
    lens = [c + 1 + i % 50 for k, c in groups for i in range(k)]
    a = Answers(device, lens, [1] * n, 2 * Hkv, Hkv, D, groups, bs=64, pad=9, seed=n).store()
    s = a.share(least=64)
    want = a.expected()
    for kw in (dict(), dict(apart=False)):
        o = run(a, s, **kw)
        check(o, want[0], want[1])
        assert not o[:, :, -9:].any() and torch.equal(o, run(a, s, **kw))


@pytest.mark.parametrize("n,D", [(5, 512), (64, 128), (90, 256), (300, 64)])
def test_numbers_that_fit_nothing(n, D, device):
    """Tables, lengths, offsets and results of share that are no such things: nothing outside the arrays is touched, the call ends,
    and the next one is right. q and the cache keep their values."""
    from gemma_triton_flash_attn_amd import kv4

    r = random.Random(n)
    a = Answers(device, [300 + i % 40 for i in range(n)], [1] * n, 8, 2, D, [(n, 256)], bs=64).store()
    s = a.share(least=64)
    want = a.expected()
    before = [t.clone() for t in (a.cache.codes, a.cache.scales)]
    big = [-2 ** 31, -70000, -5, -1, 0, 1, 3, n, n + 1, 100, 5000, 2 ** 20, 2 ** 31 - 1]
    wild = lambda t, p: torch.where(torch.rand(t.shape, generator=g) < p, torch.tensor([r.choice(big) for _ in range(t.numel())]).view(t.shape),  # noqa: E731
                                    t.cpu().long()).to(torch.int32).to(device)
    g = torch.Generator().manual_seed(n)
    q = a.q.to(device)
    for i in range(24):
        p = [0.02, 0.3, 1.0][i % 3]
        table, lens, cu = (wild(t, p if i >> k & 1 else 0) for k, t in enumerate((a.table, a.lens_dev, a.cu)))
        bad = kv4.Shared(*(wild(t, p if (i + 1) >> k & 1 else 0) for k, t in enumerate(s)))
        o = kv4.attention(q, a.cache, table, lens, cu, max_new=1, shared=bad, apart=i % 2 == 0)
        assert o.shape == q.shape
        torch.cuda.synchronize()
    assert torch.equal(q.cpu(), a.q) and all(torch.equal(x, y) for x, y in zip(before, (a.cache.codes, a.cache.scales)))
    check(run(a, s), *want)


def test_more_tokens_than_q_has(device):
    """cu of more tokens than q (not of one request): the rows that q has are right."""
    a = Answers(device, [300 + i for i in range(70)], [2] * 70, 8, 2, 128, [(70, 256)], bs=64).store()
    from gemma_triton_flash_attn_amd import kv4

    s = a.share(least=64)
    want, bound = a.expected()
    for T in (2, 7, 101, 139):
        for apart in (True, False):
            o = kv4.attention(a.q[:, :, :T].contiguous().to(device), a.cache, a.table, a.lens_dev, a.cu, max_new=2, shared=s, apart=apart)
            check(o, want[:, :T], bound[:, :T])


@pytest.mark.parametrize("n", SIZES)
def test_missing_blocks(n, device):
    """Blocks missing in a prefix, all of a prefix, all of a request's own."""
    from gemma_triton_flash_attn_amd import kv4

    lens = [513 + 16 * i % 50 for i in range(n)]
    for holes, whole in (([2], False), ([0, 1, 2, 3, 4, 5, 6, 7], False), ([1], True), ([0, 7], False)):
        a = Answers(device, lens, [1] * n, 16, 4, 128, [(n, 512)], bs=64).store()
        held = [torch.ones(m, dtype=torch.bool) for m in a.lens]
        for c in holes:
            a.table[:, c] = -1
            for h in held:
                h[c * 64:(c + 1) * 64] = False
        if whole:
            a.table[1, 8:] = 1 << 20
            held[1][512:] = False
        s = kv4.share(a.table, a.lens_dev, a.cu, block_size=64, least=64)
        assert s.skip.tolist() == [512] * n
        check(run(a, s), *a.expected(held=held))
    a.table.fill_(-1)  # nothing at all: zeros
    assert not run(a, kv4.share(a.table, a.lens_dev, a.cu, block_size=64, least=64)).any()


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_values_that_are_no_numbers(where, n, device):
    """A token of no number in the prefix reaches its whole group, one in a request's own keys that request alone."""
    lens = [530 + i for i in range(n)] + [300, 300]
    a = Answers(device, lens, [1] * len(lens), 16, 4, 128, [(n, 512), (2, 256)], bs=64)
    for b in range(n) if where == "prefix" else [1]:
        a.k[b][0, 100 if where == "prefix" else 530, 3] = float("inf")
    a.store()
    o = run(a, a.share())
    want, bound = a.expected()
    assert torch.isnan(want[:, 1]).any() and not torch.isnan(want[:, n:]).any()
    check(o, want, bound)


@pytest.mark.parametrize("n", SIZES)
def test_infinite_queries(n, device):
    """A query of infinities answers NaN in both parts and leaves its neighbours alone."""
    a = Answers(device, [530 + i for i in range(n)], [1] * n, 16, 4, 128, [(n, 512)], bs=64).store()
    plain = run(a, a.share())
    a.q[0, 2, 1] = float("inf")
    o = run(a, a.share())
    assert torch.isnan(o[0, 2, 1]).all()
    keep = torch.ones_like(o, dtype=torch.bool)
    keep[0, 2, 1] = False
    assert torch.equal(o[keep], plain[keep])


@pytest.mark.parametrize("seed", range(10))
def test_any_groups(seed, device):
    """Random groups, lengths, counts and layers."""
    r = random.Random(100 + seed)
    D, (Hq, Hkv) = r.choice([64, 128, 256, 512]), r.choice([(4, 4), (8, 1), (16, 4), (6, 2), (32, 4)])
    bs = r.choice([32, 64, 256, 1024])
    groups, lens, new = [], [], []
    for _ in range(r.choice([1, 3, 6])):
        n, common = r.choice([1, 2, 5, 20, 66]), r.choice([0, 1, 3]) * bs
        groups.append((n, common))
        for _ in range(n):
            k = r.choice([0, 1, 1, 1, r.randint(1, 4)])
            new.append(k)
            lens.append(common + r.choice([k, k + r.randint(0, 70), k + r.randint(0, 700)]))
    a = Answers(device, lens, new, Hq, Hkv, D, groups, bs=bs, seed=seed, dtype=r.choice([torch.bfloat16, torch.float16]), pad=r.choice([0, 3])).store()
    if a.T == 0:
        return
    kw = dict(softcap=r.choice([None, 15.0]), causal=r.random() < 0.8)
    want, bound = a.expected(causal=kw["causal"], softcap=kw["softcap"] or 0.0)
    check(a.attend(max_new=max(max(new), 1), shared=a.share(least=r.choice([1, bs])), apart=seed % 5 > 0, **kw), want, bound)


def test_one_token_per_batch_entry(device):
    """(R, Hq, 1, D) queries, strided, with cu."""
    from gemma_triton_flash_attn_amd import kv4

    a = answers("d128_many", device)
    s = a.share()
    want = run(a, s)
    q = a.q[0].transpose(0, 1)[:, :, None].contiguous().to(device)  # (R, Hq, 1, D)
    wide = torch.cat([q, q], 3)[..., :128]
    for x in (q, wide, wide.transpose(1, 2).contiguous().transpose(1, 2)):
        o = kv4.attention(x, a.cache, a.table, a.lens_dev, a.cu, max_new=1, shared=s, apart=True)
        assert o.shape == x.shape and torch.equal(o[:, :, 0].transpose(0, 1), want[0])


def test_captured(device):
    """A graph of share and attention replayed while lengths and tables change in device memory; another call's workspace in
    between."""
    from gemma_triton_flash_attn_amd import kv4

    a, other = answers("d256_many", device, junk=0), answers("d128_many", device)  # rows that look past what was stored: numbers
    table, lens, q = a.table.clone(), a.lens_dev.clone(), a.q.to(device)

    def step():
        s = kv4.share(table, lens, a.cu, block_size=a.bs, least=64)
        return kv4.attention(q, a.cache, table, lens, a.cu, max_new=1, shared=s, apart=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    s = other.share()
    oq = other.q.to(device)
    with torch.cuda.graph(second):
        got2 = kv4.attention(oq, other.cache, other.table, other.lens_dev, other.cu, max_new=1, shared=s, apart=True)
    r = random.Random(0)
    for i in range(4):
        lens.copy_(ints([n - r.choice([0, 0, 64, 200]) if n > 300 else n for n in a.lens], device))
        table.copy_(a.table.roll(i, 0) if i == 2 else a.table)
        q.copy_(a.q.roll(i, 3))
        graph.replay()
        second.replay()
        seen, seen2 = got.clone(), got2.clone()
        torch.cuda.synchronize()
        assert torch.equal(seen, step()) and torch.equal(seen2, run(other, s))


def test_registered(device):
    from gemma_triton_flash_attn_amd import kv4

    a = answers("d64_many", device)
    s = a.share()
    q = a.q.to(device)
    torch.library.opcheck(torch.ops.gfa.kv4_share, (a.table, a.lens_dev, a.cu, a.bs, 64))
    args = (q, a.cache.codes, a.cache.scales, True, a.table, a.lens_dev, a.cu, 1, True, 0, 0.125, 0.0, *s)
    torch.library.opcheck(torch.ops.gfa.kv4_attention, args)
    torch.library.opcheck(torch.ops.gfa.kv4_attention, (*args, True))

    def step(q, codes, scales, table, lens, cu):
        cache = kv4.Cache(codes, scales, torch.bfloat16)
        return kv4.attention(q, cache, table, lens, cu, max_new=1, shared=kv4.share(table, lens, cu, block_size=a.bs, least=64))

    args = (q, a.cache.codes, a.cache.scales, a.table, a.lens_dev, a.cu)
    assert torch.equal(torch.compile(step, fullgraph=True, backend="aot_eager")(*args), step(*args))
