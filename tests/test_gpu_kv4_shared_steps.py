"""Attention over shared prefixes in steps that hold more than answers: prompt chunks beside them, `max_new` given or not."""
from __future__ import annotations

import pytest
import torch

from kv4_cases import check
from kv4_sharing_cases import Answers

pytestmark = pytest.mark.gpu

HEADS = {64: (16, 4), 128: (16, 4), 256: (8, 2), 512: (8, 2)}


def step(D, device, where="last", chunks=(100,), n=40, pad=0, common=320, **kw):
    """n answers of one token to one prompt, prompt chunks around them; ``where`` "inside": a chunk's request shares the prompt."""
    Hq, Hkv = HEADS[D]
    answers, chunk = [(common + 1 + i % 50, 1) for i in range(n)], [(common + 60 + c, c) for c in chunks]
    if where == "inside":
        both, groups = answers[:5] + chunk + answers[5:], [(n + len(chunk), common)]
    elif where == "first":
        both, groups = chunk + answers, [(1, 0)] * len(chunk) + [(n, common)]
    else:
        both, groups = answers + chunk, [(n, common)] + [(1, 0)] * len(chunk)
    lens, new = [x for x, _ in both], [x for _, x in both]
    a = Answers(device, lens, new, Hq, Hkv, D, groups, bs=64, pad=pad, extra=400, seed=D + n, **kw).store()
    rows = torch.repeat_interleave(torch.tensor(new), torch.tensor(new)) > 1
    return a, torch.cat([rows, torch.zeros(pad, dtype=torch.bool)]).to(device)


@pytest.mark.parametrize("D", list(HEADS))
@pytest.mark.parametrize("where,chunks", [("last", (100,)), ("first", (70, 130)), ("inside", (90,))])
def test_a_chunk_beside_answers(where, chunks, D, device):
    """Without max_new: a chunk's rows are those of the call without prefixes, bit for bit; all rows are right, whoever takes them."""
    a, chunk = step(D, device, where, chunks, pad=3, dtype=torch.float16 if D == 128 else torch.bfloat16)
    s = a.share()
    assert int(s.lens.max()) == 320
    want = a.expected()
    plain = a.attend()
    for apart in (True, False):
        o = a.attend(shared=s, apart=apart)
        check(o, *want)
        assert torch.equal(o[:, :, chunk], plain[:, :, chunk])
        assert not o[:, :, -3:].any() and torch.equal(o, a.attend(shared=s, apart=apart))
    check(a.attend(shared=s, apart=True, softcap=15.0), *a.expected(softcap=15.0))
    check(a.attend(shared=s, apart=True, causal=False), *a.expected(causal=False))


@pytest.mark.parametrize("n", [100, 300])
def test_chunks_among_many_requests(n, device):
    """More requests than one wave looks through, chunks of several sizes about the line."""
    a, chunk = step(128, device, "inside", (15, 16, 17, 18, 200), n=n, pad=5)
    s = a.share()
    want, plain = a.expected(), a.attend()
    first = 5 + 15 + 16  # requests of 17 and more tokens have more than 64 rows
    large = torch.zeros_like(chunk)
    large[first:first + 17 + 18 + 200] = True
    for apart in (True, False):
        o = a.attend(shared=s, apart=apart)
        check(o, *want)
        assert torch.equal(o[:, :, large], plain[:, :, large])


def test_only_chunks(device):
    """No request of few rows is left (the average is of requests without tokens, too): all rows are the plain call's."""
    a = Answers(device, [400] * 30 + [420, 450], [0] * 30 + [100, 130], 8, 2, 128, [(30, 320), (2, 320)], bs=64, extra=100).store()
    s = a.share()
    for apart in (True, False):
        assert torch.equal(a.attend(shared=s, apart=apart), a.attend())


@pytest.mark.parametrize("D", [64, 512])
def test_captured_with_a_chunk(D, device):
    """Replayed with other lengths and counts: the requests' kinds are those of the replay."""
    from gemma_triton_flash_attn_amd import kv4

    a, _ = step(D, device, "last", (100,), junk=0)
    q, lens, cu = a.q.to(device), a.lens_dev.clone(), a.cu.clone()

    def call():
        return kv4.attention(q, a.cache, a.table, lens, cu, shared=kv4.share(a.table, lens, cu, block_size=64), apart=True)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    few = torch.tensor([0] + [3] * 40 + [20]).cumsum(0).to(torch.int32).to(device)  # three tokens each, 20 of the last
    for i in range(4):
        lens.copy_(a.lens_dev - (100 if i == 2 else 0))
        cu.copy_(few if i % 2 else a.cu)
        torch.cuda.synchronize()
        graph.replay()
        seen = got.clone()
        torch.cuda.synchronize()
        assert torch.equal(seen, call())
        if i == 0:
            check(seen, *a.expected())


# (Hq, Hkv, D, bs, softcap, prompts, answers to each, tokens of a prompt, of an answer, new tokens): which way the call goes
CHOICES = {
    # 22 us without prefixes, 25 apart
    "drafts": ((8, 4, 256, 64, 50.0, 1, 16, 3001, 333, 4), "plain"),
    # short requests in tables as short
    "short": ((16, 8, 256, 64, 0.0, 2, 32, 330, 20, 1), "plain"),
    "few": ((32, 8, 128, 64, 0.0, 3, 2, 5800, 60, 2), "plain"),
    # 215 us without, 47 apart
    "long": ((32, 8, 128, 64, 0.0, 1, 64, 16384, 600, 1), "apart"),
    "global": ((32, 4, 512, 64, 0.0, 4, 8, 8192, 1000, 1), "apart"),
    "d64": ((16, 16, 64, 64, 0.0, 8, 3, 11000, 500, 1), "apart"),
    # 145 us without, 152 whole, 184 apart
    "capped": ((8, 4, 256, 64, 50.0, 10, 5, 14000, 400, 8), "whole"),
    # 175 without, 168 whole, 156 apart; of fewer answers 49, 51 and 54
    "capped_d64": ((16, 2, 64, 64, 30.0, 9, 23, 5700, 100, 8), "apart"),
    "capped_d64_few": ((16, 2, 64, 64, 30.0, 4, 10, 5700, 100, 8), "whole"),
    # 70 without, 48 whole, 60 apart
    "d512": ((32, 4, 512, 64, 0.0, 1, 52, 2100, 60, 2), "whole"),
}


@pytest.mark.parametrize("name", list(CHOICES))
def test_the_choice(name, device):
    """Apart, whole in the same launch or the call without prefixes, told by the bits that each leaves."""
    from gemma_triton_flash_attn_amd import kv4

    (Hq, Hkv, D, bs, cap, prompts, answers, prompt, own, new), way = CHOICES[name]
    g = torch.Generator().manual_seed(len(name))
    lens = [prompt + new + int(x) for x in torch.randint(0, own, (prompts * answers,), generator=g)]
    width, whole = max(-(-n // bs) for n in lens) + 2, prompt // bs
    table = torch.arange(len(lens) * width, dtype=torch.int32).view(-1, width)
    for b in range(len(lens)):
        table[b, :whole] = table[b // answers * answers, :whole]
    ids, table = torch.unique(table, return_inverse=True)
    cache = kv4.allocate(len(ids), Hkv, D, bs, torch.bfloat16, device)
    cache.codes.random_(0, 256)
    cache.scales.fill_(125)
    table, lens = table.to(device, torch.int32), torch.tensor(lens, dtype=torch.int32, device=device)
    cu = torch.arange(len(lens) + 1, dtype=torch.int32, device=device) * new
    q = torch.randn(1, Hq, len(lens) * new, D, generator=g).to(device, torch.bfloat16)
    s = kv4.share(table, lens, cu, block_size=bs)
    call = lambda **kw: kv4.attention(q, cache, table, lens, cu, max_new=new, softcap=cap or None, **kw)  # noqa: E731
    o, plain, apart = call(shared=s), call(), call(shared=s, apart=True)
    # (whole requests may leave the plain call's bits, and calls without groups are whole with `apart`, too)
    assert torch.equal(o, plain) or way != "plain"
    assert torch.equal(o, apart) == (way == "apart" or (way == "plain" and torch.equal(plain, apart)))


@pytest.mark.parametrize("n,D", [(40, 512), (70, 128), (300, 64)])
def test_numbers_that_fit_nothing(n, D, device):
    """Without max_new: tables, lengths and offsets that are no such things touch nothing outside the arrays, and the next call is right."""
    from gemma_triton_flash_attn_amd import kv4

    a, _ = step(D, device, "inside", (100,), n=n)
    s, want, q = a.share(), a.expected(), a.q.to(device)
    before = [t.clone() for t in (a.cache.codes, a.cache.scales)]
    g = torch.Generator().manual_seed(n)
    big = torch.tensor([-2 ** 31, -70000, -1, 0, 1, 17, n, 100, 5000, 2 ** 20, 2 ** 31 - 1])

    def wild(t, p):
        other = big[torch.randint(0, len(big), t.shape, generator=g)]
        return torch.where(torch.rand(t.shape, generator=g) < p, other, t.cpu().long()).to(torch.int32).to(device)

    for i in range(18):
        p = [0.02, 0.3, 1.0][i % 3]
        table, lens, cu = (wild(t, p if i >> k & 1 else 0) for k, t in enumerate((a.table, a.lens_dev, a.cu)))
        bad = kv4.Shared(*(wild(t, p if (i + 1) >> k & 1 else 0) for k, t in enumerate(s)))
        assert kv4.attention(q, a.cache, table, lens, cu, shared=bad, apart=i % 2 == 0).shape == q.shape
        torch.cuda.synchronize()
    assert torch.equal(q.cpu(), a.q) and all(torch.equal(x, y) for x, y in zip(before, (a.cache.codes, a.cache.scales)))
    check(a.attend(shared=s, apart=True), *want)
