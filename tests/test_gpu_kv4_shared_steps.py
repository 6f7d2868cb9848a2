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
