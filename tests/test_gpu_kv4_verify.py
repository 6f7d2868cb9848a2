"""Verified drafts against exact arithmetic: which tokens are accepted, and the one drawn behind them."""
from __future__ import annotations

import random

import pytest
import torch

from oracle import kv4_sharing_oracle as orc

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(device, counts, V, dtype=torch.float32, seed=0, sharp=1.0, pad=(0, 0)):
    """target, draft, tokens, accept, sample, lens, cu of requests with so many tokens each; drafts near the target."""
    g = torch.Generator().manual_seed(seed)
    T = pad[0] + sum(counts) + pad[1]
    logits = sharp * torch.randn(T, V, generator=g)
    draft = torch.softmax(logits + 0.8 * torch.randn(T, V, generator=g), -1)
    target = torch.softmax(logits, -1).roll(-1, 0)
    tokens = torch.multinomial(draft, 1, generator=g)[:, 0]
    cu = torch.tensor([pad[0]] + (torch.tensor(counts).cumsum(0) + pad[0]).tolist(), dtype=torch.int32)
    out = dict(target=target.to(dtype), draft=draft.to(dtype), tokens=tokens, accept=torch.rand(T, generator=g),
               sample=torch.rand(len(counts), generator=g), lens=torch.randint(10, 99, (len(counts),), generator=g, dtype=torch.int32), cu=cu)
    return {k: v.to(device) for k, v in out.items()}


def expected(a):
    f = lambda x: None if x is None else x.double().tolist()  # noqa: E731
    return orc.verify(f(a["target"]), f(a["draft"]), a["tokens"].tolist(), f(a["accept"]), f(a["sample"]), a["lens"].tolist(), a["cu"].tolist())


def check(a, **over):
    from gemma_triton_flash_attn_amd import kv4

    v = kv4.verify(**{**a, **over})
    want = expected(a)
    assert v.tokens.tolist() == want[0] and v.accepted.tolist() == want[1] and v.lens.tolist() == want[2]
    return v


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 511, 512, 513, 4096, 5003])
def test_vocabularies(V, dtype, device):
    a = make(device, [5, 1, 3, 2, 8], V, dtype, seed=V, sharp=2.0)
    check(a)
    check({**a, "draft": None})


@pytest.mark.parametrize("counts", [[1], [1, 1, 1], [2], [70], [140, 1, 65, 64], [0, 3, 0], [0]])
def test_counts(counts, device):
    """Requests with no drafted token, more of them than lanes, none at all; tokens of no request on both sides. Nearly equal
    probabilities, so that long drafts are accepted far."""
    a = make(device, counts, 40, seed=1, sharp=0.5, pad=(3, 2))
    for i in range(len(a["target"]) - 1):
        a["draft"][i + 1] = a["target"][i]
    a["accept"][40:] = 0.999
    check(a)
    a["accept"].zero_()
    v = check(a)
    assert v.accepted.tolist() == [max(n - 1, 0) for n in counts]


def test_several_segments(device):
    """A row over many waves' segments and more of them than a workgroup's threads, draws from all of the row."""
    from gemma_triton_flash_attn_amd import kv4

    V = 150001
    a = make(device, [2] * 40, V, sharp=0.1, seed=3)
    a["sample"] = torch.linspace(0, 1 - 2.0 ** -24, 40).to(device)
    a["accept"].fill_(1e30)  # nothing is accepted: no ratio of the probabilities is as large
    v = kv4.verify(**a)
    t = a["cu"][:-1].long()
    w = (a["target"][t].double() - a["draft"][t + 1].double()).clamp(min=0).cpu()
    c = w.cumsum(-1)
    for b in range(40):
        i = int(v.tokens[t[b]])
        goal = float(a["sample"][b].double()) * float(c[b, -1])
        slack = 1e-12 * float(c[b, -1])  # 64-bit sums in another order: V 2^-53 of the sum at most
        assert w[b, i] > 0 and float(c[b, i]) > goal - slack and float(c[b, i] - w[b, i]) <= goal + slack
    assert not v.accepted.any() and torch.equal(v.lens, a["lens"] - 1)


def test_one_request_of_a_large_vocabulary(device):
    from gemma_triton_flash_attn_amd import kv4

    a = make(device, [3], 262144, torch.bfloat16, sharp=3.0)
    a["accept"].zero_()
    for r in (0.0, 0.3, 0.999):
        a["sample"].fill_(r)
        v = kv4.verify(**a)
        c = a["target"][2].double().cpu().cumsum(0)
        i = int(v.tokens[2])
        goal, slack = float(a["sample"].double()) * float(c[-1]), 1e-10 * float(c[-1])
        assert float(c[i]) > goal - slack and (i == 0 or float(c[i - 1]) <= goal + slack)
        assert v.accepted.tolist() == [2]


def test_borders(device):
    """Equality is no acceptance; probabilities of zero; a sum that sample reaches exactly; the last entry with weight."""
    a = make(device, [2] * 8, 4)
    p, q, x = a["target"], a["draft"], a["tokens"]
    x.fill_(1)
    p[:] = torch.tensor([0.25, 0.25, 0.5, 0.0])
    q[:] = torch.tensor([0.0, 0.5, 0.5, 0.0])
    u = [0.5, 0.5 - 2.0 ** -25, 0.5 + 2.0 ** -24, 0.0, 0.5, 0.5, 0.9, 0.9]
    a["accept"][1::2] = torch.tensor(u)
    a["sample"].copy_(torch.tensor([0.0, 0.5, 0.25, 0.75, 1.0, 5.0, -1.0, float("nan")]))
    v = check(a)
    assert v.accepted.tolist() == [0, 1, 0, 1, 0, 0, 0, 0]
    assert v.tokens[0::2].tolist() == [0, 1, 0, 1, 0, 0, 0, 0] and v.tokens[[3, 7]].tolist() == [2, 2]
    p[:, 1] = 0.0
    check(a)
    q[:, 1] = 0.0
    check(a)


def test_no_weight_left(device):
    """The draft's probabilities are the target's: the target's are drawn from. No probabilities at all: no token."""
    a = make(device, [2, 2, 3], 9)
    for t in (0, 2, 4, 5):
        a["draft"][t + 1] = a["target"][t]
    a["accept"].fill_(1.0)
    assert not check(a).accepted.any()
    a["target"].zero_()
    v = check(a)
    assert v.tokens.tolist() == [-1] * 7 and not v.accepted.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_no_probabilities(dtype, device):
    a = make(device, [3, 2, 1, 2], 40, dtype)
    for name in ("target", "draft"):
        x = a[name]
        x[:, 3], x[:, 5], x[:, 7], x[:, 9] = float("nan"), float("inf"), -0.5, float("-inf")
    check(a)
    for i, bad in enumerate((3, 5, 7, 9, 40, -1, 1 << 40)):  # tokens of no probability, and outside the vocabulary
        a["tokens"].fill_(bad)
        assert not check(a).accepted.any()
    a["accept"].fill_(float("nan"))
    check(a)


def test_weights_need_no_sum_of_one(device):
    a = make(device, [3, 2, 4], 300)
    a["target"] *= 1e6
    check(a)
    a["target"] *= 1e-30
    check(a)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype, device):
    """Rows apart, rows that start anywhere, one row for all tokens, columns apart (copied), every other token."""
    a = make(device, [3, 1, 2], 101, dtype)
    wide = lambda x, o: torch.cat([torch.full((6, o), 9.0, dtype=dtype, device=device), x, x], 1)[:, o:o + 101]  # noqa: E731
    for o in (1, 3, 8):
        check({**a, "target": wide(a["target"], o), "draft": wide(a["draft"], 5 - o % 3)})
    check({**a, "target": a["target"][:1].expand(6, 101), "draft": a["draft"].t().contiguous().t()})
    check({**a, "tokens": a["tokens"].repeat_interleave(2)[::2], "accept": a["accept"].repeat_interleave(3)[::3]})


def test_without_cu(device):
    """The same number of tokens each."""
    from gemma_triton_flash_attn_amd import kv4

    a = make(device, [4, 4, 4], 50)
    want = kv4.verify(**a)
    cu = a.pop("cu")
    got = kv4.verify(**a)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and len(cu) == 4


def test_offsets_that_are_no_prefix_sum(device):
    """cu that runs back or past the tokens names no tokens there."""
    a = make(device, [2, 2, 2], 20)
    for cu in ([0, 2, 99, 99], [4, 2, 6, 6], [-5, 2, 4, 6]):
        a["cu"] = torch.tensor(cu, dtype=torch.int32, device=device)
        got = check_counts(a)
        assert len(got) == 3


def check_counts(a):
    from gemma_triton_flash_attn_amd import kv4

    v = kv4.verify(**a)
    want = expected(a)
    assert v.accepted.tolist() == want[1] and v.lens.tolist() == want[2]
    return want[1]


def test_the_distribution(device):
    """First tokens are distributed as the target's, whatever the draft: 60000 requests, deviations below 5 of a standard one."""
    from gemma_triton_flash_attn_amd import kv4

    R, V = 60000, 6
    g = torch.Generator().manual_seed(2)
    p = torch.tensor([0.4, 0.05, 0.25, 0.0, 0.2, 0.1], dtype=torch.float64)
    q = torch.tensor([0.1, 0.3, 0.25, 0.15, 0.2, 0.0], dtype=torch.float64)
    for draft in (q, None):
        x = torch.multinomial(q, 2 * R, replacement=True, generator=g) if draft is not None else torch.full((2 * R,), 2)
        v = kv4.verify(p.float().expand(2 * R, V).to(device), None if draft is None else draft.float().expand(2 * R, V).to(device),
                       x.to(device), torch.rand(2 * R, generator=g).to(device), torch.rand(R, generator=g).to(device),
                       torch.full((R,), 50, dtype=torch.int32, device=device))
        seen = torch.bincount(v.tokens[0::2].cpu(), minlength=V).double()
        assert ((seen - R * p).abs() <= 5 * (R * p * (1 - p)).sqrt()).all(), seen


def test_random_calls(device):
    r = random.Random(0)
    for i in range(12):
        counts = [r.choice([0, 1, 2, 5, 9]) for _ in range(r.choice([1, 4, 30]))]
        a = make(device, counts, r.choice([3, 33, 700]), r.choice(TYPES), seed=i, sharp=r.choice([0.3, 3.0]), pad=(r.choice([0, 2]), 1))
        if r.random() < 0.3:
            a["draft"] = None
        check(a)


def test_captured_and_compiled(device):
    from gemma_triton_flash_attn_amd import kv4

    a = make(device, [3, 1, 5], 700)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv4.verify(**a)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kv4.verify(**a)
    for seed in range(4):
        b = make(device, [3, 1, 5], 700, seed=10 + seed)
        for k in a:
            a[k].copy_(b[k])
        graph.replay()
        seen = [x.clone() for x in got]
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(seen, kv4.verify(**a)))
        assert seen[0].tolist() == expected(a)[0]
    args = (a["target"], a["draft"], a["tokens"], a["accept"], a["sample"], a["lens"], a["cu"])
    torch.library.opcheck(torch.ops.gfa.kv4_verify, args)
    out = torch.compile(lambda *x: kv4.verify(*x), fullgraph=True, backend="aot_eager")(*args)
    assert all(torch.equal(x, y) for x, y in zip(out, kv4.verify(*args)))
