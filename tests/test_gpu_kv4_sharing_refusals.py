"""What the operators of requests with something in common refuse of device tensors: calls that are right but for one argument, each
by its message. All raise before anything is launched."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

R, M, BS, HKV, D, BLOCKS = 3, 4, 64, 2, 128, 5


@pytest.fixture(scope="module")
def made(device):
    from gemma_triton_flash_attn_amd import kv4

    ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device=device)  # noqa: E731
    caches = [kv4.allocate(BLOCKS, HKV, d, BS, torch.bfloat16, device) for d in (D, 64)]
    for c in caches:
        c.codes.zero_()
        c.scales.zero_()
    return dict(ints=ints, caches=caches, device=device)


PAGES = [
    (dict(caches=lambda m: []), ValueError, "at least one cache"),
    (dict(caches=lambda m: [m["caches"][0], _other(m, BLOCKS + 1)]), ValueError, "do not belong"),
    (dict(caches=lambda m: [m["caches"][0], _other(m, BLOCKS, 32)]), ValueError, "do not belong"),
    (dict(table=lambda m: m["ints"](R, M).long()), TypeError, "table must be"), (dict(table=lambda m: m["ints"](R * M)), ValueError, "table must be 2-D"),
    (dict(table=lambda m: m["ints"](R, M).cpu()), ValueError, "must be on"), (dict(table=lambda m: m["ints"](R + 1, M)), ValueError, "table has 4 rows"),
    (dict(table=lambda m: m["ints"](M, R).t()), ValueError, "table rows"), (dict(table=lambda m: m["ints"](R, 0)), ValueError, "block table of shape"),
    (dict(lens=lambda m: m["ints"](R).long()), TypeError, "lens must be"), (dict(lens=lambda m: m["ints"](R, 1)), ValueError, "lens must be 1-D"),
    (dict(lens=lambda m: m["ints"](R).cpu()), ValueError, "lens must be on"), (dict(free=lambda m: m["ints"](BLOCKS).long()), TypeError, "free must be"),
    (dict(free=lambda m: m["ints"](2 * BLOCKS)[::2]), ValueError, "free must be contiguous"), (dict(free=lambda m: m["ints"](BLOCKS).cpu()), ValueError, "free must be on"),
    (dict(table=lambda m: m["ints"](4097, M), lens=lambda m: m["ints"](4097)), ValueError, "4097 requests"),
]
FORK = [
    (dict(used=lambda m: m["ints"](2)), ValueError, "used must hold one"), (dict(used=lambda m: m["ints"](1).long()), TypeError, "used must be"),
    (dict(used=lambda m: m["ints"](1).cpu()), ValueError, "used must be on"), (dict(parents=lambda m: m["ints"](2).long()), TypeError, "parents must be"),
    (dict(parents=lambda m: m["ints"](2, 1)), ValueError, "parents must be 1-D"), (dict(parents=lambda m: m["ints"](2).cpu()), ValueError, "parents must be on"),
    (dict(parents=lambda m: m["ints"](0)), ValueError, "0 rows"), (dict(parents=lambda m: m["ints"](4097)), ValueError, "4097 rows"),
    (dict(keep=lambda m: m["ints"](R + 1)), ValueError, "keep holds 4 entries"), (dict(keep=lambda m: m["ints"](R).float()), TypeError, "keep must be"),
    (dict(parents=lambda m: m["ints"](2), keep=lambda m: m["ints"](R)), ValueError, "keep holds 3 entries for 2 rows"),
    (dict(keep=lambda m: m["ints"](R).cpu()), ValueError, "keep must be on"),
]


def _other(m, blocks, bs=BS):
    from gemma_triton_flash_attn_amd import kv4

    return kv4.allocate(blocks, HKV, D, bs, torch.bfloat16, m["device"])


def _with(made, over, **more):
    i = made["ints"]
    a = dict(caches=made["caches"], table=i(R, M), lens=i(R), free=torch.arange(BLOCKS, dtype=torch.int32, device=made["device"]), **more)
    return a, {**a, **{k: f(made) for k, f in over.items()}}


@pytest.mark.parametrize("over,exc,message", PAGES + FORK)
def test_fork(over, exc, message, made):
    from gemma_triton_flash_attn_amd import kv4

    right, wrong = _with(made, over, used=made["ints"](1))
    kv4.fork(**right)
    with pytest.raises(exc, match=message):
        kv4.fork(**wrong)


@pytest.mark.parametrize("over,exc,message", PAGES + [(dict(free=lambda m: m["ints"](BLOCKS - 1)), ValueError, "all of its 5 blocks")])
def test_compact(over, exc, message, made):
    from gemma_triton_flash_attn_amd import kv4

    right, wrong = _with(made, over)
    kv4.compact(**right)
    with pytest.raises(exc, match=message):
        kv4.compact(**wrong)


@pytest.mark.parametrize("src,dst,exc,message", [
    (lambda i: i(2).long(), lambda i: i(2), TypeError, "src must be"), (lambda i: i(2), lambda i: i(2, 1), ValueError, "dst must be 1-D"),
    (lambda i: i(2), lambda i: i(3), ValueError, "src holds 2 entries, dst 3"), (lambda i: i(2), lambda i: i(2).cpu(), ValueError, "dst must be on")])
def test_copy(src, dst, exc, message, made):
    from gemma_triton_flash_attn_amd import kv4

    i = made["ints"]
    kv4.copy(made["caches"], i(2) - 1, i(2))
    with pytest.raises(exc, match=message):
        kv4.copy(made["caches"], src(i), dst(i))


@pytest.mark.parametrize("over,exc,message", [
    (dict(table=lambda i: i(R, M).long()), TypeError, "table must be"), (dict(table=lambda i: i(R + 1, M)), ValueError, "table has 4 rows"),
    (dict(lens=lambda i: i(R).long()), TypeError, "lens must be"), (dict(cu=lambda i: i(R)), ValueError, "cu holds 3 entries"),
    (dict(cu=lambda i: i(R + 1).cpu()), ValueError, "cu must be on"), (dict(block_size=lambda i: 48), ValueError, "block_size=48"),
    (dict(least=lambda i: 0), ValueError, "least=0"),
    (dict(table=lambda i: i(4097, 1), lens=lambda i: i(4097), cu=lambda i: i(4098)), ValueError, "4097 requests")])
def test_share(over, exc, message, made):
    from gemma_triton_flash_attn_amd import kv4

    i = made["ints"]
    a = dict(table=i(R, M), lens=i(R), cu=i(R + 1), block_size=BS, least=64)
    kv4.share(**a)
    with pytest.raises(exc, match=message):
        kv4.share(**{**a, **{k: f(i) for k, f in over.items()}})


@pytest.mark.parametrize("over,exc,message", [
    (dict(shared=lambda k, i: k.Shared(i(R), i(R + 1).long(), i(R))), TypeError, "shared.cu must be"),
    (dict(shared=lambda k, i: k.Shared(i(R + 1), i(R + 2), i(R + 1))), ValueError, "shared is for 4 requests"),
    (dict(shared=lambda k, i: k.Shared(i(R), i(R), i(R))), ValueError, "shared is for"),
    (dict(shared=lambda k, i: k.Shared(i(R), i(R + 1), i(R).cpu())), ValueError, "shared.lens must be on"),
    (dict(shared=lambda k, i: k.Shared(i(R), None, i(R))), ValueError, "all of skip, cu and lens"), (dict(cu=lambda k, i: None), ValueError, "without"),
])
def test_attention(over, exc, message, made):
    from gemma_triton_flash_attn_amd import kv4

    i = made["ints"]
    q = torch.zeros(1, 4, R, D, dtype=torch.bfloat16, device=made["device"])
    a = dict(q=q, cache=made["caches"][0], table=i(R, M), lens=i(R), cu=i(R + 1), max_new=1, shared=kv4.Shared(i(R), i(R + 1), i(R)))
    assert not kv4.attention(**a).any()
    with pytest.raises(exc, match=message):
        kv4.attention(**{**a, **{k: f(kv4, i) for k, f in over.items()}})


@pytest.mark.parametrize("over,exc,message", [
    (dict(target=lambda p: p.double()), TypeError, "target is"), (dict(target=lambda p: p[0]), ValueError, "target must be 2-D"),
    (dict(target=lambda p: p[:, :0]), ValueError, "target of shape"), (dict(target=lambda p: p.cpu()), ValueError, "target must be on a GPU"),
    (dict(draft=lambda p: p.half()), TypeError, "draft is"), (dict(draft=lambda p: p[:, 1:]), ValueError, "shape mismatch"),
    (dict(draft=lambda p: p.cpu()), ValueError, "draft must be on"), (dict(tokens=lambda p: torch.zeros(6, dtype=torch.int32, device=p.device)), TypeError, "tokens must be"),
    (dict(tokens=lambda p: torch.zeros(5, dtype=torch.int64, device=p.device)), ValueError, "tokens holds 5 entries"),
    (dict(accept=lambda p: p[:5, 0]), ValueError, "accept 5"), (dict(accept=lambda p: p[:, 0].half()), TypeError, "accept must be"),
    (dict(sample=lambda p: p[:2, 0]), ValueError, "sample holds 2 entries"), (dict(sample=lambda p: p[:3, 0].cpu()), ValueError, "sample must be on"),
    (dict(lens=lambda p: torch.zeros(3, dtype=torch.int64, device=p.device)), TypeError, "lens must be"),
    (dict(cu=lambda p: torch.zeros(3, dtype=torch.int32, device=p.device)), ValueError, "cu holds 3 entries"),
    (dict(lens=lambda p: torch.zeros(4, dtype=torch.int32, device=p.device), sample=lambda p: p[:4, 0]), ValueError, "do not divide"),
    (dict(target=lambda p: p.clone().requires_grad_(True)), NotImplementedError, "no gradient")])
def test_verify(over, exc, message, made):
    from gemma_triton_flash_attn_amd import kv4

    p = torch.zeros(6, 9, device=made["device"])
    a = dict(target=p, draft=p, tokens=torch.zeros(6, dtype=torch.int64, device=p.device), accept=p[:, 0], sample=p[:3, 0], lens=made["ints"](3))
    kv4.verify(**a)
    with pytest.raises(exc, match=message):
        kv4.verify(**{**a, **{k: f(p) for k, f in over.items()}})
