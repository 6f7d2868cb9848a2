"""What the cache operators refuse of device tensors: calls that are right but for one argument, each by its message. All raise
before anything is launched."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

R, M, BS, HKV, D = 3, 4, 64, 2, 128


@pytest.fixture(scope="module")
def made(device):
    from gemma_triton_flash_attn_amd import kv4

    ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device=device)  # noqa: E731
    cache = kv4.allocate(5, HKV, D, BS, torch.bfloat16, device)
    cache.codes.zero_()
    cache.scales.zero_()
    rows = lambda h, n=R, d=D, dtype=torch.bfloat16: torch.zeros(1, h, n, d, dtype=dtype, device=device)  # noqa: E731
    return dict(ints=ints, cache=cache, rows=rows, slots=torch.full((R,), -1, dtype=torch.int64, device=device))


PLAN = [
    (dict(lens=lambda i: i(R).long()), TypeError, "lens must be"), (dict(lens=lambda i: i(R, 1)), ValueError, "lens must be 1-D"),
    (dict(new=lambda i: i(R).long()), TypeError, "new must be"), (dict(new=lambda i: i(R - 1)), ValueError, "new holds 2 entries"),
    (dict(new=lambda i: i(R).cpu()), ValueError, "new must be on"), (dict(table=lambda i: i(R, M).cpu()), ValueError, "table must be on"),
    (dict(table=lambda i: i(R, M).long()), TypeError, "table must be"), (dict(table=lambda i: i(R * M)), ValueError, "table must be 2-D"),
    (dict(table=lambda i: i(R + 1, M)), ValueError, "table has 4 rows"), (dict(table=lambda i: i(R, 0)), ValueError, "block table of shape"),
    (dict(table=lambda i: i(M, R).t()), ValueError, "table rows"), (dict(table=lambda i: i(1, M).expand(R, M)), ValueError, "table rows"),
    (dict(table=lambda i: i(R, 2 * M)[:, ::2]), ValueError, "table rows"), (dict(free=lambda i: i(5).long()), TypeError, "free must be"),
    (dict(free=lambda i: i(5, 1)), ValueError, "free must be 1-D"), (dict(free=lambda i: i(5).cpu()), ValueError, "free must be on"),
    (dict(used=lambda i: i(2)), ValueError, "used must hold one"), (dict(used=lambda i: i(1).long()), TypeError, "used must be"),
    (dict(used=lambda i: i(1).cpu()), ValueError, "used must be on"), (dict(block_size=lambda i: 48), ValueError, "block_size=48"),
    (dict(block_size=lambda i: 16), ValueError, "block_size=16"), (dict(block_size=lambda i: 2048), ValueError, "block_size=2048"),
    (dict(tokens=lambda i: -1), ValueError, "tokens=-1"), (dict(tokens=lambda i: 1 << 31), ValueError, "tokens=2147483648"),
]


@pytest.mark.parametrize("over,exc,message", PLAN)
def test_plan(over, exc, message, made):
    from gemma_triton_flash_attn_amd import kv4

    i = made["ints"]
    a = dict(lens=i(R), new=i(R), table=i(R, M), free=i(5), used=i(1), block_size=BS, tokens=4)
    kv4.plan(**a)  # right as it is
    with pytest.raises(exc, match=message):
        kv4.plan(**{**a, **{k: f(i) for k, f in over.items()}})


ROWS = [
    (dict(k=lambda r: r(HKV, dtype=torch.float16)), TypeError, "k is"), (dict(v=lambda r: r(HKV).float()), TypeError, "v is"),
    (dict(k=lambda r: r(HKV)[0]), ValueError, "k must be 4-D"), (dict(k=lambda r: r(HKV + 1)), ValueError, "k .*does not fit"),
    (dict(v=lambda r: r(HKV, d=64)), ValueError, "v .*does not fit"), (dict(v=lambda r: r(HKV, n=R + 1)), ValueError, "shape mismatch"),
    (dict(k=lambda r: r(HKV).cpu()), ValueError, "k must be on"), (dict(v=lambda r: r(HKV).cpu()), ValueError, "v must be on"),
    (dict(slots=lambda r: "short"), ValueError, "slots holds 2 entries"), (dict(slots=lambda r: "int32"), TypeError, "slots must be"),
    (dict(slots=lambda r: "2-D"), ValueError, "slots must be 1-D"), (dict(slots=lambda r: "cpu"), ValueError, "slots must be on"),
]


def _slots(made, kind):
    s = made["slots"]
    return {"short": s[:-1], "int32": s.int(), "2-D": s[None], "cpu": s.cpu()}[kind]


@pytest.mark.parametrize("over,exc,message", ROWS)
def test_write(over, exc, message, made):
    from gemma_triton_flash_attn_amd import kv4

    a = dict(k=made["rows"](HKV), v=made["rows"](HKV), slots=made["slots"])
    kv4.write(made["cache"], **a)
    for name, f in over.items():
        x = f(made["rows"])
        a[name] = _slots(made, x) if name == "slots" else x
    with pytest.raises(exc, match=message):
        kv4.write(made["cache"], **a)


@pytest.mark.parametrize("kind,exc,message", [("int32", TypeError, "slots must be"), ("2-D", ValueError, "slots must be 1-D"),
                                              ("cpu", ValueError, "slots must be on")])
def test_read(kind, exc, message, made):
    from gemma_triton_flash_attn_amd import kv4

    with pytest.raises(exc, match=message):
        kv4.read(made["cache"], _slots(made, kind))


ATTENTION = [
    (dict(q=lambda r, i: r(4, dtype=torch.float16)), TypeError, "q is"), (dict(q=lambda r, i: r(4)[0]), ValueError, "q must be 4-D"),
    (dict(q=lambda r, i: r(4, d=64)), ValueError, "q .*does not fit"), (dict(q=lambda r, i: r(3)), ValueError, "N_Q_HEADS=3"),
    (dict(q=lambda r, i: r(0)), ValueError, "N_Q_HEADS=0"), (dict(q=lambda r, i: r(4, n=0)), ValueError, "empty sequence"),
    (dict(q=lambda r, i: r(4).cpu()), ValueError, "q must be on"), (dict(q=lambda r, i: r(4, n=4), cu=lambda r, i: None), ValueError, "do not divide"),
    (dict(table=lambda r, i: i(R + 1, M)), ValueError, "table has 4 rows"), (dict(table=lambda r, i: i(M, R).t()), ValueError, "table rows"),
    (dict(table=lambda r, i: i(R, M).long()), TypeError, "table must be"), (dict(table=lambda r, i: i(R, M).cpu()), ValueError, "table must be on"),
    (dict(lens=lambda r, i: i(R).long()), TypeError, "lens must be"), (dict(lens=lambda r, i: i(R, 1)), ValueError, "lens must be 1-D"),
    (dict(lens=lambda r, i: i(R).cpu()), ValueError, "lens must be on"), (dict(cu=lambda r, i: i(R)), ValueError, "cu holds 3 entries"),
    (dict(cu=lambda r, i: i(R + 1).long()), TypeError, "cu must be"), (dict(cu=lambda r, i: i(R + 1).cpu()), ValueError, "cu must be on"),
    (dict(slide_size=lambda r, i: -1), ValueError, "slide_size"), (dict(max_new=lambda r, i: 0), ValueError, "max_new"),
    (dict(softcap=lambda r, i: -2.0), ValueError, "softcap"), (dict(scale=lambda r, i: 0.0), Exception, "scale=0"),
    (dict(scale=lambda r, i: float("inf")), Exception, "scale=inf"),
]


@pytest.mark.parametrize("over,exc,message", ATTENTION)
def test_attention(over, exc, message, made):
    from gemma_triton_flash_attn_amd import kv4

    r, i = made["rows"], made["ints"]
    a = dict(q=r(4), cache=made["cache"], table=i(R, M), lens=i(R), cu=i(R + 1))
    assert not kv4.attention(**a).any()
    with pytest.raises(exc, match=message):
        kv4.attention(**{**a, **{k: f(r, i) for k, f in over.items()}})


def test_caches(made):
    from gemma_triton_flash_attn_amd import kv4

    c, s = made["cache"].codes, made["cache"].scales
    odd = torch.zeros(c.numel() + 8, dtype=torch.uint8, device=c.device)[8:].view(c.shape)
    for cc, ss, message in [(c, s.cpu(), "one GPU"), (c.cpu(), s, "one GPU"), (odd, s, "aligned"), (c[:, :1], s, "belong together"),
                            (c[:, :1], s[:, :1], "contiguous")]:
        with pytest.raises(ValueError, match=message):
            kv4.Cache(cc, ss, torch.bfloat16)
