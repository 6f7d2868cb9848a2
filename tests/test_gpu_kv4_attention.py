"""Attention over the 4-bit cache against 64 bits on the values the cache keeps; bounds from the kernel's roundings
(kv4_cases.Requests.expected). What is not a request's own (other blocks, the rest of its last block) is full of NaN scales."""
from __future__ import annotations

import pytest
import torch

from kv4_cases import Requests, check

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (4, 4), (6, 2)])
def test_single_tokens(D, Hq, Hkv, dtype, device):
    lens = [1, 31, 32, 33, 64, 200, 517]
    r = Requests(device, lens, [1] * 7, Hq, Hkv, D, dtype=dtype).store()
    check(r.attend(max_new=1), *r.expected())
    check(r.attend(max_new=1, slide_size=40), *r.expected(window=40))


@pytest.mark.parametrize("bs", [32, 128, 256])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_several_tokens(D, bs, device):
    r = Requests(device, [5, 70, 300, 96, 33], [5, 3, 17, 40, 0], 8, 2, D, bs, pad=3).store()
    check(r.attend(), *r.expected())
    check(r.attend(slide_size=25, max_new=40), *r.expected(window=25))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [128, 256, 512])
def test_long_chunks(D, dtype, device):
    r = Requests(device, [400, 260, 130], [150, 260, 1], 8, 2, D, dtype=dtype, pad=5).store()
    check(r.attend(), *r.expected())
    check(r.attend(slide_size=100), *r.expected(window=100))


@pytest.mark.parametrize("D", [64, 256, 512])
def test_options(D, device):
    r = Requests(device, [90, 40, 129], [2, 40, 1], 8, 4, D, dtype=torch.float16, amp=3.0).store()
    check(r.attend(softcap=5.0), *r.expected(softcap=5.0))
    check(r.attend(softcap=50.0, slide_size=30), *r.expected(softcap=50.0, window=30))
    check(r.attend(scale=0.3), *r.expected(scale=0.3))
    check(r.attend(causal=False), *r.expected(causal=False))
    check(r.attend(causal=False, slide_size=7), *r.expected(causal=False))  # a window needs causal
    check(r.attend(slide_size=1), *r.expected(window=1))


def test_many_heads_of_one(device):
    """More query heads than a row block holds: 32 and 20 for one KV head."""
    for Hq in (32, 20):
        r = Requests(device, [100, 37], [1, 2], Hq, 1, 128).store()
        check(r.attend(), *r.expected())


def test_empty_requests_and_rows_behind(device):
    """Requests without tokens, without new ones, rows behind the last: zeros, and nothing of the junk."""
    r = Requests(device, [0, 50, 20, 0], [0, 1, 0, 0], 4, 2, 128, pad=70).store()
    o = r.attend()
    check(o, *r.expected())
    assert not o[:, :, 1:].any()
    # a request that says it has no tokens, with a row in q
    r.lens_dev[1] = 0
    assert not r.attend().any()
    # lengths below the new tokens: rows at negative positions see nothing
    r = Requests(device, [2], [1], 4, 2, 64).store()
    r.cu[1] = 1
    r.lens_dev[0] = 0
    assert not r.attend(causal=False).any()


def test_positions_without_a_block(device):
    """Entries of the table that are no block hide their positions, wherever they are."""
    for D in (64, 512):
        r = Requests(device, [200, 130], [1, 3], 8, 2, D).store()
        o, bound = r.expected()
        held = [torch.ones(n, dtype=torch.bool) for n in r.lens]
        r.table[0, 1] = -1
        held[0][64:128] = False
        r.table[1, 0] = 1 << 30
        held[1][:64] = False
        check(r.attend(), *r.expected(held=held))
        r.table[0] = -1
        held[0][:] = False
        got = r.attend()
        check(got, *r.expected(held=held))
        assert not got[:, :, 0].any()
        # lengths past the table: what has no entry is not there
        r.lens_dev[1] = 100000
        r.attend()


@pytest.mark.parametrize("D", [64, 256, 512])
@pytest.mark.parametrize("dtype", TYPES)
def test_no_number_reaches_only_who_attends(D, dtype, device):
    """A key and a value that are no numbers: NaN for the rows that attend to them (their head's), all others as without."""
    r = Requests(device, [160, 160], [60, 60], 4, 2, D, dtype=dtype)
    r.k[0][0, 120, 3] = float("inf")
    r.v[0][1, 130, 40] = float("nan")
    r.store()
    want, bound = r.expected()
    # rows at positions 100..159 of request 0: head 0, 1 from 120 on, heads 2, 3 from 130 on
    want[:2, 20:60], want[2:, 30:60] = float("nan"), float("nan")
    assert not torch.isnan(want[:, 60:]).any() and not torch.isnan(want[:2, :20]).any()
    check(r.attend(), want, bound)


def test_infinite_queries(device):
    """A query with an infinity: NaN or what the formula gives, its own rows only."""
    r = Requests(device, [70, 70], [1, 1], 4, 1, 128).store()
    clean = r.attend()
    r.q[0, 1, 0, 5] = float("inf")
    o = r.attend()
    assert torch.isnan(o[0, 1, 0]).all()
    assert torch.equal(o[0, 0], clean[0, 0]) and torch.equal(o[0, 2:], clean[0, 2:]) and torch.equal(o[0, 1, 1], clean[0, 1, 1])


@pytest.mark.parametrize("D,Hq,Hkv", [(512, 8, 1), (256, 2, 2), (128, 8, 2), (64, 4, 4)])
def test_long_axis(D, Hq, Hkv, device):
    """Few rows over a long axis, split over many workgroups and joined; twice the same bits."""
    r = Requests(device, [6001, 40, 2500], [1, 1, 2], Hq, Hkv, D).store()
    a, b = r.attend(), r.attend()
    check(a, *r.expected())
    assert torch.equal(a, b)


def test_many_requests(device):
    """More requests than a wave has lanes."""
    lens = [1 + 7 * (i % 31) for i in range(150)]
    r = Requests(device, lens, [1 if i % 5 else 2 for i in range(150)], 4, 2, 64, 32, pad=9).store()
    r.lens_dev[0] = 1
    r = Requests(device, [max(2, n) for n in lens], r.new, 4, 2, 64, 32, pad=9).store()
    check(r.attend(), *r.expected())


def test_forms_of_the_call(device):
    """Without cu, one token per batch entry, strided and unaligned queries: the same bits."""
    from gemma_triton_flash_attn_amd import kv4

    r = Requests(device, [50, 90, 33, 64], [1] * 4, 8, 2, 128).store()
    q = r.q.to(device)
    base = r.attend()
    assert torch.equal(kv4.attention(q, r.cache, r.table, r.lens_dev), base)
    steps = kv4.attention(q.transpose(0, 2), r.cache, r.table, r.lens_dev, r.cu, max_new=1)
    assert steps.shape == (4, 8, 1, 128) and torch.equal(steps.transpose(0, 2), base)
    rows = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(kv4.attention(rows, r.cache, r.table, r.lens_dev, r.cu), base)
    odd = torch.cat([q[..., :1], q], -1)[..., 1:]
    assert torch.equal(kv4.attention(odd, r.cache, r.table, r.lens_dev, r.cu), base)
    wide = torch.full((4, r.table.shape[1] + 5), -1, dtype=torch.int32, device=device)
    wide[:, :r.table.shape[1]] = r.table
    assert torch.equal(kv4.attention(q, r.cache, wide[:, :r.table.shape[1]], r.lens_dev, r.cu), base)
    two = Requests(device, [50, 90], [3, 3], 8, 2, 128).store()
    pairs = kv4.attention(two.q.to(device), two.cache, two.table, two.lens_dev)
    assert torch.equal(pairs, two.attend())


def test_a_cache_past_4_gib(device):
    from gemma_triton_flash_attn_amd import kv4

    r = Requests(device, [150, 90], [1, 2], 8, 4, 512).store()
    big = kv4.allocate(35000, 4, 512, 64, torch.bfloat16, device)
    shift = 34990 - r.cache.num_blocks
    big.codes[shift:shift + r.cache.num_blocks] = r.cache.codes
    big.scales[shift:shift + r.cache.num_blocks] = r.cache.scales
    o = kv4.attention(r.q.to(device), big, torch.where(r.table >= 0, r.table + shift, -1), r.lens_dev, r.cu)
    assert torch.equal(o, r.attend())


def test_max_new_only_chooses_kernels(device):
    """Too small, too large or none: the same rows within the roundings, nothing left out."""
    r = Requests(device, [400, 260, 700, 33], [150, 3, 40, 1], 8, 2, 128, pad=2).store()
    want, bound = r.expected()
    for most in (1, 2, 150, 1 << 20, None):
        check(r.attend(max_new=most), want, bound)


def test_offsets_that_are_no_prefix_sums(device):
    """cu, lens and tables of any content keep the call inside its arrays: other requests' rows stay right."""
    r = Requests(device, [3000, 90, 260], [2, 1, 5], 8, 2, 128, pad=2).store()
    want = r.attend()
    good = r.cu.clone()
    big = 2 ** 31 - 1
    for cu in ([0, big, 3, 8], [0, 2, -5, 8], [-big, big, 3, 8], [5, 0, 3, 8], [big] * 4, [0, 2, 3, -1]):
        r.cu.copy_(torch.tensor(cu, dtype=torch.int32))
        r.attend()
        r.attend(slide_size=50, max_new=1)
    r.cu.copy_(good)
    lens = r.lens_dev.clone()
    r.lens_dev.copy_(torch.tensor([big, -big, 4], dtype=torch.int32))
    r.attend()
    r.attend(causal=False)
    r.lens_dev.copy_(lens)
    table = r.table.clone()
    r.table.fill_(big)
    assert not r.attend().any()
    r.table.copy_(table)
    assert torch.equal(r.attend(), want)


def test_ragged_splits_of_chunks(device):
    """Prompt chunks of unequal lengths that are split over their keys, beside single tokens over a long axis."""
    for D, Hq, Hkv in ((512, 8, 1), (256, 4, 2), (64, 2, 2)):
        r = Requests(device, [2100, 900, 1500, 40, 3000], [70, 300, 1, 2, 1], Hq, Hkv, D, 64, pad=3, seed=D).store()
        a, b = r.attend(), r.attend()
        assert torch.equal(a, b)
        check(a, *r.expected())
        check(r.attend(slide_size=600), *r.expected(window=600))


def test_the_longest_table(device):
    """One request of 2^30 tokens, its table naming one block 2^20 - 1 times and another one at the end. Head 0 looks for the
    last block alone, head 1 sees the others."""
    from gemma_triton_flash_attn_amd import kv4
    from oracle import kv4_oracle as orc

    D, bs, M = 64, 1024, 1 << 20
    g = torch.Generator().manual_seed(7)
    k = torch.zeros(1, 1, 2 * bs, D)
    k[:, :, bs:, 0] = 16.0  # a value of the format
    v = torch.randn(1, 1, 2 * bs, D, generator=g)
    v[:, :, bs:] += 3.0
    k, v = k.bfloat16(), v.bfloat16()
    cache = kv4.allocate(2, 1, D, bs, torch.bfloat16, device)
    kv4.write(cache, k.to(device), v.to(device), torch.arange(2 * bs, device=device))
    table = torch.zeros(1, M, dtype=torch.int32, device=device)
    table[0, -1] = 1
    q = torch.zeros(1, 2, 1, D, dtype=torch.bfloat16)
    q[0, 0, 0, 0], q[0, 1, 0, 0] = 32.0, -32.0  # scores 64 and -64 at the end, 0 elsewhere
    lens = torch.tensor([M * bs], dtype=torch.int32, device=device)
    got = kv4.attention(q.to(device), cache, table, lens)[0, :, 0].double().cpu()
    vr = orc.rounded(v[0]).double()[0]
    # e^64 against 2^30 e^0: the other side weighs less than 2^-50
    want = torch.stack([vr[bs:].mean(0), vr[:bs].mean(0)])
    weight = torch.stack([vr[bs:].abs().mean(0), vr[:bs].abs().mean(0)])
    # P is 1 where it counts, so sums round alone: a lane adds 2^30 / (512 workgroups, 4 waves) keys of a tile 4 or 32 at a time,
    # at most 2^17 sums of at most 2^-24 of the total, in O^T and in the row sum; joining adds less than 2^10.
    bound = 2 * (2 ** 17 + 2 ** 10) * 2.0 ** -24 * weight + 2.0 ** -8 * want.abs()
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() - bound).max())
