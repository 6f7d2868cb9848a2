"""Prompt chunks over the 4-bit cache where contents go wrong: values that are no numbers, positions without a block, lengths and
offsets of any content, blocks past 4 GiB. Every request with new tokens has more query rows than the kernel of few rows takes
(64, or 128 where requests times KV heads are at most four), so that the chunk kernel and its join are what runs."""
from __future__ import annotations

import pytest
import torch

from kv4_cases import Requests, check

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]
NAN = float("nan")


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("dtype", TYPES)
def test_no_number_reaches_only_who_attends(D, dtype, device):
    """A key in a tile that every row sees whole, a key and a value in tiles that some rows see: NaN for the rows that attend to
    them (their head's), all others as without, with a window too. 160 rows a request."""
    r = Requests(device, [420, 400], [40, 40], 12, 3, D, dtype=dtype)
    r.k[0][0, 5, 3] = float("inf")
    r.k[0][1, 390, D - 1] = NAN
    r.v[0][2, 400, 40] = float("-inf")
    r.v[1][0, 7, 0] = NAN
    r.store()
    # rows at positions 380..419 of request 0 (tokens 0..39 of q), 360..399 of request 1 (40..79)
    want, bound = r.expected()
    want[0:4, 0:40] = NAN
    want[4:8, 10:40] = NAN
    want[8:12, 20:40] = NAN
    want[0:4, 40:80] = NAN
    assert not torch.isnan(want[4:8, :10]).any() and not torch.isnan(want[8:, :20]).any() and not torch.isnan(want[4:, 40:]).any()
    check(r.attend(), want, bound)
    want, bound = r.expected(window=15)
    want[4:8, 10:25] = NAN
    want[8:12, 20:35] = NAN
    assert int(torch.isnan(want[..., 0]).sum()) == 2 * 4 * 15
    check(r.attend(slide_size=15), want, bound)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("dtype", TYPES)
def test_positions_without_a_block(D, dtype, device):
    """Entries of the table that are no block, between tiles that every row sees whole and on the diagonal: their positions are
    hidden. Then all of a request's: zeros."""
    r = Requests(device, [600, 330], [40, 36], 8, 2, D, dtype=dtype).store()
    held = [torch.ones(n, dtype=torch.bool) for n in r.lens]
    r.table[0, 1], r.table[0, 3], r.table[0, 8] = -1, 1 << 30, r.cache.num_blocks
    for c in (1, 3, 8):
        held[0][c * 64:(c + 1) * 64] = False
    r.table[1, 0], r.table[1, 5] = -(1 << 31), 2 ** 31 - 1
    held[1][:64] = held[1][320:] = False
    check(r.attend(), *r.expected(held=held))
    check(r.attend(slide_size=90), *r.expected(held=held, window=90))
    check(r.attend(causal=False), *r.expected(held=held, causal=False))
    r.table[0] = -1
    held[0][:] = False
    got = r.attend()
    check(got, *r.expected(held=held))
    assert not got[:, :, :40].any()


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_joined_chunks_with_gaps(D, device):
    """A chunk split over its keys whose middle has no blocks and holds a key that is no number: the parts without a visible key
    weigh nothing, and only the rows that see the key answer NaN."""
    r = Requests(device, [2100, 40], [40, 1], 8, 1, D, seed=D)
    r.k[0][0, 2080, 9] = NAN
    r.store()
    held = [torch.ones(n, dtype=torch.bool) for n in r.lens]
    r.table[0, 4:20] = -1
    held[0][256:1280] = False
    want, bound = r.expected(held=held)
    want[:, 20:40] = NAN
    a, b = r.attend(), r.attend()
    check(a, want, bound)
    assert torch.equal(a[:, :, :20], b[:, :, :20]) and torch.equal(a[:, :, 40:], b[:, :, 40:])


@pytest.mark.parametrize("D", [64, 512])
def test_infinite_queries(D, device):
    """Queries with an infinity or NaN: their own rows only."""
    r = Requests(device, [300, 260], [150, 140], 4, 1, D).store()
    clean = r.attend()
    r.q[0, 1, 3, 5], r.q[0, 2, 200, 0] = float("inf"), NAN
    o = r.attend()
    assert torch.isnan(o[0, 1, 3]).all() and torch.isnan(o[0, 2, 200]).all()
    rest = torch.ones(o.shape[1:3], dtype=torch.bool)
    rest[1, 3] = rest[2, 200] = False
    assert torch.equal(o[0][rest], clean[0][rest])


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_contents_of_any_kind(D, device):
    """cu, lens and tables of any content keep the call inside its arrays; with good ones the results are what they were."""
    r = Requests(device, [3000, 300, 260], [140, 150, 1], 8, 1, D, pad=2).store()
    want = r.attend()
    good, lens, table = r.cu.clone(), r.lens_dev.clone(), r.table.clone()
    big, T = 2 ** 31 - 1, 293
    for cu in ([0, big, 290, T], [0, 140, -5, T], [-big, big, 290, T], [200, 0, 290, 291], [big] * 4, [0, 140, 290, -1], [0, T, 0, T]):
        r.cu.copy_(torch.tensor(cu, dtype=torch.int32))
        r.attend()
        r.attend(slide_size=50)
        r.attend(causal=False, max_new=1)
    r.cu.copy_(good)
    for n in ([big, -big, 4], [100000, big, big - 100], [0, 10, 0]):
        r.lens_dev.copy_(torch.tensor(n, dtype=torch.int32))
        r.attend()
        r.attend(slide_size=1000)
        r.attend(causal=False)
    r.lens_dev.copy_(lens)
    r.table.fill_(big)
    assert not r.attend().any()
    r.table.copy_(table)
    assert torch.equal(r.attend(), want)


@pytest.mark.parametrize("D,blocks", [(512, 35000), (64, 280000)])
def test_a_cache_past_4_gib(D, blocks, device):
    from gemma_triton_flash_attn_amd import kv4

    r = Requests(device, [350, 290], [140, 150], 8, 4, D).store()
    big = kv4.allocate(blocks, 4, D, 64, torch.bfloat16, device)
    assert big.codes.numel() > 1 << 32
    shift = blocks - 10 - r.cache.num_blocks
    big.codes[shift:shift + r.cache.num_blocks] = r.cache.codes
    big.scales[shift:shift + r.cache.num_blocks] = r.cache.scales
    o = kv4.attention(r.q.to(device), big, torch.where(r.table >= 0, r.table + shift, -1), r.lens_dev, r.cu)
    assert torch.equal(o, r.attend())


@pytest.mark.parametrize("D", [64, 128])
def test_lengths_past_the_table(D, device):
    """A request longer than its table has places for: what has no entry is not there, for rows whose own position is past it too."""
    r = Requests(device, [300], [80], 2, 1, D).store()
    r.table = r.table[:, :4]  # places for 256 tokens, rows at positions 220..299
    held = torch.ones(300, dtype=torch.bool)
    held[256:] = False
    check(r.attend(), *r.expected(held=[held]))
    check(r.attend(slide_size=30), *r.expected(held=[held], window=30))
    check(r.attend(causal=False), *r.expected(held=[held], causal=False))
