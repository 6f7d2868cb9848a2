"""The cache operators where calls go past the usual: rows of no request, many requests, contents that are no places."""
from __future__ import annotations

import pytest
import torch

from kv4_cases import Requests, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,new", [([90, 40], [1, 2]), ([400, 260, 33], [150, 200, 1])])
def test_rows_ahead_of_the_first_request(lens, new, device):
    """Offsets that begin past q's first token: the rows ahead are zeros, whatever their memory held, the others as without."""
    from gemma_triton_flash_attn_amd import kv4

    r = Requests(device, lens, new, 8, 2, 128, pad=2).store()
    want = r.attend()
    q = torch.cat([torch.randn(1, 8, 5, 128).to(r.dtype), r.q], 2).to(device)
    for _ in range(3):
        stale = torch.full_like(q, float("nan"))  # the memory that the output is likely to get
        del stale
        o = kv4.attention(q, r.cache, r.table, r.lens_dev, r.cu + 5)
        assert not o[:, :, :5].any() and torch.equal(o[:, :, 5:], want)


def _split_parts(r, rows, target, min_tiles):
    """Parts that the call leaves for the join, by the device's own count restated (test_kv4_cpu)."""
    from test_kv4_cpu import _items

    G = r.Hq // r.Hkv
    limit = 64  # more than four requests and heads
    mine = [(n, k) for n, k in zip(r.lens, r.new) if (k * G > limit) == (rows > 16)]
    return _items([n for n, _ in mine], [k for _, k in mine], G, r.Hkv, rows, target, 0, min_tiles)[1]


@pytest.mark.parametrize("count", [65, 130, 200])
@pytest.mark.parametrize("D,Hq,Hkv", [(64, 4, 2), (256, 2, 1)])
def test_joined_rows_of_many_requests(D, Hq, Hkv, count, device):
    """Few rows over long axes, more requests than a wave has lanes."""
    lens = [1500 + 17 * (i % 13) if i % 5 == 2 else 5 + 3 * (i % 40) for i in range(count)]
    new = [(1, 2, 1, 3)[i % 4] for i in range(count)]
    r = Requests(device, lens, new, Hq, Hkv, D, 32, pad=9, seed=count).store()
    assert _split_parts(r, 16, 512, 8) > 0
    a = r.attend()
    check(a, *r.expected())
    assert torch.equal(a, r.attend())


@pytest.mark.parametrize("count", [65, 130])
def test_joined_chunks_of_many_requests(count, device):
    """Chunks of 80 rows beside single tokens, more requests than a wave has lanes, long ones split over their keys in both
    kernels."""
    lens = [1500 + 17 * (i % 13) if i % 5 == 2 else 45 + 3 * (i % 40) for i in range(count)]
    new = [40 if i % 10 == 2 else 1 for i in range(count)]
    r = Requests(device, lens, new, 2, 1, 64, 32, pad=5, seed=count).store()
    assert _split_parts(r, 16, 512, 8) > 0 and _split_parts(r, 256, 512, 8) > 0
    a = r.attend()
    check(a, *r.expected())
    assert torch.equal(a, r.attend())
    check(r.attend(slide_size=700), *r.expected(window=700))
