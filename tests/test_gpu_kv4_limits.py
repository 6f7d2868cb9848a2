"""The cache operators where calls go past the usual: rows of no request, many requests, contents that are no places."""
from __future__ import annotations

import pytest
import torch

from kv4_cases import Requests

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
