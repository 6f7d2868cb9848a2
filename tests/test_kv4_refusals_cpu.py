"""What the cache operators refuse, each by its message, on CPU tensors: none of it comes as far as the device's refusal."""
from __future__ import annotations

import pytest
import torch

from gemma_triton_flash_attn_amd import kv4
from test_kv4_cpu import _codes, _Held


def _ints(*s):
    return torch.zeros(*s, dtype=torch.int32)


def _rows(h, **kw):
    return torch.zeros(1, h, 3, 128, dtype=torch.bfloat16, **kw)


SLOTS = torch.zeros(3, dtype=torch.int64)


@pytest.mark.parametrize("which", ["k", "v"])
def test_rows_that_want_a_gradient(which):
    """Stored rows keep no graph: a write of rows that want one would cut their gradients off unseen."""
    c = _Held(*_codes(), torch.bfloat16)
    rows = {"k": _rows(2), "v": _rows(2)}
    rows[which] = rows[which].requires_grad_(True)
    with pytest.raises(NotImplementedError, match="no gradient"):
        kv4.write(c, rows["k"], rows["v"], SLOTS)
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):  # past it, to the device's refusal
        kv4.write(c, rows["k"], rows["v"], SLOTS)


def test_forward_mode_tangents():
    """A dual tensor's tangent would be dropped, under no_grad too (which does not end forward mode): refused."""
    c = _Held(*_codes(), torch.bfloat16)
    calls = [lambda x: kv4.attention(x, c, _ints(3, 2), _ints(3)),
             lambda x: kv4.write(c, x[:, :2], _rows(2), SLOTS), lambda x: kv4.write(c, _rows(2), x[:, :2], SLOTS)]
    for call in calls:
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(_rows(4), torch.ones_like(_rows(4)))
            with pytest.raises(NotImplementedError, match="no gradient"):
                call(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="no gradient"):
                call(dual)
            with pytest.raises(ValueError, match="GPU"):  # rows without a tangent pass
                call(_rows(4))
        with pytest.raises(NotImplementedError, match="no gradient"):
            torch.func.jvp(call, (_rows(4),), (torch.ones_like(_rows(4)),))


@pytest.mark.parametrize("over,exc,message", [
    (dict(max_new=0), ValueError, "max_new"), (dict(max_new=-3), ValueError, "max_new"), (dict(softcap=-1.0), ValueError, "softcap"),
    (dict(softcap=float("nan")), ValueError, "softcap")])
def test_options_of_attention(over, exc, message):
    c = _Held(*_codes(), torch.bfloat16)
    with pytest.raises(exc, match=message):
        kv4.attention(_rows(4), c, _ints(3, 2), _ints(3), **over)


@pytest.mark.parametrize("arrays,exc,message", [
    (lambda c, s: (c.float(), s), TypeError, "uint8"), (lambda c, s: (c, s.float()), TypeError, "uint8"),
    (lambda c, s: (c[0], s), ValueError, "5-D"), (lambda c, s: (c, s[:1]), ValueError, "belong together"),
    (lambda c, s: (c[..., ::2], s), ValueError, "belong together"), (lambda c, s: _codes(bs=16), ValueError, "block_size"),
    (lambda c, s: _codes(bs=96), ValueError, "block_size"), (lambda c, s: _codes(d=96), ValueError, "HEAD_DIM"),
    (lambda c, s: _codes(n=0), ValueError, "0 blocks"), (lambda c, s: (c, s), ValueError, "GPU"),
    (lambda c, s: (c.transpose(0, 1).contiguous().transpose(0, 1), s), ValueError, "contiguous")])
def test_caches(arrays, exc, message):
    with pytest.raises(exc, match=message):
        kv4.Cache(*arrays(*_codes()), torch.bfloat16)
