"""What the cache operators refuse, each by its message, on CPU tensors: none of it comes as far as the device's refusal."""
from __future__ import annotations

import ctypes

import pytest
import torch

from gemma_triton_flash_attn_amd import _lib, kv4
from test_kv4_cpu import UNSUPPORTED, _attn, _cache, _codes, _Held, no_gpu


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


@no_gpu
def test_grids_past_one_launch():
    """A launch holds fewer than 2^32 threads, 2^24 workgroups of 256: calls that would need more are refused for what they are,
    not by whatever the runtime says. Calls just below come as far as the launch, which fails for want of a GPU."""
    lib = _lib.load()
    wide = lambda heads, requests: _attn(cache=_cache(heads_kv=heads), heads_q=heads, cu=0, requests=requests, seq_len=requests)  # noqa: E731
    for heads, requests, status in ((256, 65536, UNSUPPORTED), (65535, 256, UNSUPPORTED), (255, 65535, 4)):
        got = lib.gfa_kv4_attn(ctypes.byref(wide(heads, requests)))
        assert got == status, (heads, requests, got, lib.gfa_last_error())

    a = _lib.Kv4RowsArgs()
    a.k = a.v = 256
    a.k_strides = a.v_strides = _lib.Strides(0, 128, 256)
    a.batch, a.slots = 1, 64
    # a wave holds 2048 / head_dim tokens of a head
    for heads, tokens, D, status in ((1 << 10, 1 << 18, 512, UNSUPPORTED), (1 << 10, (1 << 18) - 4, 512, 4), (1 << 13, 1 << 18, 64, UNSUPPORTED)):
        a.cache, a.seq_len = _cache(heads_kv=heads, head_dim=D), tokens
        for fn in (lib.gfa_kv4_write, lib.gfa_kv4_read):
            assert fn(ctypes.byref(a)) == status, (heads, tokens, D, lib.gfa_last_error())
