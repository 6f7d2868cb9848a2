"""Which calls with shared prefixes are the call without them by the host's rule: seen in the workspace that it asks for."""
from __future__ import annotations

import ctypes

import pytest

from gemma_triton_flash_attn_amd import _lib
from test_kv4_sharing_cpu import _attn, _cache

SHARED = dict(shared_skip=64, shared_cu=64, shared_lens=64)


def _bytes(Hq, Hkv, D, bs, softcap, R, width, new, **kw):
    return _lib.load().gfa_kv4_attn_workspace_bytes(ctypes.byref(_attn(
        cache=_cache(heads_kv=Hkv, head_dim=D, block_size=bs), heads_q=Hq, softcap=softcap, requests=R, seq_len=R * new,
        table_width=width, table_stride=width, max_new=new, **kw)))


@pytest.mark.parametrize("call,plain", [
    ((8, 4, 256, 64, 50.0, 16, 55, 4), True),     # 16 answers of 4 drafted tokens, 3k
    ((16, 8, 256, 64, 0.0, 64, 8, 1), True),      # 64 short requests
    ((32, 8, 128, 64, 0.0, 6, 94, 2), True),      # two answers to each of three prompts of 6k
    ((8, 1, 512, 64, 0.0, 4, 16, 1), True),       # four answers to a short question
    ((32, 8, 128, 64, 0.0, 64, 268, 1), False),   # 64 answers to a 16k prompt
    ((32, 4, 512, 64, 0.0, 32, 146, 1), False),   # eight answers to each of four prompts of 8k
    ((8, 1, 512, 64, 0.0, 26, 26, 8), False),     # at D = 512 the shared launch gains by itself
    ((8, 4, 256, 64, 50.0, 16, 300, 4), False),   # the drafts in a wide table
])
def test_tables_too_narrow(call, plain):
    without = _bytes(*call)
    assert (_bytes(*call, **SHARED) == without) == plain
    assert _bytes(*call, shared_apart=1, **SHARED) != without
