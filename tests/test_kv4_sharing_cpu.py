"""The operators of requests with something in common without a GPU: the oracle's own rules by hand, refusals before any launch, the
C layout, workspaces."""
from __future__ import annotations

import ctypes
import os
import random
import shutil
import subprocess

import pytest
import torch

from gemma_triton_flash_attn_amd import _lib, kv4
from oracle import kv4_sharing_oracle as orc
from test_kv4_cpu import HEADER, INVALID, UNSUPPORTED, WORKSPACE, _attn, _cache, _codes, _Held, no_gpu


# ---- the oracle ----

def test_fork_by_hand():
    free = [7, 3, 5, 0, 1, 9, 2]
    # row 0 goes on from request 0 inside its second block, row 1 as well, row 2 keeps request 1's first block whole
    got = orc.fork([[7, 3, -1], [7, 5, 0]], [40, 70], [0, 0, 1], [40, 33, 32], free, 4, 32, 10)
    assert got == ([[7, 3, -1], [7, 0, -1], [7, -1, -1]], [40, 33, 32], 3, [(3, 0)])
    assert free == [7, 3, 0, 5, 1, 9, 2]  # 0 and 5 came back, 0 was taken again


def test_a_part_of_a_block_that_another_row_holds_whole():
    free = [4, 6, 1]
    got = orc.fork([[4], [4]], [32, 32], None, [32, 10], free, 2, 32, 8)
    assert got == ([[4], [1]], [32, 10], 3, [(4, 1)]) and free == [4, 6, 1]


def test_compact_by_hand():
    table, n, pairs = orc.compact([[9, 2, 0], [9, 5, 7]], [64, 96], 32, 12)
    assert n == 4 and pairs == [(5, 0), (7, 1), (9, 3)] and table == [[3, 2, -1], [3, 0, 1]]


def test_share_by_hand():
    table = [[5, 6, 7, 1], [5, 6, 7, 2], [5, 6, 8, 3], [9, 6, 7, 1], [9, 4, 0, 0]]
    assert orc.share(table, [256, 250, 200, 130, 70], [0, 1, 3, 4, 5, 6], 64, 64) == (
        [128, 128, 128, 64, 64], [0, 4, 4, 4, 6, 6], [128, 0, 0, 64, 0])


def test_verify_by_hand():
    p = [[0.25, 0.75, 0.0], [0.5, 0.25, 0.25], [0.0, 0.0, 1.0]]
    q = [[1.0, 0.0, 0.0], [0.5, 0.5, 0.0], [0.25, 0.25, 0.5]]
    # token 1 is accepted (0.9 0.5 < 0.75), token 2 is not (0.6 0.5 >= 0.25): 0.25 of max(p - q, 0) is 0's
    assert orc.verify(p, q, [0, 1, 2], [0.0, 0.9, 0.6], [0.9], [10], [0, 3]) == ([1, 0, -1], [1], [9])
    assert orc.verify(p, q, [0, 1, 2], [0.0, 0.9, 0.4], [0.9], [10], [0, 3]) == ([1, 2, 2], [2], [10])
    assert orc.verify(p, None, [0, 1, 2], [0.0, 0.7, 0.3], [0.5], [10], [0, 3]) == ([1, 0, -1], [1], [9])


def test_verified_tokens_have_the_targets_distribution():
    """Over a grid of random numbers the oracle's first token is distributed as the target's, exactly."""
    p, q = [0.5, 0.125, 0.375], [0.25, 0.5, 0.25]
    count = [0, 0, 0]
    n = 64
    for x, weight in ((0, 1), (1, 2), (2, 1)):  # the draft's token, by its probability
        for i in range(n):
            for j in range(n):
                got = orc.verify([p, p], [q, q], [0, x], [0.0, (i + 0.5) / n], [(j + 0.5) / n], [5], [0, 2])
                count[got[0][0]] += weight
    assert [c / (4 * n * n) for c in count] == pytest.approx(p, abs=2 / n)


# ---- refusals of the Python entry points ----

def _ints(*s):
    return torch.zeros(*s, dtype=torch.int32)


def test_python_refusals():
    c = _Held(*_codes(), torch.bfloat16)
    t, lens, free, used = _ints(3, 2), _ints(3), _ints(2), _ints(1)
    for call in (lambda: kv4.fork([], t, lens, free, used), lambda: kv4.compact([], t, lens, free), lambda: kv4.copy([], used, used)):
        with pytest.raises(ValueError, match="at least one cache"):
            call()
    for call in (lambda: kv4.fork(c, t, lens, free, used), lambda: kv4.compact([c], t, lens, free), lambda: kv4.copy(c, used, used),
                 lambda: kv4.share(t, lens, _ints(4), block_size=64)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    p = torch.zeros(3, 5)
    x = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        kv4.verify(p, p, x, torch.zeros(3), torch.zeros(3), lens)
    with pytest.raises(TypeError, match="target is"):
        kv4.verify(p.double(), None, x, torch.zeros(3), torch.zeros(3), lens)
    with pytest.raises(TypeError, match="lens must be"):
        kv4.share(t, lens.long(), _ints(4), block_size=64)


def test_probabilities_that_want_a_gradient():
    p, x = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64)
    args = (x, torch.zeros(3), torch.zeros(3), _ints(3))
    for target, draft in ((p.clone().requires_grad_(True), p), (p, p.clone().requires_grad_(True)), (p.clone().requires_grad_(True), None)):
        with pytest.raises(NotImplementedError, match="no gradient"):
            kv4.verify(target, draft, *args)
        with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
            kv4.verify(target, draft, *args)


# ---- the C ABI ----

@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layout_matches_c(tmp_path):
    structs = {"gfa_kv4_pages_args": _lib.Kv4PagesArgs, "gfa_kv4_share_args": _lib.Kv4ShareArgs, "gfa_kv4_verify_args": _lib.Kv4VerifyArgs}
    lines = []
    for name, cls in structs.items():
        lines.append(f'printf("%zu ", sizeof({name}));')
        lines += [f'printf("%zu ", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{ {" ".join(lines)} return 0; }}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for cls in structs.values():
        want.append(ctypes.sizeof(cls))
        want += [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


def _pages(caches=None, **over):
    a = _lib.Kv4PagesArgs()
    caches = [_cache(), _cache(heads_kv=1, head_dim=64)] if caches is None else caches
    a.caches = (_lib.Kv4Cache * len(caches))(*caches) if caches else None
    a.layers = len(caches)
    for f in ("table", "lens", "parents", "keep", "free_ids", "used", "table_out", "lens_out", "used_out", "workspace"):
        setattr(a, f, 64)
    a.table_stride, a.requests, a.table_width, a.rows, a.free_count, a.workspace_bytes = 4, 2, 4, 5, 10, 1 << 30
    for k, v in over.items():
        setattr(a, k, v)
    return a


@no_gpu
@pytest.mark.parametrize("over,status", [
    (dict(caches=[]), INVALID), (dict(caches=[_cache(codes=0)]), INVALID), (dict(caches=[_cache(), _cache(num_blocks=11)]), INVALID),
    (dict(caches=[_cache(), _cache(block_size=32)]), INVALID), (dict(caches=[_cache(num_blocks=(1 << 18) + 1)], free_count=(1 << 18) + 1), UNSUPPORTED),
    (dict(requests=0), INVALID), (dict(requests=4097), UNSUPPORTED), (dict(table_width=0), INVALID), (dict(table_width=1 << 25, table_stride=1 << 25), UNSUPPORTED),
    (dict(table_stride=3), INVALID), (dict(table=0), INVALID), (dict(table=2), INVALID), (dict(lens=0), INVALID), (dict(free_ids=0), INVALID),
    (dict(free_count=-1), INVALID), (dict(table_out=0), INVALID), (dict(used_out=2), INVALID), (dict(workspace=0), WORKSPACE),
    (dict(workspace_bytes=8), WORKSPACE)])
def test_page_refusals(over, status):
    lib = _lib.load()
    for fn in (lib.gfa_kv4_fork, lib.gfa_kv4_compact):
        assert fn(ctypes.byref(_pages(**over))) == status, lib.gfa_last_error()
    assert lib.gfa_last_error()


@no_gpu
def test_refusals_of_one():
    lib = _lib.load()
    assert lib.gfa_kv4_fork(None) == lib.gfa_kv4_compact(None) == lib.gfa_kv4_share(None) == lib.gfa_kv4_verify(None) == INVALID
    for over, status in [(dict(rows=0), INVALID), (dict(rows=4097), UNSUPPORTED), (dict(parents=2), INVALID), (dict(keep=6), INVALID),
                         (dict(used=0), INVALID), (dict(lens_out=0), INVALID)]:
        assert lib.gfa_kv4_fork(ctypes.byref(_pages(**over))) == status, over
    # a compacted pool's free list is all of it
    assert lib.gfa_kv4_compact(ctypes.byref(_pages(free_count=9))) == INVALID
    one = (_lib.Kv4Cache * 1)(_cache())
    assert lib.gfa_kv4_copy(None, 0, 64, 64, 1, None) == lib.gfa_kv4_copy(one, 1, 0, 64, 1, None) == lib.gfa_kv4_copy(one, 1, 64, 2, 1, None) == INVALID
    assert lib.gfa_kv4_copy(one, 1, 64, 64, -1, None) == INVALID and lib.gfa_kv4_copy(one, 1, 0, 0, 0, None) == 0
    big = (_lib.Kv4Cache * 1)(_cache(heads_kv=4096, block_size=1024, head_dim=512))
    assert lib.gfa_kv4_copy(big, 1, 64, 64, 1 << 20, None) == UNSUPPORTED


@no_gpu
def test_share_refusals():
    def share(**over):
        a = _lib.Kv4ShareArgs()
        for f in ("table", "lens", "cu", "skip", "cu_out", "lens_out"):
            setattr(a, f, 64)
        a.table_stride, a.requests, a.table_width, a.block_size, a.least = 4, 2, 4, 64, 512
        for k, v in over.items():
            setattr(a, k, v)
        return a

    lib = _lib.load()
    for over, status in [(dict(block_size=48), UNSUPPORTED), (dict(requests=0), INVALID), (dict(requests=4097), UNSUPPORTED), (dict(least=0), INVALID),
                         (dict(table_width=0), INVALID), (dict(table_width=1 << 25, table_stride=1 << 25), UNSUPPORTED), (dict(table_stride=3), INVALID),
                         (dict(cu=0), INVALID), (dict(skip=2), INVALID), (dict(lens_out=0), INVALID)]:
        assert lib.gfa_kv4_share(ctypes.byref(share(**over))) == status, over


@no_gpu
def test_verify_refusals():
    def verify(**over):
        a = _lib.Kv4VerifyArgs()
        for f in ("target", "draft", "tokens", "accept", "sample", "lens", "cu", "follows", "accepted", "lens_out", "workspace"):
            setattr(a, f, 64)
        a.target_stride = a.draft_stride = 100
        a.type, a.token_count, a.vocab, a.requests, a.workspace_bytes = 2, 7, 100, 3, 1 << 40
        for k, v in over.items():
            setattr(a, k, v)
        return a

    lib = _lib.load()
    for over, status in [(dict(target=0), INVALID), (dict(target=2), INVALID), (dict(draft=66), INVALID), (dict(type=3), INVALID), (dict(token_count=0), INVALID),
                         (dict(vocab=0), INVALID), (dict(vocab=(1 << 30) + 1), UNSUPPORTED), (dict(requests=0), INVALID), (dict(requests=65536), UNSUPPORTED),
                         (dict(requests=65535, vocab=1 << 30), UNSUPPORTED), (dict(cu=0), INVALID), (dict(cu=2), INVALID), (dict(tokens=4), INVALID),
                         (dict(follows=4), INVALID), (dict(accept=0), INVALID), (dict(lens=2), INVALID), (dict(target_stride=-1), INVALID),
                         (dict(workspace=4), WORKSPACE), (dict(workspace_bytes=71), WORKSPACE)]:
        assert lib.gfa_kv4_verify(ctypes.byref(verify(**over))) == status, over


@no_gpu
@pytest.mark.parametrize("over,status", [
    (dict(shared_skip=2), INVALID), (dict(shared_cu=0), INVALID), (dict(shared_lens=6), INVALID), (dict(cu=0), INVALID), (dict(workspace_bytes=64), WORKSPACE)])
def test_shared_attention_refusals(over, status):
    lib = _lib.load()
    a = dict(shared_skip=64, shared_cu=64, shared_lens=64, shared_apart=1, max_new=1)
    assert lib.gfa_kv4_attn(ctypes.byref(_attn(**{**a, **over}))) == status, lib.gfa_last_error()


# ---- what the host sizes for shared prefixes ----

def _parts(a, heads, D, besides):
    """(chunk kernel's slots, split kernel's) that the workspace can be made of: rows of sums and two statistics each."""
    need = _lib.load().gfa_kv4_attn_workspace_bytes(ctypes.byref(a)) - besides
    assert need % (heads * (D + 2) * 4 * 16) == 0
    return need // (heads * (D + 2) * 4)  # rows


@pytest.mark.parametrize("seed", range(30))
def test_the_workspace_holds_every_part(seed):
    """Every item of the groups' prefixes and of the requests' rests has a slot: rows of the workspace are at least those of the
    items that the device makes of any groups (gfa_kv4_sched.h, with the host's own targets left out: what row blocks there are at
    least, and the bound's growth with the requests)."""
    rng = random.Random(seed)
    D, G, Hkv = rng.choice([64, 128, 256, 512]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
    R, n = rng.choice([2, 5, 64, 300]), rng.choice([1, 1, 2, 5])
    if n * G > 64:
        n = 1
    a = _attn(cache=_cache(heads_kv=Hkv, head_dim=D), heads_q=G * Hkv, requests=R, seq_len=R * n, table_width=300, table_stride=300, max_new=n,
              shared_skip=64, shared_cu=64, shared_lens=64, shared_apart=1)
    rows = _parts(a, Hkv, D, 64 + (R * n * G + 15 * R) // 16 * 48)  # and where each row block's sums are
    big = 128 if D >= 128 else 256
    # any cut of the requests into groups of two and more
    left, groups = R, []
    while left >= 2:
        k = min(left, rng.choice([2, 3, 10, 70]))
        groups.append(k)
        left -= k
    limit = 32 if Hkv >= 4 and D >= 128 else 64
    blocks = sum(-(-n * G // 16) for _ in range(R)) * 16
    blocks += sum(-(-k * n * G // 16) * 16 if k * n * G <= limit else -(-k * n * G // big) * big for k in groups)
    assert rows >= blocks


def test_workspace_without_effect():
    """With a window, or for requests of many rows, the call is the plain one."""
    ws = lambda **k: _lib.load().gfa_kv4_attn_workspace_bytes(ctypes.byref(_attn(**k)))  # noqa: E731
    shared = dict(shared_skip=64, shared_cu=64, shared_lens=64)
    assert ws(max_new=1) != ws(max_new=1, shared_apart=1, **shared) and ws(max_new=1) == ws(max_new=1, shared_apart=1)
    wide = dict(table_width=10000, table_stride=10000, requests=64, seq_len=64, max_new=1)
    assert ws(**wide) != ws(**wide, **shared) == ws(**wide, **shared, shared_apart=1)
    narrow = dict(wide, table_width=1, table_stride=1)  # nothing there that would pay
    assert ws(**narrow) == ws(**narrow, **shared) != ws(**narrow, **shared, shared_apart=1)
    assert ws(window=3000, max_new=1) == ws(window=3000, max_new=1, **shared)
    assert ws(max_new=100, seq_len=400) == ws(max_new=100, seq_len=400, **shared)
    assert ws(requests=1, max_new=1) == ws(requests=1, max_new=1, **shared)


def test_page_workspace():
    lib = _lib.load()
    assert lib.gfa_kv4_pages_workspace_bytes(7) == 60 and lib.gfa_kv4_pages_workspace_bytes(-1) == 0
    for R, V in ((1, 1), (1, 512), (3, 513), (64, 262144), (65535, 1000)):
        step = min(4, -(-V * R // (4096 * 512))) * 512
        assert lib.gfa_kv4_verify_workspace_bytes(R, V) == R * (-(-V // step) * 16 + 8)
    assert lib.gfa_kv4_verify_workspace_bytes(0, 5) == 0 and os.path.exists(HEADER)
