"""The key/value cache in 4 bits without a GPU: the oracle's own rules, refusals before any launch, the C layout, and that the
workspace the host sizes holds the partial sums of any lengths."""
from __future__ import annotations

import ctypes
import math
import os
import random
import shutil
import subprocess

import numpy as np
import pytest
import torch

import gemma_triton_flash_attn_amd as gfa
from gemma_triton_flash_attn_amd import _lib, kv4
from oracle import kv4_oracle as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "gfa.h")
CSRC = os.path.join(ROOT, "gemma-triton-flash-attn_amd", "csrc")
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="passes fake device pointers; runs only without a visible GPU")


# ---- the format ----

def test_rounding_by_hand():
    x = torch.zeros(1, 32, dtype=torch.bfloat16)
    x[0, :8] = torch.tensor([6.0, 5.0, 2.5, -1.75, 0.25, 0.75, -3.5, 0.2])
    assert orc.rounded(x)[0, :8].tolist() == [6.0, 4.0, 2.0, -2.0, 0.0, 1.0, -4.0, 0.0]
    x[0, 0] = 7.0  # the midpoint of 6 and the next scale's 8 stays, and saturates
    assert orc.rounded(x)[0, 0] == 6.0
    x[0, 0] = 7.03125  # the next bf16: the scale doubles
    assert orc.rounded(x)[0, :4].tolist() == [8.0, 4.0, 2.0, -2.0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rounding_errors(dtype):
    """Each value is off by at most a quarter of its block's largest / 4 (half of the widest step, 2 in 7), or saturates by 1/7."""
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(200, 256, generator=g) * torch.exp(3 * torch.randn(200, 1, generator=g))).to(dtype)
    y = orc.rounded(x)
    top = x.double().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, 32).flatten(-2)
    assert ((x.double() - y).abs() <= top / 3.5 + 2.0 ** -24).all()
    assert (y.abs() <= torch.finfo(dtype).max).all() and torch.equal(y.to(dtype).double(), y)
    err = torch.linalg.norm(x.double() - y) / torch.linalg.norm(x.double())
    assert 0.09 < err < 0.13


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_ends_of_the_range(dtype):
    info = torch.finfo(dtype)
    x = torch.full((1, 32), info.max, dtype=dtype)
    assert torch.isfinite(orc.rounded(x).to(dtype)).all()
    x[0, 1:] = 0
    x[0, 0] = info.tiny / 64
    y = orc.rounded(x)
    assert torch.equal(y.to(dtype).double(), y)
    assert not orc.rounded(torch.zeros(1, 32, dtype=dtype)).any()


def test_plan_by_hand():
    table = [[7, -1, -1], [-1, -1, -1], [3, 4, -1]]
    got = orc.plan([30, 0, 64], [4, 0, 1], table, [9, 1, 2], 1, 32, 7)
    assert got == ([254, 255, 32, 33, 64, -1, -1], [30, 31, 32, 33, 64, 0, 0], [0, 4, 4, 5], [34, 0, 65], 3)
    assert table == [[7, 1, -1], [-1, -1, -1], [3, 4, 2]]


# ---- refusals of the Python entry points ----

def _codes(n=2, h=2, bs=64, d=128):
    return torch.zeros(n, h, 2, bs, d // 2, dtype=torch.uint8), torch.zeros(n, h, 2, bs, d // 32, dtype=torch.uint8)


def test_cache_refusals():
    c, s = _codes()
    for bad in (lambda: kv4.Cache(c, s, torch.float32), lambda: kv4.Cache(c.float(), s, torch.bfloat16)):
        with pytest.raises(TypeError):
            bad()
    for cc, ss in [(c[0], s), (c, s[:1]), _codes(bs=16), _codes(bs=96), _codes(d=96), (c[..., ::2], s), _codes(n=0), (c, s)]:
        with pytest.raises(ValueError):  # the last for its device: there is no CPU path
            kv4.Cache(cc, ss, torch.bfloat16)
    with pytest.raises(ValueError):
        kv4.allocate(4, 2, 128, block_size=48, device="cpu")
    with pytest.raises(ValueError):
        kv4.allocate(4, 2, 96, device="cpu")


def test_plan_refusals():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    good = dict(lens=i(3), new=i(3), table=i(3, 4), free=i(5), used=i(1))

    def call(block_size=64, tokens=4, **over):
        a = {**good, **over}
        return kv4.plan(a["lens"], a["new"], a["table"], a["free"], a["used"], block_size=block_size, tokens=tokens)

    with pytest.raises(TypeError):
        call(lens=i(3).long())
    for over in (dict(lens=i(3, 1)), dict()):
        with pytest.raises(ValueError):
            call(**over)


class _Held(kv4.Cache):
    """A cache of CPU tensors, past the constructor's refusal: every call refuses it again."""

    def __init__(self, codes, scales, dtype):
        self.codes, self.scales, self.dtype = codes, scales, dtype


def test_call_refusals():
    c = _Held(*_codes(), torch.bfloat16)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    q = torch.zeros(1, 4, 3, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        kv4.attention(q, c, i(3, 2), i(3))
    with pytest.raises(ValueError):
        kv4.attention(q, c, i(3, 2), i(3), max_new=0)
    with pytest.raises(ValueError):
        kv4.attention(q, c, i(3, 2), i(3), softcap=-1.0)
    with pytest.raises(NotImplementedError):
        kv4.attention(q.requires_grad_(True), c, i(3, 2), i(3))
    with pytest.raises(ValueError):
        kv4.write(c, q[:, :2].detach(), q[:, :2].detach(), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError):
        kv4.read(c, torch.zeros(3, dtype=torch.int64))


# ---- the C ABI ----

@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layout_matches_c(tmp_path):
    structs = {"gfa_kv4_cache": _lib.Kv4Cache, "gfa_kv4_rows_args": _lib.Kv4RowsArgs, "gfa_kv4_plan_args": _lib.Kv4PlanArgs,
               "gfa_kv4_attn_args": _lib.Kv4AttnArgs}
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


def _cache(**over):
    c = _lib.Kv4Cache(4096, 8192, 10, 2, 64, 128, _lib.GFA_DTYPE_BF16)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def _attn(**over):
    a = _lib.Kv4AttnArgs()
    a.cache = over.pop("cache", _cache())
    a.q = a.o = 256
    a.q_strides = a.o_strides = _lib.Strides(8 * 128, 128, 8 * 128)
    a.batch, a.heads_q, a.seq_len, a.requests = 1, 8, 4, 4
    a.table, a.table_stride, a.lens, a.cu = 256, 40, 512, 1024
    a.table_width, a.causal, a.scale = 40, 1, 0.1
    a.workspace, a.workspace_bytes = 4096, 1 << 40
    for k, v in over.items():
        setattr(a, k, v)
    return a


INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3


@no_gpu
@pytest.mark.parametrize("over,status", [
    (dict(q=0), INVALID), (dict(o=8), INVALID), (dict(table=2), INVALID), (dict(lens=0), INVALID), (dict(cu=2), INVALID),
    (dict(batch=0), INVALID), (dict(requests=0), INVALID), (dict(table_width=0), INVALID), (dict(heads_q=3), INVALID),
    (dict(scale=0.0), INVALID), (dict(scale=math.nan), INVALID), (dict(softcap=-1.0), INVALID), (dict(softcap=math.inf), INVALID),
    (dict(window=-1), INVALID), (dict(max_new=-1), INVALID), (dict(table_stride=3), INVALID), (dict(cu=0, seq_len=5), INVALID),
    (dict(q_strides=_lib.Strides(1024, 128, 1025)), INVALID), (dict(q_strides=_lib.Strides(1024, -128, 1024)), INVALID),
    (dict(requests=70000, cu=0, seq_len=70000), UNSUPPORTED), (dict(table_width=1 << 26), UNSUPPORTED),
    (dict(seq_len=1 << 29), UNSUPPORTED), (dict(workspace=0), WORKSPACE), (dict(workspace_bytes=64), WORKSPACE),
    (dict(workspace=4100), WORKSPACE), (dict(cache=_cache(codes=0)), INVALID), (dict(cache=_cache(scales=8)), INVALID),
    (dict(cache=_cache(head_dim=96)), UNSUPPORTED), (dict(cache=_cache(block_size=48)), UNSUPPORTED),
    (dict(cache=_cache(block_size=16)), UNSUPPORTED), (dict(cache=_cache(num_blocks=0)), INVALID), (dict(cache=_cache(dtype=7)), INVALID)])
def test_attention_refusals(over, status):
    lib = _lib.load()
    assert lib.gfa_kv4_attn(ctypes.byref(_attn(**over))) == status, lib.gfa_last_error()
    assert lib.gfa_last_error()


@no_gpu
def test_other_refusals():
    lib = _lib.load()
    assert lib.gfa_kv4_attn(None) == lib.gfa_kv4_write(None) == lib.gfa_kv4_read(None) == lib.gfa_kv4_plan(None) == INVALID

    def rows(**over):
        a = _lib.Kv4RowsArgs()
        a.cache = over.pop("cache", _cache())
        a.k = a.v = 256
        a.k_strides = a.v_strides = _lib.Strides(1024, 128, 256)
        a.batch, a.seq_len, a.slots = 1, 4, 64
        for k, v in over.items():
            setattr(a, k, v)
        return a

    for over, status in [(dict(k=0), INVALID), (dict(v=8), INVALID), (dict(slots=4), INVALID), (dict(seq_len=0), INVALID),
                         (dict(k_strides=_lib.Strides(4, 128, 256)), INVALID), (dict(batch=1 << 16, seq_len=1 << 15), UNSUPPORTED),
                         (dict(cache=_cache(head_dim=32)), UNSUPPORTED)]:
        for fn in (lib.gfa_kv4_write, lib.gfa_kv4_read):
            assert fn(ctypes.byref(rows(**over))) == status, over

    def plan(**over):
        a = _lib.Kv4PlanArgs()
        for f in ("lens", "fresh", "table", "free_ids", "used", "slots", "positions", "cu", "lens_out", "used_out"):
            setattr(a, f, 64)
        a.table_stride, a.requests, a.table_width, a.free_count, a.block_size, a.tokens = 4, 2, 4, 5, 64, 7
        for k, v in over.items():
            setattr(a, k, v)
        return a

    for over, status in [(dict(lens=0), INVALID), (dict(table=2), INVALID), (dict(slots=4), INVALID), (dict(requests=0), INVALID),
                         (dict(table_width=0), INVALID), (dict(table_stride=3), INVALID), (dict(free_ids=0), INVALID),
                         (dict(tokens=-1), INVALID), (dict(free_count=-1), INVALID), (dict(block_size=31), UNSUPPORTED),
                         (dict(used_out=1), INVALID)]:
        assert lib.gfa_kv4_plan(ctypes.byref(plan(**over))) == status, over


# ---- the work split ----

def _items(lens, new, G, Hkv, rows, target, window, min_tiles):
    """(work items, those of split row blocks) of one kernel for these requests, as the device counts them
    (gfa_kv4_sched.h)."""
    f32 = np.float32
    blocks, tiles = [], []
    for n, k in zip(lens, new):
        blocks.append(-(-k * G // rows))
        lo = max(n - k - window + 1, 0) if window else 0
        t = -(-n // 32) - lo // 32 if n > lo else 0
        if window:
            t = min(t, (window + (rows + G - 2) // G + 1 + 29) // 32 + 1)
        tiles.append(t)
    total = f32(0)
    for b, t in zip(blocks, tiles):
        total = f32(total + f32(f32(b) * f32(t)))
    share = f32(Hkv / target * (1.0 + 1.0 / 4096))
    per = max(int(min(math.ceil(f32(total * share)), 1e9)), min_tiles)
    counts = [(b, max(1, -(-t // per))) for b, t in zip(blocks, tiles)]
    return sum(b * n for b, n in counts), sum(b * n for b, n in counts if n > 1)


@pytest.mark.parametrize("seed", range(40))
def test_the_workspace_holds_every_part(seed):
    """Requests of one token count: all are one kernel's, whose slots the workspace counts; and the grid's bound."""
    rng = random.Random(seed)
    lib = _lib.load()
    D, G, Hkv = rng.choice([64, 128, 256, 512]), rng.choice([1, 2, 3, 8, 16]), rng.choice([1, 2, 4, 8])
    R, n = rng.choice([1, 3, 64, 300]), rng.choice([1, 1, 2, 7, 40, 300])
    width = rng.choice([4, 40, 300])
    window = rng.choice([0, 0, 100, 1024])
    lens = [min(width * 64, n + int(width * 64 * rng.random() ** rng.choice([1, 4]))) for _ in range(R)]
    lens = [max(x, n) if width * 64 >= n else width * 64 for x in lens]
    a = _attn(cache=_cache(heads_kv=Hkv, head_dim=D), cu=0, heads_q=G * Hkv, requests=R, seq_len=R * n, table_width=width,
              table_stride=width, window=window)
    need = lib.gfa_kv4_attn_workspace_bytes(ctypes.byref(a))
    limit = 128 if R * Hkv <= 4 else 64
    large = n * G > limit
    rows = (128 if D >= 128 else 256) if large else 16
    target = 256 * {512: 1, 256: 2, 128: 3, 64: 2}[D] if large else 512
    alone = R * -(-n * G // rows) * Hkv
    min_tiles = (64 if alone >= 256 else 32 if alone >= 128 else 8) if large else 8
    items, parts = _items(lens, [n] * R, G, Hkv, rows, target, window, min_tiles)
    if need == 0:  # one chunk each
        assert width * 2 <= max(16, min_tiles) or window
        return
    groups, rest = divmod(need, rows * (D + 2) * 4)
    assert rest == 0 and groups % Hkv == 0 and parts <= groups // Hkv <= 2 * target // Hkv + 1
    assert items <= R * -(-n * G // rows) + -(-target // Hkv)


def test_workspace_follows_the_call():
    lib = _lib.load()
    ws = lambda **k: lib.gfa_kv4_attn_workspace_bytes(ctypes.byref(_attn(**k)))  # noqa: E731
    assert ws(table_width=8, table_stride=8) == 0  # 512 tokens: one chunk
    assert ws(window=300) == 0 < ws(window=3000)   # a window of few tiles too
    assert ws(requests=0) == 0                     # nothing for arguments the call refuses


def test_exports():
    assert "kv4" in gfa.__all__ and gfa.kv4 is kv4


# ---- the kernels' divisions ----

@pytest.mark.skipif(shutil.which("hipcc") is None, reason="hipcc not available")
def test_divisions_are_exact(tmp_path):
    """Quotients of the work split over their whole range, with reciprocals a unit in the last place off to either side: a
    wrong one loses key tiles of a long table, or counts a row block's chunks from below zero."""
    src = tmp_path / "div.hip"
    src.write_text(r'''
#include "gfa_kv4.h"
#include <cstdio>
#include <random>
static long check(int x, int d) {
  long wrong = 0;
  const float r = 1.0f / (float)d;
  for (const float rcp : {std::nextafter(r, 0.f), r, std::nextafter(r, 2.f)}) wrong += gfa::quotient_by(x, d, rcp) != x / d;
  return wrong;
}
int main() {
  std::mt19937 gen(5);
  long wrong = 0;
  for (int d = 1; d < 2100; ++d) {
    for (const long q : {0l, 1l, 2l, 1l << 22, (1l << 22) + 1, 0x7fffffffl / d}) {
      for (long x = q * d - 2; x <= q * d + 2; ++x)
        if (x >= 0 && x <= 0x7fffffffl) wrong += check((int)x, d);
    }
    for (int i = 0; i < 2000; ++i) wrong += check((int)(gen() >> 1), d) + check((int)(gen() >> (1 + gen() % 31)), d);
  }
  for (int i = 0; i < 1000000; ++i) wrong += check((int)(gen() >> 1), (int)(gen() >> (1 + gen() % 31)) | 1);
  for (const int d : {1 << 30, 0x3fffffff, 0x7fffffff, 0x7ffffffe})
    for (const int x : {0, 1, d - 1, d, 0x7fffffff}) wrong += check(x, d);
  std::printf("%ld\n", wrong);
}
''')
    exe = tmp_path / "div"
    subprocess.run(["hipcc", "--offload-host-only", "-O2", "-std=c++17", "-I", CSRC, "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.strip() == "0"
