"""What the host sizes for attention over shared prefixes holds what the device makes of any lengths: both restated here, the host's
sizes checked against the workspace it asks for, the device's items against each part's own slots."""
from __future__ import annotations

import ctypes
import math
import random
from dataclasses import dataclass

import numpy as np
import pytest

from gemma_triton_flash_attn_amd import _lib
from test_kv4_sharing_cpu import _attn, _cache

NONE = 0x3FFFFFFF
KINDS = ("many", "few", "rest")


@dataclass
class Call:
    D: int
    G: int
    Hkv: int
    requests: int
    tokens: int
    width: int  # blocks of a table row
    bs: int = 64
    max_new: int = 1

    @property
    def args(self):
        return _attn(cache=_cache(heads_kv=self.Hkv, head_dim=self.D, block_size=self.bs), heads_q=self.G * self.Hkv, requests=self.requests,
                     seq_len=self.tokens, table_width=self.width, table_stride=self.width, max_new=self.max_new, shared_skip=64, shared_cu=64,
                     shared_lens=64, shared_apart=1)

    @property
    def tiles(self):
        return self.width * self.bs // 32


@dataclass
class Part:
    row_blocks: int
    slots: int
    min_tiles: int
    share: np.float32
    rows: int

    def bytes(self, c):
        return self.slots * c.Hkv * self.rows * (c.D + 2) * 4


def part(c, row_blocks, rows, min_tiles, target, whole=False):
    chunks = 1 if c.tiles <= 16 else -(-c.tiles // min_tiles)
    slots = min(row_blocks * chunks, 2 * target // c.Hkv + 1 if whole else row_blocks + -(-target // c.Hkv))
    return Part(row_blocks, 0 if whole and chunks == 1 else slots, min_tiles if chunks > 1 else NONE,
                np.float32(c.Hkv / target * (1 + 1 / 4096)), rows)


def row_limit(c):
    return 128 if c.requests * c.Hkv <= 4 else 64


def group_limit(c):
    return 32 if c.Hkv >= 4 and c.D >= 128 else 64


def sizes(c):
    """The host's parts by kind, the groups' line between few rows and many, and the chunk kernel's part of the requests."""
    rows, groups = c.tokens * c.G, max(1, c.requests // 2)
    limit = group_limit(c)
    few, many = (rows + 15 * groups) // 16, 0
    if rows > limit:
        few, many = min(few, groups * -(-limit // 16)), rows // 128 + min(groups, rows // (limit + 1))
    short = 4 if c.requests * c.Hkv <= 16 else 8
    parts = {"many": part(c, many, 128, 4 if many * c.Hkv <= 16 else 8, 256 if c.D < 512 else 160),
             "few": part(c, few, 16, short, 512 if c.D < 512 else 256),
             "rest": part(c, (rows + 15 * c.requests) // 16, 16, short, 512 if c.D < 512 else 128)}
    large, most, big = 0, min(c.max_new, c.tokens) if c.max_new else c.tokens, 128 if c.D >= 128 else 256
    if most * c.G > row_limit(c):
        large = rows // big + min(c.requests, rows // (row_limit(c) + 1))
    alone = large * c.Hkv
    chunk = part(c, large, big, 64 if alone >= 256 else 32 if alone >= 128 else 8, 256 * {512: 1, 128: 3}.get(c.D, 2), whole=True)
    return parts, limit if rows > limit else NONE, chunk


def asked(c):
    return _lib.load().gfa_kv4_attn_workspace_bytes(ctypes.byref(c.args))


def workspace(c):
    parts, _, chunk = sizes(c)
    return sum(p.bytes(c) for p in parts.values()) + 64 + 48 * parts["rest"].row_blocks + chunk.bytes(c)


def items(c, new, lens, groups, apart=True):
    """Items of each kind that the device makes, and row blocks: ``groups`` are (first request, requests, prefix in tokens).

    The device sums tiles in 32 bits, lane by lane and then over lanes; `share` is rounded up by 2^-12 of itself, far more than 75 additions'
    rounding, 2^-24 of the sum each, so the sum rounded once stands for any order."""
    parts, line, _ = sizes(c)
    blocks = lambda rows, n: -(-rows // n)  # noqa: E731
    skip, own, pre = [0] * c.requests, [], []
    for first, n, prefix in groups:
        skip[first:first + n] = [prefix] * n
        rows = sum(new[first:first + n]) * c.G
        kind = "many" if rows > line else "few"
        pre.append((kind, blocks(rows, 128 if kind == "many" else 16), blocks(min(prefix, c.width * c.bs), 32)))
    for n, length, s in zip(new, lens, skip):
        held = min(length, c.width * c.bs)
        whole = blocks(held, 32)
        rows = n * c.G
        large = not c.max_new and c.tokens * c.G > row_limit(c) and rows > row_limit(c)  # the chunk kernel's
        own.append((0 if large else blocks(rows, 16), (whole - s // 32 if held > s else 0) if apart else whole))
    total = {k: sum(b * t for kind, b, t in pre if kind == k) for k in ("many", "few")}
    total["rest"] = sum(b * t for b, t in own)
    per = {k: max(int(min(math.ceil(np.float32(total[k]) * parts[k].share), 1e9)), parts[k].min_tiles) for k in KINDS}
    count = lambda b, t, k: b * max(-(-t // per[k]), 1)  # noqa: E731
    out = {k: sum(count(b, t, k) for kind, b, t in pre if kind == k) if apart else 0 for k in ("many", "few")}
    out["rest"] = sum(count(b, t, "rest") for b, t in own)
    return out, sum(b for b, _ in own), sum(b for _, b, _ in pre)


def any_call(r):
    D, G, Hkv = r.choice([64, 128, 256, 512]), r.choice([1, 2, 3, 4, 8]), r.choice([1, 2, 4, 8, 16])
    R = r.choice([2, 3, 5, 16, 64, 65, 300])
    most = max(1, min(8, 64 // G))
    new = [r.choice([0, 1, 1, 1, r.randint(1, most)]) for _ in range(R)]
    if not any(new):
        new[-1] = 1
    max_new = r.choice([max(new), 0])
    if max_new == 0 and R > 16:
        new[r.randrange(R)] = max(1, (16 * R - sum(new) * G) // (2 * G))  # a prompt's chunk
    c = Call(D, G, Hkv, R, sum(new) + r.choice([0, 0, 3]), r.choice([1, 8, 9, 40, 257, 5000]), r.choice([32, 64, 256]), max_new)
    longest = r.choice([c.width * c.bs, c.width * c.bs, max(1, c.width * c.bs // 7), c.width * c.bs + 100])
    groups, b = [], 0
    while R - b >= 2:
        n = min(R - b, r.choice([1, 2, 2, 3, 10, 70]))
        if n > 1:
            groups.append((b, n, r.choice([1, r.randint(1, c.width)]) * c.bs))
        b += n
    lens = [r.choice([longest, r.randint(0, longest)]) for _ in range(R)]
    for first, n, prefix in groups:
        for i in range(first, first + n):
            lens[i] = max(lens[i], prefix)
    return c, new, lens, groups


def shared(c):
    """Whether the call takes prefixes at all."""
    rows = c.max_new or -(-c.tokens // c.requests)
    return rows * c.G <= row_limit(c)


@pytest.mark.parametrize("seed", range(60))
def test_every_item_has_a_slot(seed):
    r = random.Random(seed)
    seen = 0
    for _ in range(40):
        c, new, lens, groups = any_call(r)
        if not shared(c):
            continue
        seen += 1
        assert asked(c) == workspace(c), c
        parts, _, _ = sizes(c)
        for apart in (True, False):
            got, own, pre = items(c, new, lens, groups, apart)
            assert own <= parts["rest"].row_blocks and pre <= parts["many"].row_blocks + parts["few"].row_blocks
            for k in KINDS:
                assert got[k] <= parts[k].slots, (k, c, got[k], parts[k])
    assert seen > 10


FULL = {
    # as many items as slots, of the part alone: one slot less would not hold them
    "rest": (Call(128, 1, 2, 10, 10, 40), [1] * 10, [2560] * 10, []),
    "few": (Call(128, 1, 2, 20, 10, 20), [0, 1] * 10, [1280] * 20, [(2 * i, 2, 1280) for i in range(10)]),
    "many": (Call(64, 1, 1, 65, 65, 32), [1] * 65, [2048] * 65, [(0, 65, 2048)]),
    "many_shared_keys": (Call(512, 1, 4, 66, 65, 12), [1] * 65 + [0], [768] * 66, [(0, 66, 768)]),
}


@pytest.mark.parametrize("name", list(FULL))
def test_no_slot_to_spare(name):
    """The check above is sharp for each part: calls that fill one to the last slot."""
    c, new, lens, groups = FULL[name]
    kind = name.split("_")[0]
    assert asked(c) == workspace(c)
    parts, _, _ = sizes(c)
    got, _, _ = items(c, new, lens, groups, apart=kind != "rest")
    assert got[kind] == parts[kind].slots > 0
