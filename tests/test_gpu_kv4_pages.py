"""Forked, compacted and copied pages of the 4-bit cache against the definitions in plain Python: tables, free list and every
byte of the caches."""
from __future__ import annotations

import random

import pytest
import torch

from kv4_sharing_cases import LAYERS, Pool, ints
from oracle import kv4_sharing_oracle as orc

pytestmark = pytest.mark.gpu


def run_fork(p, parents=None, keep=None):
    from gemma_triton_flash_attn_amd import kv4

    dev = p.device
    table, lens, free, used = p.lists()
    f = kv4.fork(p.caches, p.table, p.lens_dev, p.free, p.used, parents=None if parents is None else ints(parents, dev),
                 keep=None if keep is None else ints(keep, dev))
    want = orc.fork(table, lens, parents, keep, free, used, p.bs, p.blocks)
    assert f.table.tolist() == want[0] and f.lens.tolist() == want[1] and f.used.tolist() == [want[2]]
    assert p.free.tolist() == free
    assert p.table.tolist() == table and p.used.tolist() == [used]  # only read
    p.check_bytes(want[3])
    return f, want


@pytest.mark.parametrize("bs", [32, 64, 1024])
def test_answers_to_one_prompt(bs, device):
    """One request forked into many: whole blocks shared, the last one copied for all but the first; with whole blocks alone
    nothing is copied."""
    for n in (bs * 3 + 5, bs * 3, 1, bs - 1):
        _, want = run_fork(Pool(device, [n], bs, spare=9, layers=LAYERS[1:2]), [0] * 8)
        assert len(want[3]) == (7 if n % bs else 0)


def test_requests_that_leave(device):
    """Dropped requests' blocks are given back, those that others hold stay."""
    p = Pool(device, [300, 130, 64, 0, 257], common=1)
    f, want = run_fork(p, [4, -1, 1, 9, 3])
    assert want[2] < int(p.used)
    run_fork(Pool(device, [300, 130], common=2), [-1, 2])  # all of them


def test_tokens_taken_back(device):
    """keep shortens rows: inside the last block, to a whole block, by whole blocks, into blocks that others hold whole."""
    p = Pool(device, [300, 300, 310, 64, 65], common=4)
    _, want = run_fork(p, None, [295, 256, 100, 64, 0])
    assert want[3]  # row 2 kept a part of a block that the others hold whole
    run_fork(Pool(device, [70, 5]), None, [1000, -4])


@pytest.mark.parametrize("seed", range(12))
def test_any_tables(seed, device):
    """Random tables with common and missing blocks, wide rows apart from each other, lengths past the table, any parents."""
    r = random.Random(seed)
    bs, B = r.choice([32, 64, 128]), r.choice([1, 2, 7, 40])
    lens = [r.choice([0, 1, bs, r.randint(0, 12 * bs), r.randint(0, 3 * bs)]) for _ in range(B)]
    p = Pool(device, lens, bs, spare=r.choice([0, 3, 60]), layers=r.sample(LAYERS, r.choice([1, 3])), common=r.choice([0, 0, 2, 5]),
             seed=seed, missing=r.choice([0.0, 0.1]), width=r.choice([None, 4, 13]), gap=r.choice([0, 5]))
    rows = r.choice([1, B, 3 * B])
    parents = r.choice([None, [r.randint(-1, B) for _ in range(rows)], [r.randrange(B) for _ in range(rows)]])
    keep = r.choice([None, [r.randint(-2, 14 * bs) for _ in range(len(parents or lens))]])
    run_fork(p, parents, keep)


def test_a_full_pool(device):
    """Copies beyond the free list are left out, and used tells of it; blocks given back by the same call are taken first."""
    f, want = run_fork(Pool(device, [70], spare=2), [0] * 6)
    assert f.used.tolist() == [7] and (f.table[:, 1] == -1).sum() == 3
    p = Pool(device, [70, 640], spare=0)
    f, want = run_fork(p, [0] * 6)  # the second request's ten blocks come back
    assert (f.table[:, 1] >= 0).all() and want[2] == 7


def test_counts_out_of_range(device):
    """used beyond the list is the list's end, below zero its start; a list too short for what comes back keeps the lowest ids."""
    for used in (100, -3, 0, 2):
        p = Pool(device, [200, 200, 90], spare=4)
        p.used.fill_(used)
        run_fork(p, [0, 0, -1])
    p = Pool(device, [64, 64])
    p.free, p.used = ints([], device), ints([0], device)
    run_fork(p, [0, -1, 1], [10, 64, 64])


def test_many_requests(device):
    """More rows than a workgroup has threads, tables that several workgroups write."""
    r = random.Random(5)
    lens = [r.randint(0, 200) for _ in range(1500)]
    p = Pool(device, lens, 32, spare=800, layers=[(1, 64)], common=1, extra=40)
    run_fork(p, [r.randrange(1500) for _ in range(2100)], [r.randint(0, 220) for _ in range(2100)])
    run_fork(Pool(device, lens[:1100], 32, spare=2, layers=[(1, 64)]), [b for b in range(1100) if b % 3])


def test_the_largest_pool(device):
    """2^18 blocks, whose sets fill the LDS."""
    p = Pool(device, [32 * 5 + 3, 32 * 90], 32, spare=(1 << 18) - 96, layers=[(1, 64)])
    assert p.blocks == 1 << 18 and p.table.max() > 1 << 16
    run_fork(p, [0, 0, 0], None)
    run_compact(Pool(device, [32 * 5 + 3, 32 * 90], 32, spare=(1 << 18) - 96, layers=[(1, 64)]))


def run_compact(p):
    from gemma_triton_flash_attn_amd import kv4

    table, lens, _, _ = p.lists()
    f = kv4.compact(p.caches, p.table, p.lens_dev, p.free)
    want = orc.compact(table, lens, p.bs, p.blocks)
    assert f.table.tolist() == want[0] and f.used.tolist() == [want[1]]
    assert p.free.tolist() == list(range(p.blocks)) and p.table.tolist() == table
    p.check_bytes(want[2])
    return f, want


@pytest.mark.parametrize("seed", range(8))
def test_compacted(seed, device):
    r = random.Random(seed)
    bs, B = r.choice([32, 64, 256]), r.choice([1, 5, 60])
    lens = [r.choice([0, 1, r.randint(0, 9 * bs)]) for _ in range(B)]
    run_compact(Pool(device, lens, bs, spare=r.choice([0, 1, 30, 300]), layers=r.sample(LAYERS, r.choice([1, 2])),
                     common=r.choice([0, 3]), seed=seed, missing=r.choice([0.0, 0.2]), width=r.choice([None, 5]), gap=r.choice([0, 3])))


def test_compacted_ends(device):
    """Nothing held, everything held, one block at the pool's end; many rows."""
    run_compact(Pool(device, [0, 0], spare=5))
    run_compact(Pool(device, [64 * 9], spare=0))
    p = Pool(device, [1], spare=700)
    p.table[0, 0] = p.blocks - 1
    _, want = run_compact(p)
    assert want[2] == [(700, 0)]
    r = random.Random(1)
    run_compact(Pool(device, [r.randint(0, 300) for _ in range(1300)], 32, spare=3000, layers=[(1, 64)]))


def test_copied(device):
    """Blocks of caches of any shape, pairs that are none, none at all."""
    from gemma_triton_flash_attn_amd import kv4

    p = Pool(device, [640], spare=30, layers=LAYERS)
    pairs = [(3, 9), (3, 11), (0, 39), (38, 1)]
    kv4.copy(p.caches, ints([3, -1, 3, 4, 0, 40, 38], device), ints([9, 2, 11, -7, 39, 5, 1], device))
    p.check_bytes(pairs)
    p = Pool(device, [640], spare=30, layers=LAYERS[:1])
    kv4.copy(p.caches[0], ints([], device), ints([], device))
    p.check_bytes([])


def test_more_layers_than_a_launch_takes(device):
    """Forty caches of two shapes: two launches of copies."""
    run_fork(Pool(device, [100, 40], layers=[(1, 64), (2, 128)] * 20), [0, 0, 1, 1])


def test_large_blocks(device):
    """Blocks of 4.25 MB, and a cache past 4 GiB: bytes on both sides of 2^32."""
    from gemma_triton_flash_attn_amd import kv4

    c = kv4.allocate(1030, 8, 512, 1024, torch.bfloat16, device)
    assert c.codes.numel() > 1 << 32
    g = torch.Generator(device=device).manual_seed(0)
    for b in (2, 1028):
        c.codes[b].random_(0, 256, generator=g)
        c.scales[b].random_(0, 256, generator=g)
    kv4.copy(c, ints([2, 1028], device), ints([1029, 5], device))
    for s, d in ((2, 1029), (1028, 5)):
        assert torch.equal(c.codes[s], c.codes[d]) and torch.equal(c.scales[s], c.scales[d])


def test_captured(device):
    """A graph of a fork and a compaction, replayed over tables that change in place, with eager calls between."""
    from gemma_triton_flash_attn_amd import kv4

    p = Pool(device, [200, 130, 64, 90], spare=20, common=1)
    parents, keep = ints([0, 0, 2, 1], device), ints([190, 200, 64, 100], device)
    start = (p.table.clone(), p.lens_dev.clone(), p.free.clone(), p.used.clone())

    def step():
        f = kv4.fork(p.caches, p.table, p.lens_dev, p.free, p.used, parents=parents, keep=keep)
        return f, kv4.compact(p.caches, f.table, f.lens, p.free)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f, c = step()
    r = random.Random(3)
    for _ in range(4):
        parents.copy_(ints([r.randint(-1, 3) for _ in range(4)], device))
        keep.copy_(ints([r.randint(0, 220) for _ in range(4)], device))
        for x, y in zip((p.table, p.lens_dev, p.free, p.used), start):
            x.copy_(y)
        for k, (codes, scales) in zip(p.caches, p.before):
            k.codes.copy_(codes)
            k.scales.copy_(scales)
        graph.replay()
        got = [f.table.clone(), f.lens.clone(), f.used.clone(), c.table.clone(), c.used.clone(), p.free.clone()]
        got += [x.clone() for k in p.caches for x in (k.codes, k.scales)]
        torch.cuda.synchronize()
        for x, y in zip((p.table, p.lens_dev, p.free, p.used), start):
            x.copy_(y)
        for k, (codes, scales) in zip(p.caches, p.before):
            k.codes.copy_(codes)
            k.scales.copy_(scales)
        f2, c2 = step()
        want = [f2.table, f2.lens, f2.used, c2.table, c2.used, p.free] + [x for k in p.caches for x in (k.codes, k.scales)]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_another_stream_and_compiled(device):
    from gemma_triton_flash_attn_amd import kv4

    p = Pool(device, [200, 130, 64], spare=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_fork(p, [0, 0, 2, 1])
    p = Pool(device, [200, 130, 64], spare=20)
    codes, scales = [c.codes for c in p.caches], [c.scales for c in p.caches]
    torch.library.opcheck(torch.ops.gfa.kv4_fork, (codes, scales, p.table.contiguous(), p.lens_dev, p.free, p.used, ints([0, 0], device), None))
    torch.library.opcheck(torch.ops.gfa.kv4_compact, (codes, scales, p.table.contiguous(), p.lens_dev, p.free))
    torch.library.opcheck(torch.ops.gfa.kv4_copy, (codes, scales, ints([1], device), ints([2], device)))

    p, q = (Pool(device, [200, 130, 64], spare=20, seed=4) for _ in range(2))
    for c, d in zip(p.caches, q.caches):
        d.codes.copy_(c.codes)
        d.scales.copy_(c.scales)
    parents = ints([0, 2, 2, 0], device)

    def both(codes, scales, table, lens, free, used):
        caches = [kv4.Cache(c, s, torch.bfloat16) for c, s in zip(codes, scales)]
        f = kv4.fork(caches, table, lens, free, used, parents=parents)
        return f, kv4.compact(caches, f.table, f.lens, free)

    args = lambda x: ([c.codes for c in x.caches], [c.scales for c in x.caches], x.table, x.lens_dev, x.free, x.used)  # noqa: E731
    want = both(*args(p))
    got = torch.compile(both, fullgraph=True, backend="aot_eager")(*args(q))
    for a, b in zip(want[0] + want[1], got[0] + got[1]):
        assert torch.equal(a, b)
    assert torch.equal(p.free, q.free)
    for c, d in zip(p.caches, q.caches):
        assert torch.equal(c.codes, d.codes) and torch.equal(c.scales, d.scales)
