"""A step's block tables and slot maps against plain Python: equal."""
from __future__ import annotations

import random

import pytest
import torch

from oracle import kv4_oracle as orc

pytestmark = pytest.mark.gpu


def _run(lens, new, table, free, used, bs, tokens, device, wide=0):
    from gemma_triton_flash_attn_amd import kv4

    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    tab = torch.full((len(lens), len(table[0]) + wide), -7, dtype=torch.int32, device=device)
    view = tab[:, :len(table[0])]
    view.copy_(ints(table))
    before = (ints(lens), ints(new), ints(free) if free else ints([]), ints([used]))
    kept = [t.clone() for t in before]
    got = kv4.plan(before[0], before[1], view, before[2], before[3], block_size=bs, tokens=tokens)
    want_table = [list(r) for r in table]
    slots, positions, cu, total, taken = orc.plan(lens, new, want_table, free, used, bs, tokens)
    assert got.slots.tolist() == slots and got.slots.dtype == torch.int64
    assert got.positions.tolist() == positions
    assert got.cu.tolist() == cu
    assert got.lens.tolist() == total
    assert got.used.tolist() == [taken]
    assert view.tolist() == want_table
    assert not wide or (tab[:, -wide:] == -7).all()
    assert all(torch.equal(a, b) for a, b in zip(before, kept))


def _batch(rng, B, bs, longest, most):
    lens = [rng.choice([0, rng.randint(0, longest), bs * rng.randint(0, longest // bs)]) for _ in range(B)]
    new = [rng.choice([0, 1, 1, rng.randint(0, most)]) for _ in range(B)]
    width = max(-(-(n + k) // bs) for n, k in zip(lens, new)) + 1
    ids = list(range(3 * B + sum(-(-(n + k) // bs) for n, k in zip(lens, new))))
    rng.shuffle(ids)
    table = [[ids.pop() if c < -(-n // bs) else -1 for c in range(width)] for n in lens]
    return lens, new, table, ids


@pytest.mark.parametrize("bs", [32, 64, 256])
@pytest.mark.parametrize("B,longest,most", [(1, 200, 1), (3, 500, 700), (64, 300, 40), (255, 90, 9), (256, 90, 9), (257, 90, 5),
                                            (1000, 300, 3)])
def test_plans(B, longest, most, bs, device):
    rng = random.Random(B + bs)
    lens, new, table, free = _batch(rng, B, bs, longest, most)
    for pad in (0, 29):
        _run(lens, new, table, free, 2, bs, sum(new) + pad, device, wide=3)


def test_nothing_new(device):
    _run([5, 0, 64], [0, 0, 0], [[1, -1], [-1, -1], [2, -1]], [3, 4], 0, 64, 0, device)
    _run([5, 0, 64], [0, 0, 0], [[1, -1], [-1, -1], [2, -1]], [3, 4], 0, 64, 300, device)
    _run([0], [0], [[-1]], [], 0, 32, 1, device)


def test_shortages(device):
    """The free list ends, a request outgrows the table, fewer tokens than are new, negative counts."""
    _run([10, 60, 0], [30, 100, 40], [[4, -1, -1, -1, -1], [5, 6, -1, -1, -1], [-1] * 5], [7, 8, 9], 1, 32, 170, device)
    _run([10, 0], [300, 40], [[4, -1], [-1, -1]], list(range(10, 40)), 0, 32, 340, device)
    _run([10, 0], [300, 40], [[4, -1], [-1, -1]], list(range(10, 40)), 0, 32, 64, device)
    _run([-3, 7], [5, -2], [[-1, -1], [3, -1]], [1, 2], 0, 32, 8, device)
    _run([32], [1], [[9, -1]], [], 0, 32, 1, device)


def test_steps_follow_each_other(device):
    """The outputs of a step are the inputs of the next; a prompt comes in parts, then single tokens."""
    from gemma_triton_flash_attn_amd import kv4

    bs, B = 32, 4
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    table, lens, used, free = torch.full((B, 8), -1, dtype=torch.int32, device=device), ints([0] * B), ints([0]), ints(list(range(40))[::-1])
    want = [[-1] * 8 for _ in range(B)]
    total, taken = [0] * B, 0
    for new in ([40, 0, 31, 1], [1, 64, 1, 1], [33, 1, 1, 0], [1, 1, 1, 1]):
        p = kv4.plan(lens, ints(new), table, free, used, block_size=bs, tokens=150)
        slots, positions, cu, total, taken = orc.plan(total, new, want, free.tolist(), taken, bs, 150)
        assert (p.slots.tolist(), p.positions.tolist(), p.cu.tolist(), p.lens.tolist(), p.used.tolist()) == (
            slots, positions, cu, total, [taken])
        assert table.tolist() == want
        lens, used = p.lens, p.used
