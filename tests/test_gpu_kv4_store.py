"""Rows in the 4-bit cache and back, against the format's rounding in 64 bits: equal values."""
from __future__ import annotations

import pytest
import torch

from oracle import kv4_oracle as orc

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def _roundtrip(k, v, device, bs=64, spare=2, seed=0):
    """(cache, slots, k back, v back) of rows (1, H, T, D) stored at random slots."""
    from gemma_triton_flash_attn_amd import kv4

    H, T, D = k.shape[1:]
    blocks = -(-T // bs) + spare
    cache = kv4.allocate(blocks, H, D, bs, k.dtype, device)
    cache.codes.fill_(255)
    cache.scales.fill_(255)
    slots = torch.randperm(blocks * bs, generator=torch.Generator().manual_seed(seed))[:T].to(device)
    kv4.write(cache, k.to(device), v.to(device), slots)
    return cache, slots, *kv4.read(cache, slots)


def _same(got, want):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("H,T,bs", [(1, 1, 32), (3, 37, 64), (2, 300, 128)])
def test_rows_come_back_rounded(D, H, T, bs, dtype, device):
    g = torch.Generator().manual_seed(T)
    k, v = ((torch.randn(1, H, T, D, generator=g) * torch.exp(2 * torch.randn(1, H, T, 1, generator=g))).to(dtype) for _ in range(2))
    v[0, 0, 0, :40] = 0  # a block of zeros
    _, _, ko, vo = _roundtrip(k, v, device, bs)
    assert ko.dtype == vo.dtype == dtype and ko.shape == k.shape
    _same(ko, orc.rounded(k))
    _same(vo, orc.rounded(v))


@pytest.mark.parametrize("dtype", TYPES)
def test_every_value_of_the_type(dtype, device):
    """All 65536 bit patterns, as neighbours of their own size and each beside a larger value of several sizes."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    k = every.reshape(1, 1, -1, 64).clone()
    tops = torch.tensor([4.0, 6.0, 7.0, 7.01, 3.99, 0.0]).to(dtype)
    rows = []
    for scale in (2.0 ** -20, 2.0 ** -8, 1.0, 2.0 ** 7):
        for top in tops:
            big = (top.double() * scale).to(dtype)
            part = every[every.double().abs() <= big.double()]
            part = torch.cat([part, part.new_zeros(-part.numel() % 31)]).reshape(-1, 31)
            rows.append(torch.cat([part, big.expand(part.shape[0], 1)], 1))
    x = torch.cat(rows)
    x = torch.cat([x, x.new_zeros(x.shape[0] % 2, 32)]).reshape(1, 1, -1, 64)
    for y in (k, x):
        other = y.flip(2).clone()
        other[~torch.isfinite(other)] = 0
        clean = torch.where(torch.isfinite(y), y, torch.zeros_like(y))
        _, _, ko, vo = _roundtrip(clean, other, device)
        _same(ko, orc.rounded(clean))
        _same(vo, orc.rounded(other))


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_no_numbers(dtype, device):
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(1, 2, 50, 128, generator=g).to(dtype) for _ in range(2))
    k[0, 0, 3, 70] = float("inf")
    k[0, 1, 4, 0] = float("nan")
    v[0, 1, 7, 127] = float("-inf")
    _, _, ko, vo = _roundtrip(k, v, device)
    wk, wv = orc.rounded(k), orc.rounded(v)
    assert torch.isnan(wk).sum() == 64 and torch.isnan(wv).sum() == 32
    wk[0, 1, 7, :32] = float("nan")  # the token whose value is none: its first key block says so
    _same(ko, wk)
    _same(vo, wv)


@pytest.mark.parametrize("D", [64, 512])
def test_other_slots_are_left_alone(D, device):
    from gemma_triton_flash_attn_amd import kv4

    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(1, 2, 20, D, generator=g).to(device, torch.bfloat16) for _ in range(2))
    cache, slots, k0, v0 = _roundtrip(k, v, device)
    codes, scales = cache.codes.clone(), cache.scales.clone()
    total = cache.num_blocks * cache.block_size
    bad = torch.tensor([-1, total, -(1 << 40), 1 << 40, total + 7], device=device)
    kv4.write(cache, k[:, :, :5] * 3, v[:, :, :5] * 3, bad)  # no slot: nothing happens
    assert torch.equal(cache.codes, codes) and torch.equal(cache.scales, scales)
    kr, vr = kv4.read(cache, bad)
    assert not kr.any() and not vr.any()
    taken = set(slots.tolist())
    other = torch.tensor([s for s in range(total) if s not in taken], device=device)[:9]
    kv4.write(cache, k[:, :, 5:14], v[:, :, 5:14], other)
    k1, v1 = kv4.read(cache, slots)
    assert torch.equal(k0, k1) and torch.equal(v0, v1)


def test_views_and_token_orders(device):
    """Strided projections, one token per batch entry, a copied unaligned view: the same bytes."""
    from gemma_triton_flash_attn_amd import kv4

    g = torch.Generator().manual_seed(3)
    H, T, D = 3, 24, 128
    k, v = (torch.randn(T, H, D, generator=g).to(device, torch.float16) for _ in range(2))
    slots = torch.randperm(64, generator=g)[:T].to(device)
    forms = {
        "packed": [x[None].transpose(1, 2) for x in (k, v)],
        "steps": [x[:, :, None] for x in (k, v)],
        "batch": [x.reshape(4, 6, H, D).transpose(1, 2) for x in (k, v)],
        "unaligned": [torch.cat([x.new_zeros(T, H, 1), x], 2)[:, :, 1:][None].transpose(1, 2) for x in (k, v)],
        "fused": [torch.cat([k, v], 1)[:, i * H:(i + 1) * H][None].transpose(1, 2) for i in (0, 1)],
    }
    seen = []
    for a, b in forms.values():
        cache = kv4.allocate(1, H, D, 64, torch.float16, device)
        cache.codes.zero_()
        cache.scales.zero_()
        kv4.write(cache, a, b, slots)
        seen.append((cache.codes, cache.scales))
    assert all(torch.equal(c, seen[0][0]) and torch.equal(s, seen[0][1]) for c, s in seen)


def test_a_cache_past_4_gib(device):
    """Slots whose bytes lie past 32-bit offsets."""
    from gemma_triton_flash_attn_amd import kv4

    g = torch.Generator().manual_seed(4)
    cache = kv4.allocate(35000, 4, 512, 64, torch.bfloat16, device)  # 4.6 GB of codes
    assert cache.codes.numel() > 1 << 32
    total = cache.num_blocks * cache.block_size
    slots = torch.tensor([0, 77, total // 2, total - 1, total - 64, total - 100])
    k, v = (torch.randn(1, 4, len(slots), 512, generator=g).to(torch.bfloat16) for _ in range(2))
    kv4.write(cache, k.to(device), v.to(device), slots.to(device))
    ko, vo = kv4.read(cache, slots.to(device))
    _same(ko, orc.rounded(k))
    _same(vo, orc.rounded(v))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_runs_of_slots(D, dtype, device):
    """Slots in a row from every alignment, ends inside a group of four, a gap and a repeat-free reversal."""
    from gemma_triton_flash_attn_amd import kv4

    g = torch.Generator().manual_seed(D)
    runs = [list(range(a, a + n)) for a, n in [(0, 1), (4, 9), (17, 4), (23, 6), (31, 3), (64, 33), (101, 2)]]
    runs += [[104, 105, -1, 107, 108, 109, 110, 111], [115, 114, 113, 112], [120, 121, 122, -1]]
    cache = kv4.allocate(2, 3, D, 64, dtype, device)
    cache.codes.fill_(255)
    cache.scales.fill_(255)
    for run in runs:
        k, v = (torch.randn(1, 3, len(run), D, generator=g).to(dtype) for _ in range(2))
        slots = torch.tensor(run, device=device)
        kv4.write(cache, k.to(device), v.to(device), slots)
        dead = torch.tensor(run) < 0
        for got, x in zip(kv4.read(cache, slots), (k, v)):
            want = orc.rounded(x)
            want[:, :, dead] = 0
            _same(got, want)
    untouched = torch.tensor([3, 13, 16, 21, 22, 29, 34, 63, 97, 103, 106, 123], device=device)
    for got in kv4.read(cache, untouched):
        assert torch.isnan(got).all()
