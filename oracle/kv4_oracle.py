"""The key/value cache in 4 bits, restated in float64 and plain Python: the format's rounding, a step's plan and
attention over cached values. No code of the package; torch tensors on the CPU in and out."""
from __future__ import annotations

import math

import torch

EXPONENTS = {torch.bfloat16: (-125, 125), torch.float16: (-23, 13)}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def nearest(a: torch.Tensor) -> torch.Tensor:
    """The grid value nearest to each a >= 0, ties to the value with the even index, the largest beyond it."""
    grid = torch.tensor(GRID, dtype=torch.float64)
    d = (a[..., None] - grid).abs()
    best = d.min(-1, keepdim=True).values
    tied = d == best
    even = torch.arange(8) % 2 == 0
    pick = torch.where((tied & even).any(-1, keepdim=True), tied & even, tied)
    return grid[pick.to(torch.uint8).argmax(-1)]


def rounded(x: torch.Tensor) -> torch.Tensor:
    """The float64 values a cache keeps of 16-bit rows x (..., D): blocks of 32, NaN for a block that is not finite."""
    lo, hi = EXPONENTS[x.dtype]
    y = x.double().unflatten(-1, (-1, 32))
    amax = y.abs().amax(-1, keepdim=True)
    safe = torch.where(torch.isfinite(amax) & (amax > 0), amax, torch.ones_like(amax))
    e = torch.floor(torch.log2(safe)) - 2
    e = torch.where(safe > 7 * torch.exp2(e), e + 1, e)
    e = torch.where(amax > 0, e, torch.full_like(e, lo)).clamp(lo, hi)
    s = torch.exp2(e)
    a = torch.where(torch.isfinite(y), y, torch.zeros_like(y)).abs() / s
    v = torch.sign(torch.where(torch.isfinite(y), y, torch.zeros_like(y))) * nearest(a) * s
    v = torch.where(torch.isfinite(y).all(-1, keepdim=True), v, torch.full_like(v, math.nan))
    return v.flatten(-2)


def plan(lens, new, table, free, used, bs, tokens):
    """(slots, positions, cu, lens, used) as lists, ``table`` (a list of lists) changed in place."""
    width = len(table[0])
    slots, positions, cu, taken = [], [], [0], used
    for b, (n, k) in enumerate(zip(lens, new)):
        n, k = max(n, 0), max(k, 0)
        for col in range(-(-n // bs), -(-(n + k) // bs)):
            if col < width:
                table[b][col] = free[taken] if taken < len(free) else -1
            taken += 1
        for pos in range(n, n + k):
            block = table[b][pos // bs] if pos // bs < width else -1
            slots.append(block * bs + pos % bs if block >= 0 else -1)
            positions.append(pos)
        cu.append(cu[-1] + k)
    pad = tokens - len(slots)
    slots = slots[:tokens] + [-1] * pad
    positions = positions[:tokens] + [0] * pad
    return slots, positions, [min(c, tokens) for c in cu], [max(n, 0) + max(k, 0) for n, k in zip(lens, new)], taken


def attend(q, k, v, n_total, causal=True, window=0, scale=None, softcap=0.0, held=None):
    """One request: q (Hq, n, D) its last n tokens, k, v (Hkv, L, D) float64 cached values of its n_total tokens (L >= n_total
    or as many as have a place), ``held`` a mask of positions that have one. Returns (o, weight): float64 (Hq, n, D) and
    sum_j p_j |v_j| in the same shape, which bounds what a rounding of p can do."""
    Hq, n, D = q.shape
    L = min(n_total, k.shape[1])
    G = Hq // k.shape[0]
    scale = D ** -0.5 if scale is None else scale
    pos = torch.arange(n_total - n, n_total)[:, None]
    j = torch.arange(L)[None]
    seen = (j <= pos) if causal else (j < n_total).expand(n, L)
    if causal and window:
        seen = seen & (j > pos - window)
    if held is not None:
        seen = seen & held[None, :L]
    o = torch.zeros((Hq, n, D), dtype=torch.float64)
    weight = torch.zeros((Hq, n, D), dtype=torch.float64)
    for h in range(Hq):
        kh, vh = k[h // G, :L], v[h // G, :L]
        s = (q[h].double() @ kh.t()) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        for i in range(n):
            w = seen[i].nonzero().flatten()
            if len(w):
                p = torch.softmax(s[i, w], 0)
                o[h, i] = p @ vh[w]
                weight[h, i] = p @ vh[w].abs()
    return o, weight
