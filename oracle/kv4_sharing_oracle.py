"""What requests have in common, restated in plain Python: forked and compacted block tables, common prefixes, verified drafts.
No code of the package; lists in and out. A block is a number in [0, blocks); other entries of a table are no block."""
from __future__ import annotations

from fractions import Fraction

import math


def _held(row, tokens, bs, blocks):
    return [x if 0 <= x < blocks else -1 for x in row[: -(-max(tokens, 0) // bs)]]


def fork(table, lens, parents, keep, free, used, bs, blocks):
    """(table, lens, used, pairs of blocks copied); ``free`` is changed in place. parents, keep: lists or None."""
    width = len(table[0])
    parents = list(range(len(table))) if parents is None else parents
    used = min(max(used, 0), len(free))
    old = {x for row, n in zip(table, lens) for x in _held(row, n, bs, blocks)} - {-1}
    rows, tokens = [], []
    for r, p in enumerate(parents):
        there = 0 <= p < len(table)
        n = max(lens[p], 0) if there else 0
        n = min(n, max(keep[r], 0)) if keep is not None else n
        rows.append(_held(table[p], n, bs, blocks) if there else [])
        tokens.append(n)
    whole = {x for row, n in zip(rows, tokens) for x in row[: n // bs]} - {-1}
    back = sorted(old - {x for row in rows for x in row})[:used]
    free[used - len(back):used] = back
    used -= len(back)
    # the list with what was given back at its new top
    owner, pairs = {}, []
    for r, (row, n) in enumerate(zip(rows, tokens)):
        if n % bs and n // bs < width and row[n // bs] >= 0:
            x = row[n // bs]
            if x in whole or owner.setdefault(x, r) != r:
                to = free[used] if used < len(free) else -1
                to = to if 0 <= to < blocks else -1
                row[n // bs] = to
                if to >= 0:
                    pairs.append((x, to))
                used += 1
    return [row + [-1] * (width - len(row)) for row in rows], tokens, used, pairs


def compact(table, lens, bs, blocks):
    """(table, used, pairs of blocks moved)."""
    width = len(table[0])
    rows = [_held(row, n, bs, blocks) for row, n in zip(table, lens)]
    live = {x for row in rows for x in row} - {-1}
    n = len(live)
    holes = (x for x in range(n) if x not in live)
    to = {x: next(holes) for x in sorted(live) if x >= n}
    return [[to.get(x, x) for x in row] + [-1] * (width - len(row)) for row in rows], n, list(to.items())


def share(table, lens, cu, bs, least):
    """(skip, cu, lens) of the groups."""
    R, width = len(table), len(table[0])
    limit = [min(max(n - max(cu[b + 1] - cu[b], 0), 0) // bs, width) for b, n in enumerate(lens)]
    common, groups = [0], [[0]]
    for b in range(1, R):
        n = 0
        while n < min(limit[b - 1], limit[b]) and table[b][n] == table[b - 1][n]:
            n += 1
        common.append(n * bs)
        if n * bs >= least:
            groups[-1].append(b)
        else:
            groups.append([b])
    skip, first, seen = [0] * R, [0] * R + [cu[R]], [0] * R
    for g in groups:
        n = min((common[b] for b in g[1:]), default=0)
        for b in g:
            skip[b] = n
            first[b] = cu[b] if b == g[0] else cu[g[-1] + 1]
        seen[g[0]] = n
    return skip, first, seen


def _probability(x):
    return Fraction(x) if math.isfinite(x) and x > 0 else Fraction(0)


def draw(weights, r):
    """The first entry at which the running sum of weights (Fractions) exceeds r times their sum; the last with weight for r = 1."""
    total = sum(weights)
    if total == 0:
        return -1
    goal, run, last = Fraction(r) * total, Fraction(0), -1
    for i, w in enumerate(weights):
        run += w
        if w > 0:
            last = i
            if run > goal:
                return i
    return last


def verify(target, draft, tokens, accept, sample, lens, cu):
    """(follows, accepted, lens), from lists of Python floats, in exact arithmetic."""
    T, V = len(target), len(target[0])
    follows, accepted, left = [-1] * T, [], []
    for b, n in enumerate(lens):
        t0 = min(max(cu[b], 0), T)
        count = min(max(cu[b + 1], t0), T) - t0
        if count == 0:
            accepted.append(0)
            left.append(n)
            continue
        a = 0
        while a < count - 1:
            t = t0 + a
            x = tokens[t + 1]
            if not 0 <= x < V:
                break
            q = Fraction(1) if draft is None else _probability(draft[t + 1][x])
            u = accept[t + 1]
            if not (math.isfinite(u) and Fraction(u) * q < _probability(target[t][x])):
                break
            follows[t] = x
            a += 1
        t = t0 + a
        w = whole = [_probability(x) for x in target[t]]
        if a < count - 1:
            if draft is None:
                q = [Fraction(int(i == tokens[t + 1])) for i in range(V)]
            else:
                q = [_probability(x) for x in draft[t + 1]]
            w = [max(x - y, Fraction(0)) for x, y in zip(whole, q)]
            w = w if any(w) else whole
        r = sample[b]
        follows[t] = draw(w, min(max(r, 0.0), 1.0) if r == r else 0.0)
        accepted.append(a)
        left.append(n - (count - 1 - a))
    return follows, accepted, left
