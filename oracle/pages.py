"""The life of a paged cache's pages in plain Python: forks, releases and
compaction, page by page."""

from __future__ import annotations

import numpy as np


def held(length: int, page: int, columns: int) -> int:
    return min(max(0, -(-length // page)), columns)


def fork(lengths, tables, shares, stack, count, parents, tokens, page):
    """(lengths, tables, shares, count, sources, targets, overflow) of the
    children and of the pool."""

    n, columns = len(parents), tables.shape[1]
    shares = list(shares)
    rows = np.full((n, columns), -1)
    sources, targets = [-1] * n, [-1] * n
    wrong = any(not 0 <= p < len(lengths) for p in parents)
    wrong = wrong or any(not 0 <= t <= lengths[p] or -(-t // page) > columns
                         for p, t in zip(parents, tokens))
    if wrong or sum(t % page > 0 for t in tokens) > count:
        return [0] * n, rows, shares, count, sources, targets, 1
    for i, (p, t) in enumerate(zip(parents, tokens)):
        for j in range(t // page):
            rows[i, j] = tables[p, j]
            if 0 <= tables[p, j] < len(shares):
                shares[tables[p, j]] += 1
        if t % page:
            count -= 1
            sources[i], targets[i] = int(tables[p, t // page]), int(stack[count])
            rows[i, t // page] = stack[count]
    return list(tokens), rows, shares, count, sources, targets, 0


def release(lengths, tables, shares, stack, count, named, page):
    """(lengths, shares, stack, count)."""

    lengths, shares, stack = list(lengths), list(shares), list(stack)
    entries = []
    for r in dict.fromkeys(r for r in named if 0 <= r < len(lengths)):
        entries += [int(p) for p in tables[r, :held(lengths[r], page, tables.shape[1])]
                    if 0 <= p < len(shares)]
        lengths[r] = 0
    last = {p: i for i, p in enumerate(entries)}
    for i, p in enumerate(entries):
        shares[p] -= 1
    for i, p in enumerate(entries):
        if last[p] == i and shares[p] < 0:
            stack[count] = p
            count += 1
            shares[p] = 0
    return lengths, shares, stack, count


def compact(lengths, tables, shares, page):
    """(tables, shares, stack, count, sources, targets)."""

    pages, columns = len(shares), tables.shape[1]
    mine = [[int(p) for p in row[:held(n, page, columns)]] for n, row in zip(lengths, tables)]
    used = sorted({p for row in mine for p in row if 0 <= p < pages})
    total = len(used)
    movers = [p for p in used if p >= total]
    holes = [p for p in range(total) if p not in set(used)]
    to = {p: p for p in used} | dict(zip(movers, holes))
    out = np.full(tables.shape, -1)
    for r, row in enumerate(mine):
        for j, p in enumerate(row):
            out[r, j] = to.get(p, -1)
    new = [0] * pages
    for p in used:
        new[to[p]] = shares[p]
    pad = [-1] * (pages // 2 - len(movers))
    stack = list(range(pages - 1, total - 1, -1)) + [-1] * total
    return out, new, stack, pages - total, movers + pad, holes + pad


def check(lengths, tables, shares, stack, count, page):
    """Every page is free, or held by one request more than its shares say."""

    holders = [0] * len(shares)
    for n, row in zip(lengths, tables):
        for p in row[:held(n, page, tables.shape[1])]:
            holders[p] += 1
    free = [int(p) for p in stack[:count]]
    assert len(set(free)) == len(free)
    for p, n in enumerate(holders):
        assert (n == 0) == (p in set(free)), p
        assert shares[p] == max(0, n - 1), p
