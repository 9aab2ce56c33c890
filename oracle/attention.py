"""Attention over packed prompts and over a paged cache in 8 bits, page tables
and the cache's codes, in numpy: the definitions, in 64 bits, row by row."""

from __future__ import annotations

import numpy as np

MOST_CODE = 448.0


# --------------------------------------------------------------- attention


def attend_row(q, k, v, scale):
    """One query row [D] over what it sees, k and v [n, D]: the output and
    the two magnitudes that error bounds go by, sum p |v| and the largest
    sum |q| |k| scale.  Nothing seen gives 0."""

    if not len(k):
        zero = np.zeros(v.shape[1])
        return zero, zero, 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        logits = (k @ q) * scale
        p = np.exp(logits - logits.max())
        p = p / p.sum()
        return p @ v, p @ np.abs(v), float((np.abs(k) @ np.abs(q)).max() * scale)


def prompt(query, key, value, offsets, scale=None):
    """Causal attention of packed sequences: query [T, H, D], key and value
    [T, G, D].  Returns (out, weight, logit) as ``attend_row``'s, [T, H, D],
    [T, H, D] and [T, H]."""

    rows, heads, width = query.shape
    group = heads // key.shape[1]
    scale = width ** -0.5 if scale is None else scale
    out, weight = np.zeros(query.shape), np.zeros(query.shape)
    logit = np.zeros((rows, heads))
    for begin, end in zip(offsets, offsets[1:]):
        for i in range(begin, end):
            for h in range(heads):
                seen = slice(begin, i + 1)
                out[i, h], weight[i, h], logit[i, h] = attend_row(
                    query[i, h], key[seen, h // group], value[seen, h // group], scale)
    return out, weight, logit


def cached(query, keys, values, page_tables, lengths, scale=None):
    """The newest tokens of each request, query [B, n, H, D], over the cache's
    values keys [P, G, page, D'] and values [P, G, D', page]."""

    batch, tokens, heads, width = query.shape
    page = keys.shape[2]
    group = heads // keys.shape[1]
    scale = width ** -0.5 if scale is None else scale
    out, weight = np.zeros(query.shape), np.zeros(query.shape)
    logit = np.zeros((batch, tokens, heads))
    for b, length in enumerate(lengths):
        at = np.arange(length)
        pages = page_tables[b, at // page]
        for h in range(heads):
            k = keys[pages, h // group, at % page, :width]
            v = values[pages, h // group, :width, at % page]
            for i in range(tokens):
                n = max(0, length - tokens + i + 1)
                out[b, i, h], weight[b, i, h], logit[b, i, h] = attend_row(
                    query[b, i, h], k[:n], v[:n], scale)
    return out, weight, logit


# ------------------------------------------------------------- page tables


def extend(lengths, added, page_tables, free_pages, free_count, page, tokens):
    """Page tables, lengths, free count, offsets, positions, slots, overflow."""

    tables = page_tables.copy()
    needs = [-(-(n + m) // page) - -(-n // page) for n, m in zip(lengths, added)]
    offsets = [0]
    for m in added:
        offsets.append(offsets[-1] + m)
    positions, slots = np.full(tokens, -1), np.full(tokens, -1)
    short = (min(list(lengths) + list(added) + [0]) < 0 or sum(needs) > free_count
             or offsets[-1] > tokens
             or any(-(-(n + m) // page) > tables.shape[1] for n, m in zip(lengths, added)))
    if short:
        return tables, list(lengths), free_count, offsets, positions, slots, 1
    top, t = free_count, 0
    for b, (n, m) in enumerate(zip(lengths, added)):
        for column in range(-(-n // page), -(-(n + m) // page)):
            top -= 1
            tables[b, column] = free_pages[top]
        for position in range(n, n + m):
            positions[t] = position
            slots[t] = tables[b, position // page] * page + position % page
            t += 1
    return (tables, [n + m for n, m in zip(lengths, added)], top, offsets, positions, slots, 0)


# ------------------------------------------------------------------- codes


def codes_table() -> np.ndarray:
    """The value of each e4m3 code: sign, 4 bits of exponent (bias 7), 3 of
    mantissa; 0x7f and 0xff are NaN."""

    code = np.arange(256)
    exponent, mantissa = (code >> 3) & 15, code & 7
    x = np.where(exponent == 0, mantissa * 2.0 ** -9,
                 (1 + mantissa / 8) * 2.0 ** (exponent - 7.0))
    x = np.where((code & 127) == 127, np.nan, x)
    return np.where(code & 128, -x, x)


CODES = codes_table()
_POSITIVE = CODES[:127]
# between neighbours lies the tie, which goes to the even code
_TIES = (_POSITIVE[1:] + _POSITIVE[:-1]) / 2


def encode(x) -> np.ndarray:
    """Codes of x: nearest, ties to even; what is not finite is NaN."""

    x = np.asarray(x, dtype=np.float64)
    size = np.minimum(np.where(np.isfinite(x), np.abs(x), 0.0), MOST_CODE)
    below = np.searchsorted(_TIES, size, side="left")
    tie = np.isin(size, _TIES) & (below % 2 == 1)
    code = np.where(tie, below + 1, below) | np.where(np.signbit(x), 128, 0)
    return np.where(np.isfinite(x), code, 127).astype(np.uint8)


def power_scale(most: float) -> float:
    """The least power of two from 2^-100 to 2^119 by which `most` is at most 448."""

    e = -100
    while e < 119 and most > MOST_CODE * 2.0 ** e:
        e += 1
    return 2.0 ** e


def write(x, slots, codes, scales):
    """Writes x [T, H, D] into codes [P, H, page, D'] (uint8) and scales
    [P, H], in place."""

    page = codes.shape[2]
    at = 0
    while at < len(slots):
        end = at + 1
        while (slots[at] >= 0 and end < len(slots) and slots[end] == slots[end - 1] + 1
               and slots[end] % page):
            end += 1
        if slots[at] >= 0:
            into, first = divmod(int(slots[at]), page)
            for h in range(codes.shape[1]):
                rows = x[at:end, h].astype(np.float64)
                finite = np.abs(rows[np.isfinite(rows)])
                scale = power_scale(finite.max() if finite.size else 0.0)
                if first:
                    old = float(scales[into, h])
                    if old < scale:
                        codes[into, h] = encode(CODES[codes[into, h]] * (old / scale))
                    scale = max(old, scale)
                scales[into, h] = scale
                codes[into, h, first:first + end - at] = 0
                codes[into, h, first:first + end - at, :x.shape[2]] = encode(rows / scale)
        at = end
