"""Inputs and error bounds of the attention tests."""

from __future__ import annotations

import numpy as np
import torch

# half a unit in the last place of 1 and of the smallest normal number
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def bound(out, weight, logit, dtype, *, width, longest, largest, parts=1):
    """How far a kernel's output may be from the definition's, element by
    element.

    A logit is a sum of ``width`` rounded products in float32: it is off by at
    most width * 2^-24 of its terms' magnitudes (``logit``, the largest of a
    row), scaled and moved by the maximum in a few more roundings of a number
    no larger than that.  A probability is off by that twice (it and the
    sum), by the exponential (2 units) and by its rounding to the type the
    product takes it in, times ``weight`` = sum p |v|; sums over ``longest``
    keys add 2^-24 of it each.  The output rounds once more.  Probabilities
    below the type's normal numbers round in steps of its smallest one.
    ``parts``: numbers of bfloat16 that carry a probability."""

    unit = UNIT[dtype]
    product = unit if parts == 1 else 2.0 ** (-8 * parts - 1) + 2.0 ** -24
    relative = (product + 2 * ((width + 8) * 2.0 ** -24 * (logit[..., None] + 1) + 2.0 ** -22)
                + 2 * longest * 2.0 ** -24)
    floor = TINY[dtype] + longest * (TINY[dtype] if parts == 1 else 2.0 ** -133) * largest
    return relative * weight * 1.01 + unit * (np.abs(out) + weight * relative) + floor


def assert_within(got: torch.Tensor, out, weight, logit, *, longest, values, parts=1):
    finite = np.abs(values[np.isfinite(values)])
    largest = float(finite.max()) if finite.size else 0.0
    tolerance = bound(out, weight, logit, got.dtype, width=got.shape[-1], longest=longest,
                      largest=largest, parts=parts)
    x = got.double().cpu().numpy()
    same = np.isfinite(out)
    assert np.array_equal(np.isnan(x), np.isnan(out))
    assert np.array_equal(x[~same & ~np.isnan(out)], out[~same & ~np.isnan(out)])
    off = np.abs(x[same] - out[same]) - tolerance[same]
    assert not off.size or off.max() <= 0, (off.max(), int((off > 0).sum()), off.size)


def packed(lengths, heads, kv_heads, width, dtype, seed, device, *, gap=0):
    """Slices of one fused projection, as a model holds them, with `gap` rows
    of no sequence before and after, and the offsets."""

    g = torch.Generator().manual_seed(seed)
    rows = sum(lengths) + 2 * gap
    x = (1.3 * torch.randn(rows, heads + 2 * kv_heads, width, generator=g)).to(dtype).to(device)
    offsets = np.cumsum([gap] + list(lengths))
    return (x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:],
            torch.tensor(offsets, dtype=torch.int32, device=device))


def wide(t: torch.Tensor) -> np.ndarray:
    return t.double().cpu().numpy()
