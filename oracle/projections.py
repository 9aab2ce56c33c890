"""Projections with their epilogue, and heads normed and rotated by position, in
64 bits from their definitions, with the magnitudes that error bounds go by."""

from __future__ import annotations

import math
from fractions import Fraction

import numpy as np
from scipy.special import erf

# pi to 60 digits
PI = Fraction(3141592653589793238462643383279502884197169399375105820974944, 10 ** 60)


def activated(y, activation):
    with np.errstate(over="ignore", invalid="ignore"):
        if activation == "relu":
            return np.where(y < 0, 0.0, y)
        if activation == "gelu":
            return 0.5 * y * (1 + erf(y / math.sqrt(2)))
        if activation == "gelu_tanh":
            return 0.5 * y * (1 + np.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        if activation == "silu":
            return y / (1 + np.exp(-y))
        return y


def linear(x, weight, bias=None, activation=None, residual=None):
    """(out, before, size): the result, what the activation is of, and the sum
    of the magnitudes that this is a sum of."""

    y, size = x @ weight.T, np.abs(x) @ np.abs(weight).T
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    out = activated(y, activation)
    if residual is not None:
        out = residual + out
    return out, y, size


def point(position, frequency):
    """(cos, sin) of position * frequency, the angle taken within a turn exactly."""

    turns = Fraction(frequency) * int(position) / (2 * PI)
    angle = float((turns - round(turns)) * 2 * PI)
    return math.cos(angle), math.sin(angle)


def rotate(x, positions, frequencies, *, weight=None, eps=1e-6, interleaved=False):
    """(out, size): heads x [T, H, D], and for each element the magnitudes it
    is a sum of."""

    y = np.array(x, dtype=np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(axis=-1, keepdims=True) + eps) * weight
    half = len(frequencies)
    out, size = y.copy(), np.abs(y)
    if not half:
        return out, size
    table = np.array([[point(p, f) for f in frequencies] for p in positions])
    cos, sin = table[:, None, :, 0], table[:, None, :, 1]
    first = np.arange(0, 2 * half, 2) if interleaved else np.arange(half)
    second = first + 1 if interleaved else first + half
    a, b = y[..., first], y[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    size[..., first] = size[..., second] = np.abs(a) + np.abs(b)
    return out, size
