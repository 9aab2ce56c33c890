"""Heads normed and rotated by position against the definition in 64 bits, with
angles taken within a turn exactly."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import copy_on_write_sdm_amd as cow
from attention_cases import TINY, UNIT, wide
from oracle import projections as ref

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def normal(*shape, dtype, device, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dtype).to(device)


def assert_rotated(got, x, positions, rotation, weight, eps):
    """A norm's sum of ``width`` squares is off by at most width 2^-24 of
    itself, its root by half of that; root, quotient and products add a few
    units more.  A point on the circle is off by at most 2^-23 (the angle's
    rounding and the polynomials'), the pair's sum by three more roundings."""

    frequencies = rotation.frequencies if rotation is not None else ()
    interleaved = rotation is not None and rotation.interleaved
    want, size = ref.rotate(wide(x), positions.tolist(), frequencies,
                            weight=None if weight is None else wide(weight), eps=eps,
                            interleaved=interleaved)
    error = size * 2.0 ** -21
    if weight is not None:
        error = error + size * (x.shape[-1] / 2 + 6) * 2.0 ** -24
    error = error + UNIT[x.dtype] * (np.abs(want) + error) + TINY[x.dtype]
    off = np.abs(wide(got) - want) - error
    assert got.dtype is x.dtype and got.is_contiguous() and off.max() <= 0, off.max()


def run(device, dtype, rows, heads, kv_heads, width, rotation, norms, positions, eps=1e-6):
    x = normal(rows, heads + 2 * kv_heads, width, dtype=dtype, device=device, seed=1)
    q, k = x[:, :heads], x[:, heads:heads + kv_heads]
    weights = [normal(width, dtype=dtype, device=device, seed=2 + i) if n else None
               for i, n in enumerate(norms)]
    at = torch.tensor(positions, dtype=torch.int32, device=device)
    got = cow.rotate_heads(q, k, at, rotation, query_norm=weights[0], key_norm=weights[1],
                           eps=eps)
    for y, z, w in zip(got, (q, k), weights):
        assert_rotated(y, z, at, rotation, w, eps)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("width,rotated", [
    (8, 8), (32, 32), (40, 40), (64, 64), (64, 24), (72, 8), (80, 80), (96, 48), (128, 128),
    (128, 64), (136, 136), (192, 192), (256, 256), (256, 64), (248, 240)])
def test_widths(device, dtype, interleaved, width, rotated):
    rotation = cow.HeadRotation(rotated, interleaved=interleaved, device=device)
    run(device, dtype, 7, 6, 2, width, rotation, (True, True), [0, 1, 2, 3, 1000, 5, 99])
    run(device, dtype, 3, 1, 1, width, rotation, (False, True), [4, 0, 123456])


@pytest.mark.parametrize("norms", [(True, True), (True, False), (False, False)])
def test_without_a_rotation(device, norms):
    run(device, torch.bfloat16, 5, 3, 3, 64, None, norms, [0] * 5)


def test_far_positions_are_exact(device):
    """In float32 an angle of some 10^9 radians has no digit left."""

    rotation = cow.HeadRotation(64, base=500000.0, device=device)
    far = [2 ** 31 - 1, -2 ** 31, -1, 2 ** 30 + 7, 1 << 20, 16777217, -65537]
    run(device, torch.float32, len(far), 2, 1, 64, rotation, (False, False), far)
    fast = cow.HeadRotation(32, frequencies=[3.0, -2.5, 6.283185307179586, 100.0] * 4,
                            device=device)
    run(device, torch.float32, len(far), 2, 1, 64, fast, (True, True), far)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 32, 8), (64, 4, 4), (4101, 3, 1),
                                                 (4096, 1, 1), (20, 40, 40)])
def test_rows_and_heads(device, dtype, rows, heads, kv_heads):
    rotation = cow.HeadRotation(32, device=device)
    run(device, dtype, rows, heads, kv_heads, 32, rotation, (True, True),
        [(i * 7) % 2560 for i in range(rows)])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows", [4097, 4100])
def test_some_tokens_to_a_workgroup(device, rows, interleaved):
    """Heads whose tokens take a workgroup a step each, and more tokens than
    that many workgroups are launched for: the last has one or two left."""

    rotation = cow.HeadRotation(80, interleaved=interleaved, device=device)
    run(device, torch.float16, rows, 16, 8, 80, rotation, (True, True),
        [(i * 31) % 70000 for i in range(rows)])


def test_sizes_of_the_norm(device):
    """Rows of zeros, the smallest and the largest numbers, with eps and none."""

    rotation = cow.HeadRotation(32, device=device)
    at = torch.zeros(4, dtype=torch.int32, device=device)
    x = normal(4, 2, 32, dtype=torch.float32, device=device, seed=5)
    x[0] = 0.0
    x[1] *= 1e-12
    x[2] *= 1e12
    w = torch.ones(32, device=device)
    for eps in (1e-6, 1e-30):
        got = cow.rotate_heads(x, x, at, rotation, query_norm=w, key_norm=w, eps=eps)
        for y in got:
            assert_rotated(y, x, at, rotation, w, eps)


def test_what_is_not_finite_stays_in_its_row(device):
    rotation = cow.HeadRotation(64, device=device)
    x = normal(6, 3, 64, dtype=torch.bfloat16, device=device, seed=6)
    x[1, 1, 3], x[4, 0, 9] = float("nan"), float("inf")
    w = torch.ones(64, dtype=torch.bfloat16, device=device)
    at = torch.arange(6, dtype=torch.int32, device=device)
    for y in cow.rotate_heads(x, x, at, rotation, query_norm=w, key_norm=w):
        bad = ~torch.isfinite(y).all(dim=-1)
        assert bad.nonzero().tolist() == [[1, 1], [4, 0]]


def test_strides_and_alignment(device):
    """Slices in any order are read as they are, odd ones copied; nothing
    beside them is read into the result."""

    rotation = cow.HeadRotation(40, device=device)
    at = torch.tensor([3, 1, 4, 1, 5], dtype=torch.int32, device=device)
    big = torch.full((4, 5, 64), float("nan"), dtype=torch.float16, device=device)
    big[:, :, 8:48] = normal(4, 5, 40, dtype=torch.float16, device=device, seed=7)
    w = normal(40, dtype=torch.float16, device=device, seed=8)
    turned = big[:, :, 8:48].transpose(0, 1)
    odd = torch.full((5, 4, 45), float("nan"), dtype=torch.float16, device=device)
    odd[:, :, 3:43] = turned
    for x in (turned, odd[:, :, 3:43], turned[:, 1:2].expand(5, 4, 40)):
        got = cow.rotate_heads(x, x[:, :1], at, rotation, query_norm=w, key_norm=w)
        for y, z in zip(got, (x, x[:, :1])):
            assert_rotated(y, z, at, rotation, w, 1e-6)


def test_no_rows(device):
    q, k = cow.rotate_heads(torch.zeros(0, 4, 64, device=device),
                            torch.zeros(0, 2, 64, device=device),
                            torch.zeros(0, dtype=torch.int32, device=device),
                            cow.HeadRotation(64, device=device))
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)


def test_more_than_four_gigabytes(device):
    rows = 33000
    x = normal(rows, 2, 256, dtype=torch.float16, device=device, seed=9)
    q = x.repeat(1, 130, 1)                              # 2.2 billion elements
    at = torch.arange(rows, dtype=torch.int32, device=device)
    rotation = cow.HeadRotation(256, device=device)
    got, _ = cow.rotate_heads(q, x, at, rotation)
    want, _ = cow.rotate_heads(x, x, at, rotation)
    assert torch.equal(got[-5:, -2:], want[-5:]) and torch.equal(got[:5, :2], want[:5])
    assert torch.equal(got[20000:20005, 100:102], want[20000:20005])
