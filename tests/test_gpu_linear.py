"""Projections with bias, activation and residual against the definition in 64
bits."""

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


def assert_linear(x, weight, bias=None, activation=None, residual=None):
    """The sum of ``inner`` rounded products and the bias in float32 is off by
    at most (inner + 2) 2^-24 of the terms' magnitudes (and by 2^-23 more
    where float32 products are made of three parts of each number, whose least
    products are left out).  No activation's slope
    is over 1.13.  An activation is off by at most 2^-21 of its argument:
    exponential and reciprocal are within 2^-22 and the rest within a few units
    of 2^-24, or 0.75e-7 for the approximated normal distribution.  The sum
    with the residual rounds in float32 and once in the type; what may lie
    past its largest number may be infinite."""

    out = cow.linear(x, weight, bias, activation=activation, residual=residual)
    inner, outer = weight.shape[1], weight.shape[0]
    assert out.shape == (*x.shape[:-1], outer) and out.dtype is x.dtype and out.is_contiguous()
    rows = out.numel() // outer
    want, before, size = ref.linear(
        wide(x).reshape(rows, inner), wide(weight), None if bias is None else wide(bias),
        activation, None if residual is None else wide(residual).reshape(rows, outer))
    unit = UNIT[x.dtype]
    error = (inner + (4 if x.dtype is torch.float32 else 2)) * 2.0 ** -24 * size
    if activation is not None:
        error = 1.13 * error + 2.0 ** -21 * np.abs(before)
    error = error + 2.0 ** -24 * (np.abs(want) + error)
    error = error + unit * (np.abs(want) + error) + TINY[x.dtype]
    got = wide(out).reshape(rows, outer)
    past = np.abs(want) + error >= torch.finfo(x.dtype).max
    past &= np.isinf(got) & ((got > 0) == (want > 0))
    off = np.abs(np.where(past, want, got) - want) - error
    assert off.max() <= 0, (off.max(), int((off > 0).sum()), off.size)
    return out


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,inner,outer", [
    (1, 8, 4), (1, 4096, 1024), (5, 72, 33), (16, 128, 384), (17, 264, 130), (33, 512, 48),
    (64, 128, 384), (64, 2056, 100), (65, 64, 65), (130, 520, 260), (300, 96, 1), (129, 1024, 513),
    (700, 136, 640), (1, 8, 1), (2000, 64, 2100)])
def test_sizes(device, dtype, rows, inner, outer):
    print(f"{dtype} {rows} {inner} {outer}", flush=True)
    x = normal(rows, inner, dtype=dtype, device=device, seed=1)
    w = normal(outer, inner, dtype=dtype, device=device, seed=2, scale=inner ** -0.5)
    assert_linear(x, w)
    assert_linear(x, w, normal(outer, dtype=dtype, device=device, seed=3), "gelu",
                  normal(rows, outer, dtype=dtype, device=device, seed=4))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large_tiles(device, dtype):
    """More than one workgroup of the largest tiles a CU, with odd ends."""

    assert_large(device, dtype, 4099, 200, 4102)


@pytest.mark.parametrize("inner", [8, 64, 72, 128, 136, 320, 328, 512, 1032])
def test_large_tiles_of_few_steps(device, inner):
    """The ring of half tiles from one step on, whole and with an end."""

    assert_large(device, torch.bfloat16, 2500, inner, 8196)


def assert_large(device, dtype, rows, inner, outer):
    x = normal(rows, inner, dtype=dtype, device=device, seed=5)
    w = normal(outer, inner, dtype=dtype, device=device, seed=6, scale=0.1)
    assert_linear(x, w, normal(outer, dtype=dtype, device=device, seed=7), "silu")


def workspace(rows, inner, outer, dtype):
    from copy_on_write_sdm_amd import _native as nat

    return nat.lib().cowsdm_linear_workspace_bytes(rows, inner, outer, nat.FLOAT_TYPES[dtype])


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,inner,outer", [
    (100, 4000, 100), (20, 8192, 515), (70, 2056, 66), (128, 8192, 512), (64, 4096, 1024),
    (256, 2568, 256), (1, 16384, 64), (65, 1096, 1), (2910, 7848, 1421)])
def test_splits_of_the_summed_axis(device, dtype, rows, inner, outer):
    """Sums joined in a workspace: of aligned and of odd widths, with the
    epilogue in the join."""

    assert workspace(rows, inner, outer, dtype) > 0
    x = normal(rows, inner, dtype=dtype, device=device, seed=30)
    w = normal(outer, inner, dtype=dtype, device=device, seed=31, scale=inner ** -0.5)
    out = assert_linear(x, w, normal(outer, dtype=dtype, device=device, seed=32), "gelu_tanh",
                        normal(rows, outer, dtype=dtype, device=device, seed=33))
    assert torch.equal(out, cow.linear(
        x, w, normal(outer, dtype=dtype, device=device, seed=32), activation="gelu_tanh",
        residual=normal(rows, outer, dtype=dtype, device=device, seed=33)))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,inner,outer", [
    (1, 1, 1), (3, 7, 5), (70, 131, 67), (16, 2, 129), (40, 4, 8), (200, 100, 3)])
def test_widths_that_are_not_aligned(device, dtype, rows, inner, outer):
    x = normal(rows, inner, dtype=dtype, device=device, seed=8)
    w = normal(outer, inner, dtype=dtype, device=device, seed=9)
    assert_linear(x, w, normal(outer, dtype=dtype, device=device, seed=10), "relu",
                  normal(rows, outer, dtype=dtype, device=device, seed=11))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("activation", [None, "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [3, 150])
def test_activations(device, dtype, activation, rows):
    """Arguments from the smallest to where the types end."""

    inner = 16
    x = normal(rows, inner, dtype=dtype, device=device, seed=12)
    w = normal(96, inner, dtype=dtype, device=device, seed=13)
    w *= torch.logspace(-6, 3, 96, device=device).to(dtype)[:, None]
    assert_linear(x, w, activation=activation)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows", [6, 40, 140])
def test_strides(device, dtype, rows):
    """Slices whose neighbours are NaN, rows far apart, and axes turned."""

    inner, outer = 104, 70
    nan = float("nan")
    big = torch.full((rows + 2, 3, inner + 24), nan, dtype=dtype, device=device)
    big[1:-1, 1, 8:8 + inner] = normal(rows, inner, dtype=dtype, device=device, seed=14)
    x = big[1:-1, 1, 8:8 + inner]
    store = torch.full((outer + 1, inner + 8), nan, dtype=dtype, device=device)
    store[:outer, :inner] = normal(outer, inner, dtype=dtype, device=device, seed=15)
    w = store[:outer, :inner]
    both = normal(rows, 2 * outer + 1, dtype=dtype, device=device, seed=16)
    residual = both[:, 1:outer + 1]
    bias = normal(outer, 2, dtype=dtype, device=device, seed=17)[:, 1]
    assert_linear(x, w, bias, None, residual)
    odd = big[1:-1, 1, 9:8 + inner]                     # rows that are not aligned
    assert_linear(odd, store[:outer, 1:inner], bias, "relu", residual)
    turned = normal(inner, rows, dtype=dtype, device=device, seed=18).t()
    assert_linear(turned, normal(inner, outer, dtype=dtype, device=device, seed=19).t())
    one = normal(1, inner, dtype=dtype, device=device, seed=20).expand(rows, inner)
    assert_linear(one, w[:1].expand(outer, inner), residual=residual[:1].expand(rows, outer))
    assert_linear(x.reshape(2, rows // 2, inner), w, residual=residual.reshape(2, -1, outer))
    assert_linear(x[0], w, residual=residual[0])


@pytest.mark.parametrize("rows,inner,outer", [(70, 64, 50), (300, 520, 260), (130, 4096, 40),
                                              (4100, 40, 4100)])
def test_float32_of_all_sizes(device, rows, inner, outer):
    """Numbers of every binary order in one sum, the largest among them: what
    three parts of 16 bits cannot hold is summed as it is."""

    g = torch.Generator().manual_seed(40)
    x = torch.randn(rows, inner, generator=g) * 2.0 ** torch.randint(-60, 20, (rows, inner),
                                                                    generator=g)
    w = torch.randn(outer, inner, generator=g) * 2.0 ** torch.randint(-20, 20, (outer, inner),
                                                                     generator=g)
    x[3, 1], w[5, 1] = 3.4028234e38, 0.5
    x, w = x.to(device), w.to(device)
    out = assert_linear(x, w)
    assert bool(torch.isfinite(out[:, 5]).all()) and float(out[3, 5]) > 1.7e38


@pytest.mark.parametrize("power", [-100, -108, -116])
def test_float32_near_the_smallest(device, power):
    """Numbers whose later parts are below bfloat16's normal ones."""

    x = normal(130, 72, dtype=torch.float32, device=device, seed=41) * 2.0 ** power
    w = normal(200, 72, dtype=torch.float32, device=device, seed=42)
    assert_linear(x, w)
    assert_linear(w, x)


@pytest.mark.parametrize("rows", [4, 60, 200])
@pytest.mark.parametrize("dtype", FLOATS)
def test_what_is_not_finite_stays_in_its_row_and_column(device, dtype, rows):
    x = normal(rows, 72, dtype=dtype, device=device, seed=21)
    w = normal(50, 72, dtype=dtype, device=device, seed=22)
    x[2, 5], w[7, 70] = float("nan"), float("inf")
    x[:, 70] = 1.0
    residual = normal(rows, 50, dtype=dtype, device=device, seed=23)
    residual[0, 3] = float("-inf")
    out = cow.linear(x, w, residual=residual)
    assert bool(torch.isnan(out[2]).all())
    others = [r for r in range(rows) if r != 2]
    assert bool((out[others, 7] == float("inf")).all())
    assert out[0, 3] == float("-inf")
    rest = torch.ones_like(out, dtype=torch.bool)
    rest[2], rest[:, 7], rest[0, 3] = False, False, False
    assert bool(torch.isfinite(out[rest]).all())


def test_nothing_to_sum_and_nothing_to_write(device):
    x = torch.zeros(3, 0, device=device)
    bias = torch.tensor([1.0, -2.0], device=device)
    assert cow.linear(x, torch.zeros(2, 0, device=device)).tolist() == [[0.0, 0.0]] * 3
    out = cow.linear(x, torch.zeros(2, 0, device=device), bias, activation="relu",
                     residual=torch.ones(3, 2, device=device))
    assert out.tolist() == [[2.0, 1.0]] * 3
    assert cow.linear(torch.zeros(0, 8, device=device),
                      torch.zeros(2, 8, device=device)).shape == (0, 2)
    assert cow.linear(torch.zeros(2, 8, device=device),
                      torch.zeros(0, 8, device=device)).shape == (2, 0)


def test_more_than_four_gigabytes(device):
    """Offsets of more than 32 bits in the output and in x."""

    rows, inner, outer = 70001, 8, 32768
    x = normal(rows, inner, dtype=torch.float16, device=device, seed=24)
    w = normal(outer, inner, dtype=torch.float16, device=device, seed=25)
    out = cow.linear(x, w)
    for part in (slice(0, 3), slice(32767, 32770), slice(rows - 3, rows)):
        assert torch.equal(out[part], cow.linear(x[part], w))
    del out
    far = torch.zeros(2100, 1 << 20, dtype=torch.float16, device=device)
    far[:, :inner] = x[:2100]
    assert torch.equal(cow.linear(far[:, :inner], w[:100]), cow.linear(x[:2100], w[:100]))


def test_the_residual_may_be_written_over(device):
    """At the C entry, where the output is the caller's."""

    from copy_on_write_sdm_amd import _native as nat

    for rows in (9, 100):
        x = normal(rows, 64, dtype=torch.bfloat16, device=device, seed=26)
        w = normal(128, 64, dtype=torch.bfloat16, device=device, seed=27)
        r = normal(rows, 128, dtype=torch.bfloat16, device=device, seed=28)
        want = cow.linear(x, w, residual=r)
        a = nat.Linear(x.data_ptr(), w.data_ptr(), None, r.data_ptr(), r.data_ptr(), 64, 64, 128,
                       rows, 64, 128, 2, 0)
        assert nat.lib().cowsdm_linear(a, None, 0, nat.stream_handle(device)) == 0
        assert torch.equal(r, want)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("activation", ["relu", "gelu", "gelu_tanh", "silu"])
def test_activations_of_what_is_not_finite(device, dtype, activation):
    """As the formulas have it: NaN stays, infinity stays, and minus infinity
    times nothing is NaN (of relu 0); the largest numbers stay or vanish."""

    x = torch.zeros(70, 8, dtype=dtype, device=device)
    w = torch.zeros(6, 8, dtype=dtype, device=device)
    most = torch.finfo(dtype).max
    bias = torch.tensor([float("nan"), float("inf"), float("-inf"), most, -most, 0.0],
                        dtype=dtype, device=device)
    out = cow.linear(x, w, bias, activation=activation)
    want = torch.tensor([float("nan"), float("inf"), 0.0 if activation == "relu" else float("nan"),
                         most, 0.0, 0.0], dtype=dtype, device=device)
    assert torch.equal(out.isnan(), want.isnan().expand(70, 6))
    assert torch.equal(out.nan_to_num(nan=1.0, posinf=2.0), want.nan_to_num(nan=1.0, posinf=2.0)
                       .expand(70, 6))


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,inner,outer", [
    (100, 4001, 100), (1, 8191, 65), (70, 2055, 66), (64, 4096, 1024), (2910, 2504, 131),
    (130, 63, 600), (130, 65, 600)])
def test_splits_of_rows_that_are_not_aligned(device, dtype, rows, inner, outer):
    """Widths that no row of which is aligned, and operands that start one
    element past an aligned address, between NaN."""

    def loose(count, seed, scale=1.0):
        flat = torch.full((count * inner + 16,), float("nan"), dtype=dtype, device=device)
        part = flat[1:1 + count * inner].view(count, inner)
        part.copy_(normal(count, inner, dtype=dtype, device=device, seed=seed, scale=scale))
        return part

    x, w = loose(rows, 50), loose(outer, 51, inner ** -0.5)
    assert x.data_ptr() % 16 and w.data_ptr() % 16
    assert_linear(x, w, normal(outer, dtype=dtype, device=device, seed=52), "silu",
                  normal(rows, outer, dtype=dtype, device=device, seed=53))
