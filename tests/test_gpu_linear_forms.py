"""Every form of a product by itself: tiles of each size, their rings from one
step to many, with and without splits, in each type; and float32's second
summation in each.  Each test says which form its sizes take, so that a plan
that takes another one shows here."""

from __future__ import annotations

import pytest
import torch

import copy_on_write_sdm_amd as cow
from copy_on_write_sdm_amd import _native as nat
from test_gpu_linear import assert_linear, normal
from test_linear_plan import plan

pytestmark = pytest.mark.gpu

FLOAT, HALVES = [torch.float32], [torch.float16, torch.bfloat16]

# (types, tile, split, rows, columns, steps of 128 bytes); 65 rows and more, as
# fewer are read once, 16 rows of W a workgroup
FORMS = [
    (FLOAT, (64, 64), False, 65, 33, (1, 2, 3, 4, 5)),
    (FLOAT, (64, 64), False, 130, 901, (9,)),
    (FLOAT, (64, 64), False, 2001, 258, (33,)),
    (FLOAT, (64, 64), True, 65, 33, (9, 17, 33, 65)),
    (FLOAT, (64, 128), False, 200, 4102, (1, 2, 3, 4, 5, 9, 17)),
    (FLOAT, (64, 128), True, 65, 2054, (17,)),
    (FLOAT, (64, 128), True, 65, 1300, (33,)),
    (FLOAT, (64, 128), True, 65, 901, (65,)),
    (FLOAT, (128, 128), False, 2001, 1030, (2, 3, 4, 5, 9, 17)),
    (FLOAT, (128, 128), True, 2910, 130, (33,)),
    (FLOAT, (128, 128), True, 65, 4102, (65,)),
    (FLOAT, (256, 256), False, 5000, 1543, (1, 2, 3)),
    (FLOAT, (256, 256), False, 2500, 4102, (4, 5, 9)),
    (FLOAT, (256, 256), True, 4100, 901, (33,)),
    (FLOAT, (256, 256), True, 2001, 1030, (65,)),
    (HALVES, (64, 64), False, 65, 33, (1, 2, 3, 4, 5, 9)),
    (HALVES, (64, 64), False, 2910, 130, (33,)),
    (HALVES, (64, 64), True, 65, 33, (17, 33, 65)),
    (HALVES, (64, 128), False, 200, 4102, (1, 2, 3, 4, 5, 9, 17)),
    (HALVES, (64, 128), True, 2001, 66, (33,)),
    (HALVES, (64, 128), True, 65, 901, (65,)),
    (HALVES, (128, 128), False, 2001, 1030, (3, 4, 5, 9, 17, 33)),
    (HALVES, (128, 128), True, 200, 4102, (65,)),
    (HALVES, (256, 256), False, 1500, 4102, (1, 2, 3)),
    (HALVES, (256, 256), False, 5000, 1543, (4, 5, 9)),
    (HALVES, (256, 256), True, 4100, 901, (65,)),
]
CASES = [(dtype, tile, split, rows, outer, s) for types, tile, split, rows, outer, steps in FORMS
         for dtype in types for s in steps]


def sizes(dtype, tile, split, rows, outer, steps):
    """The inner size of so many steps, the last one a chunk short of whole
    where their number is odd, and checked to take the form."""

    each = 128 // dtype.itemsize
    inner = steps * each - each // 8 * (steps % 2)
    got, splits, _ = plan(rows, inner, outer, nat.FLOAT_TYPES[dtype])
    assert got == tile and (splits > 1) is split, (got, splits)
    print(f"{dtype} {tile} {splits} splits: {rows} {inner} {outer}", flush=True)
    return inner


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_each_form(device, case):
    dtype, _, _, rows, outer, _ = case
    inner = sizes(*case)
    x = normal(rows, inner, dtype=dtype, device=device, seed=70)
    w = normal(outer, inner, dtype=dtype, device=device, seed=71, scale=inner ** -0.5)
    bias = normal(outer, dtype=dtype, device=device, seed=72)
    residual = normal(rows, outer, dtype=dtype, device=device, seed=73)
    out = assert_linear(x, w, bias, "gelu", residual)
    assert torch.equal(out, cow.linear(x, w, bias, activation="gelu", residual=residual))
    assert_linear(x, w)


@pytest.mark.parametrize("case", [c for c in CASES if c[0] is torch.float32],
                         ids=lambda c: "-".join(str(x) for x in c[1:]))
def test_float32_that_is_summed_again(device, case):
    """The largest numbers, which parts of 16 bits round to infinity, in the
    first and the last tile and step: of some tiles, and splits, only."""

    _, _, _, rows, outer, _ = case
    inner = sizes(*case)
    x = normal(rows, inner, dtype=torch.float32, device=device, seed=74)
    w = normal(outer, inner, dtype=torch.float32, device=device, seed=75, scale=inner ** -0.5)
    most = torch.finfo(torch.float32).max
    x[0, 0], x[-1, -1] = most, -most
    w[0, 0], w[-1, -1] = 0.5, 0.25
    out = assert_linear(x, w)
    assert out[0, 0].item() == pytest.approx(most / 2, rel=1e-6)
    assert out[-1, -1].item() == pytest.approx(-most / 4, rel=1e-6)
    assert torch.equal(out, cow.linear(x, w))


LAST = {(c[0], c[1], c[2]): c for c in CASES}.values()     # each form's longest sum


@pytest.mark.parametrize("case", LAST, ids=lambda c: "-".join(str(x) for x in c))
def test_what_is_not_finite_in_each_form(device, case):
    """NaN stays in its row, and an infinite weight in its column; the rest is
    what it is without them, bit for bit where nothing is summed again."""

    dtype, _, _, rows, outer, _ = case
    inner = sizes(*case)
    x = normal(rows, inner, dtype=dtype, device=device, seed=76)
    w = normal(outer, inner, dtype=dtype, device=device, seed=77, scale=inner ** -0.5)
    x[:, 0] = 1.0
    clean = assert_linear(x, w)
    x[-1, -1], w[-1, 0] = float("nan"), float("inf")
    out = cow.linear(x, w)
    assert bool(torch.isnan(out[-1]).all()) and bool((out[:-1, -1] == float("inf")).all())
    out, clean = out[:-1, :-1], clean[:-1, :-1]
    if dtype is not torch.float32:
        assert torch.equal(out, clean)
        return
    # both within (inner + 4) 2^-24 of the terms' magnitudes, and rounded
    size = x[:-1].double().abs() @ w[:-1].double().abs().t()
    off = (out.double() - clean.double()).abs() - 2 * (inner + 6) * 2.0 ** -24 * size
    assert float(off.max()) <= 0
