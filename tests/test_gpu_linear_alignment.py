"""Products of aligned widths whose rows do not start on 16 bytes all the same:
by an operand's address, or by a stride."""

from __future__ import annotations

import pytest
import torch

import copy_on_write_sdm_amd as cow
from copy_on_write_sdm_amd import _native as nat
from test_gpu_linear import FLOATS, assert_linear, normal
from test_linear_plan import plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,inner,outer", [(1, 4096, 1024), (8, 2048, 200), (33, 1096, 64),
                                              (64, 264, 70), (130, 4096, 66), (300, 64, 140)])
def test_views_of_something_wider(device, dtype, rows, inner, outer):
    """x, W or both one element past an aligned address, or in rows of an odd
    length, with NaN round them: the same sums as of aligned copies' bounds."""

    def within(count, wide, first, seed, scale=1.0):
        big = torch.full((count, wide), float("nan"), dtype=dtype, device=device)
        part = big[:, first:first + inner]
        part.copy_(normal(count, inner, dtype=dtype, device=device, seed=seed, scale=scale))
        return part

    bias = normal(outer, dtype=dtype, device=device, seed=62)
    residual = normal(rows, outer, dtype=dtype, device=device, seed=63)
    splits = plan(rows, inner, outer, nat.FLOAT_TYPES[dtype], False)[1]
    for wide, first in ((inner + 16, 1), (inner + 9, 0), (inner + 9, 8)):
        print(f"{dtype} {rows} {inner} {outer} in {splits} splits, {first} of {wide}", flush=True)
        x = within(rows, wide, first, 60)
        w = within(outer, wide, first, 61, inner ** -0.5)
        for a, b in ((x, w), (x, w.contiguous()), (x.contiguous(), w)):
            out = assert_linear(a, b, bias, "gelu", residual)
            assert torch.equal(out, cow.linear(a, b, bias, activation="gelu", residual=residual))


def test_odd_views_of_nothing_to_sum(device):
    x, w = torch.zeros(9, device=device)[1:1].view(1, 0).expand(3, 0), torch.zeros(2, 0,
                                                                                   device=device)
    bias = torch.tensor([1.0, -2.0], device=device)
    assert cow.linear(x, w, bias).tolist() == [[1.0, -2.0]] * 3
    at = torch.zeros(9, device=device).data_ptr()
    for rows in (3, 300):
        out = torch.empty(rows, 2, device=device)
        a = nat.Linear(at + 4, at + 4, bias.data_ptr(), None, out.data_ptr(), 0, 0, 0, rows, 0, 2,
                       0, 0)
        assert nat.lib().cowsdm_linear(a, None, 0, nat.stream_handle(device)) == 0
        assert out.tolist() == [[1.0, -2.0]] * rows
