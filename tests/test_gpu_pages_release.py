"""cowsdm_pages_release, which returns the pages of requests that share none in
place: against page by page Python, and against release_page_tables, which gives
the same where nothing is shared."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import copy_on_write_sdm_amd as cow
from copy_on_write_sdm_amd import _native as nat
from oracle import pages as ref
from test_gpu_pages import ints, on_device, pool

pytestmark = pytest.mark.gpu


def release(state, named, page):
    """The state itself, changed."""

    lengths, tables, _, stack, count = state
    rc = nat.lib().cowsdm_pages_release(
        lengths.data_ptr(), tables.data_ptr(), *tables.shape, named.data_ptr(), named.numel(),
        stack.data_ptr(), stack.numel(), count.data_ptr(), page,
        nat.stream_handle(lengths.device))
    assert rc == 0


@pytest.mark.parametrize("lengths,page,spare", [
    ([5], 16, 3), ([64, 0, 1, 63, 65, 128], 64, 9), ([(37 * i) % 300 for i in range(700)], 32, 90),
    ([70000, 5, 40001], 16, 20)])
def test_release_in_place(device, lengths, page, spare):
    n = len(lengths)
    tables, shares, stack, count = pool(lengths, page, spare, 3)
    named = np.random.default_rng(n).permutation(n)[:-(-2 * n // 3)].tolist()
    state = on_device(device, lengths, tables, shares, stack, count)
    other = [t.clone() for t in state]
    release(state, ints(named, device), page)
    left, _, pages, top = ref.release(lengths, tables, shares, stack, count, named, page)
    assert state[0].tolist() == left and state[3].tolist() == pages and state[4].item() == top
    held = [-(-k // page) for k in lengths]
    for r in named:
        tables[r, :held[r]] = -1
    assert np.array_equal(state[1].cpu().numpy(), tables)
    same = cow.release_page_tables(*other, ints(named, device), page_tokens=page)
    assert torch.equal(same.lengths, state[0]) and torch.equal(same.free_count, state[4])
    assert torch.equal(other[3], state[3])
    rest = [r for r in range(n) if r not in set(named)]
    release(state, ints(rest + [n, -1], device), page)       # and numbers that are no request
    assert state[4].item() == len(shares) and not state[0].any()
    assert sorted(state[3].tolist()) == list(range(len(shares)))
