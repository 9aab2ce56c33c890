"""extend_page_tables with a free stack smaller than the pool."""

from __future__ import annotations

import numpy as np
import pytest

import copy_on_write_sdm_amd as cow
from oracle import attention as ref
from test_gpu_kv_cache import ints, pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 64])
def test_a_stack_smaller_than_the_pool(device, page):
    """The stack's size says nothing of the pool's: requests hold pages whose
    numbers are larger than the stack has entries."""

    lengths, added = [5 * page + 3, page - 1, 0, 7], [1, page, 2 * page + 1, 0]
    tables, free = pool(lengths, page, 8, 6, 61)
    stack = free[:6]
    want = ref.extend(lengths, added, tables, stack, 6, page, sum(added))
    assert tables.max() >= len(stack) and not want[6]
    t = ints(tables, device)
    step = cow.extend_page_tables(ints(lengths, device), ints(added, device), t,
                                  ints(stack, device), ints([6], device), page_tokens=page,
                                  tokens=sum(added))
    for name, x, y in zip(("tables", *cow.PageTableStep._fields), (t, *step), want):
        assert np.array_equal(x.cpu().numpy().reshape(-1), np.asarray(y).reshape(-1)), name


def test_table_entries_that_are_no_pages(device):
    """They give no slot, or one that lies past every pool."""

    tables = np.array([[-1], [-(1 << 31)], [(1 << 31) - 1], [1 << 27], [(1 << 27) - 1]])
    step = cow.extend_page_tables(ints([1] * 5, device), ints([1] * 5, device),
                                  ints(tables, device), ints([0], device), ints([1], device),
                                  page_tokens=16, tokens=5)
    assert step.slots.tolist() == [-1, -1, -1, -1, (1 << 31) - 15]
