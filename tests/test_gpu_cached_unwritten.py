"""Attention over a paged cache some of whose pages nobody has written."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import copy_on_write_sdm_amd as cow
from test_gpu_kv_cache import TYPES, filled, ints, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 32, 64])
def test_pages_that_nobody_has_written(device, dtype, page):
    """A pool straight from the allocator: pages without a request hold any
    codes and any scale, NaN and infinity too, the pool's first page among
    them."""

    lengths = [1, 10, 70, 0, 129]
    cache, numbers, tables = filled(lengths, 2, 64, page, device, 35)
    q = queries(5, 2, 4, 64, dtype, 36, device)
    want = cow.cached_attention(q, *cache, ints(tables, device), ints(lengths, device))
    for odd in (float("nan"), float("inf"), -1.0, 0.0):
        used = torch.zeros(len(cache[1]) + 1, dtype=torch.bool, device=device)
        pool = []
        for t in cache:
            code = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
            first = torch.full_like(code[:1], 127 if code is not t else odd)
            pool.append(torch.cat((first, code)).view(t.dtype))
        used[torch.from_numpy(tables[tables >= 0] + 1).to(device)] = True
        pool[1][~used], pool[3][~used] = odd, odd
        got = cow.cached_attention(q, *pool, ints(np.where(tables >= 0, tables + 1, -1), device),
                                   ints(lengths, device))
        assert torch.equal(got, want), odd
