"""Releases of more requests than a launch takes, and one that fails between
its launches."""

from __future__ import annotations

import pytest
import torch

import copy_on_write_sdm_amd as cow
from copy_on_write_sdm_amd import kv_cache
from test_gpu_paged_lifecycle import PAGE, assert_whole

pytestmark = pytest.mark.gpu


def test_a_release_that_fails_half_way_can_be_made_again(device, monkeypatch):
    cache = cow.PagedKVCache(1, 1, 32, capacity=48, pages=9000, page_tokens=PAGE, device=device)
    cache.admit(4000)
    cache.extend([(7 * r) % 40 for r in range(4000)])
    cache.admit(1000)
    free, lengths, tables = cache.free, cache.lengths.clone(), cache.page_tables.clone()
    assert_whole(cache)
    order = list(range(4999, -1, -1))
    real, calls = kv_cache.release_page_tables, []

    def failing(*args, **kw):
        calls.append(args)
        if len(calls) == 2:
            raise MemoryError
        return real(*args, **kw)

    monkeypatch.setattr(kv_cache, "release_page_tables", failing)
    with pytest.raises(MemoryError):
        cache.release(order)
    monkeypatch.undo()
    assert cache.free == free and torch.equal(cache.lengths, lengths)
    assert torch.equal(cache.page_tables, tables)
    assert_whole(cache)
    assert cache.release(order) == 9000 - free
    assert cache.free == 9000 and not cache.lengths.any()
    assert_whole(cache)
