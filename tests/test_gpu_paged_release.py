"""Releases in place, of caches that share nothing, and by the operator that
knows of shares; of more requests than a launch takes, and one that fails between
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
    assert cache.fork([3]) == [4000]           # of 21 tokens: a page is shared
    cache.admit(999)
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
    assert len(calls) == 2
    assert cache.free == free and torch.equal(cache.lengths, lengths)
    assert torch.equal(cache.page_tables, tables)
    assert_whole(cache)
    assert cache.release(order) == 9000 - free
    assert cache.free == 9000 and not cache.lengths.any()
    assert_whole(cache)


def refuse(*args, **kw):
    raise AssertionError("a release by the operator")


@pytest.mark.parametrize("lengths,named", [
    ([40], [0]), ([37, 48, 0, 16, 1], [3, 0, 2]), ([(7 * r) % 300 for r in range(300)],
                                                   list(range(299, 20, -1))),
    ([(7 * r) % 40 for r in range(4000)], list(range(4000)))])
def test_a_cache_that_shares_nothing(device, monkeypatch, lengths, named):
    """One launch in place gives what the operator gives, the same pages in the
    same places of the stack."""

    caches = [cow.PagedKVCache(1, 1, 32, capacity=320, pages=9000, page_tokens=PAGE,
                               device=device) for _ in range(2)]
    for c in caches:
        c.admit(len(lengths))
        c.extend(lengths)
    with monkeypatch.context() as m:
        m.setattr(kv_cache, "release_page_tables", refuse)
        freed = caches[0].release(named)
    with monkeypatch.context() as m:
        m.setattr(kv_cache, "_IN_PLACE_PAGES", 0)
        assert caches[1].release(named) == freed == sum(-(-lengths[r] // PAGE) for r in named)
    a, b = caches
    assert torch.equal(a.free_pages[:a.free], b.free_pages[:b.free])
    assert torch.equal(a.lengths, b.lengths) and torch.equal(a.free_count, b.free_count)
    for c in caches:
        assert_whole(c)
        assert bool((c.page_tables[named] == -1).all())
        with pytest.raises(ValueError, match="no KV cache step"):
            c.take_back()
    assert a.compact() == b.compact()
    if a.requests:
        a.extend(3), b.extend(3)
        assert torch.equal(a.page_tables, b.page_tables)
        assert_whole(a)


def test_what_is_shared_goes_by_the_operator(device, monkeypatch):
    """As long as any page has been shared and is held, and one long request."""

    cache = cow.PagedKVCache(1, 1, 32, capacity=4096, pages=400, page_tokens=PAGE, device=device)
    cache.admit(3)
    cache.extend([33, 20, 2100])
    cache.fork([0], 16)
    with monkeypatch.context() as m:
        m.setattr(kv_cache, "release_page_tables", refuse)
        for named in ([0], [1], [3]):
            with pytest.raises(AssertionError, match="by the operator"):
                cache.release(named)
    assert cache.release([0]) == 2 and cache.release([3]) == 1      # the shared page with the last
    assert_whole(cache)
    with monkeypatch.context() as m:
        m.setattr(kv_cache, "release_page_tables", refuse)
        assert cache.release([1]) == 2                              # nothing is shared any more
        with pytest.raises(AssertionError, match="by the operator"):
            cache.release([2])                                      # 132 pages
    assert cache.release([2]) == 132 and cache.free == 400
    assert_whole(cache)
