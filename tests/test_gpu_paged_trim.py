"""What a trimmed pool gives up, and how far one grows."""

from __future__ import annotations

import pytest
import torch

import copy_on_write_sdm_amd as cow
from test_gpu_paged_lifecycle import PAGE, assert_whole, contents, fill, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layers", [1, 3])
def test_trimmed_memory_is_given_up(device, layers):
    """No tensor of the cache keeps more memory than its own numbers, whatever
    the layers' number."""

    g = torch.Generator().manual_seed(layers)
    cache = cow.PagedKVCache(layers, 2, 32, capacity=64, pages=100, page_tokens=PAGE,
                             device=device)
    cache.admit(3)
    fill(cache, [40, 20, 16], g)
    cache.release([0])
    kept = [contents(cache, r) for r in (1, 2)]
    assert cache.trim_pages(headroom_pages=2) == 100 - 3 - 2
    assert_whole(cache)
    assert all(same(contents(cache, r), k) for r, k in zip((1, 2), kept))
    for name in ("key_pages", "key_scales", "value_pages", "value_scales", "page_tables",
                 "page_shares", "free_pages", "free_count"):
        t = getattr(cache, name)
        assert t.untyped_storage().nbytes() == t.numel() * t.element_size(), name


def test_a_pool_grows_no_further_than_its_operators_count(device):
    """Slots are 32-bit: past them no step, and no trim, would be taken any
    more.  Refused before anything is allocated."""

    cache = cow.PagedKVCache(1, 1, 32, capacity=64, pages=4, page_tokens=PAGE, device=device)
    cache.admit(1)
    cache.extend(20)
    for more in ((1 << 31) // PAGE - 4, 1 << 40):
        with pytest.raises(ValueError, match="fewer than 2\\^31 tokens"):
            cache.grow_pages(more)
    assert cache.free == 2 and cache.key_pages.shape[1] == 4
    cache.take_back()                          # nothing has changed
    cache.grow_pages(3)
    assert cache.free == 7
    assert_whole(cache)
