"""How far a caller that keeps the tensors from before a call can go back: past
forks and compactions, and after a release to states of no larger a free count."""

from __future__ import annotations

import numpy as np
import pytest

import copy_on_write_sdm_amd as cow
from oracle import pages as ref
from test_gpu_pages import ints, on_device, pool

pytestmark = pytest.mark.gpu

PAGE = 16


def whole(state):
    """Every page of the state is free or held, once for each sharer."""

    lengths, tables, shares, stack, count = state
    ref.check(lengths.tolist(), tables.cpu().numpy(), shares.tolist(), stack.tolist(),
              count.item(), PAGE)


def forked(state, parents, tokens):
    import torch

    lengths, tables, shares, stack, count = state
    fork = cow.fork_page_tables(*state, ints(parents, lengths.device),
                                ints(tokens, lengths.device), page_tokens=PAGE)
    assert fork.overflow.item() == 0
    return (torch.cat((lengths, fork.lengths)), torch.cat((tables, fork.page_tables)),
            fork.page_shares, stack, fork.free_count)


def released(state, named):
    lengths, tables, shares, stack, count = state
    left = cow.release_page_tables(*state, ints(named, lengths.device), page_tokens=PAGE)
    return left.lengths, tables, left.page_shares, stack, left.free_count


@pytest.mark.parametrize("requests", [3, 900])          # one workgroup, and launches of their own
def test_going_back(device, requests):
    lengths = [(37 * i + 21) % 200 for i in range(requests)]
    tables, shares, stack, count = pool(lengths, PAGE, 3 * requests, 8)
    first = on_device(device, lengths, tables, shares, stack, count)
    parents, tokens = list(range(requests)), [n - n // 3 for n in lengths]
    # a fork by itself, and more than once
    for _ in range(2):
        second = forked(first, parents, tokens)
        whole(second)
        whole(first)
    # a release by itself: what was there before it stays whole, and goes on
    some = list(range(0, requests, 2)) + list(range(requests, 2 * requests, 3))
    kept = second[3].clone()
    for _ in range(2):
        third = released(second, some)
        whole(third)
        whole(second)
    held = second[4].item()
    assert np.array_equal(second[3][:held].cpu().numpy(), kept[:held].cpu().numpy())
    whole(forked(second, parents, tokens))
    whole(released(second, list(range(requests, 2 * requests))))
    # a compaction has a stack of its own
    moved = cow.compact_page_tables(*second[:3], page_tokens=PAGE)
    whole((second[0], moved.page_tables, moved.page_shares, moved.free_pages, moved.free_count))
    whole(second)


def test_going_back_past_a_fork_is_void():
    """Why no further (on the definition): the release has written over what the
    fork took off the stack."""

    lengths, tables, shares, stack, count = [20], np.array([[0, 1]]), [0] * 4, [3, 2, -1, -1], 2
    new, rows, more, left, *_ = ref.fork(lengths, tables, shares, stack, count, [0], [20], PAGE)
    assert rows.tolist() == [[0, 2]] and left == 1
    both = np.concatenate((tables, rows))
    _, _, after, _ = ref.release(lengths + new, both, more, stack, left, [0], PAGE)
    assert after[:2] == [3, 1]                           # 2 is gone from the first state's stack
