"""Forks, releases and compaction of cache pages, and their copies, against
page by page Python."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import copy_on_write_sdm_amd as cow
from oracle import pages as ref

pytestmark = pytest.mark.gpu


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def pool(lengths, page, spare, seed, columns=None):
    """(tables, shares, stack, count) of requests that share nothing."""

    rng = np.random.default_rng(seed)
    counts = [-(-n // page) for n in lengths]
    columns = max(counts + [1]) + 2 if columns is None else columns
    order = rng.permutation(sum(counts) + spare)
    tables = np.full((len(lengths), columns), -1)
    at = 0
    for row, n in zip(tables, counts):
        row[:n] = order[at:at + n]
        at += n
    stack = list(order[at:]) + [-7] * at
    return tables, [0] * len(order), stack, spare


def on_device(device, lengths, tables, shares, stack, count):
    return (ints(lengths, device), ints(tables, device).reshape(tables.shape),
            ints(shares, device), ints(stack, device), ints([count], device))


def assert_fork(device, lengths, state, parents, tokens, page):
    tables, shares, stack, count = state
    before = on_device(device, lengths, *state)
    kept = [t.clone() for t in before]
    got = cow.fork_page_tables(*before, ints(parents, device), ints(tokens, device),
                               page_tokens=page)
    want = ref.fork(lengths, tables, shares, stack, count, parents, tokens, page)
    for name, g, w in zip(got._fields, got, want):
        assert g.cpu().numpy().reshape(-1).tolist() == np.asarray(w).reshape(-1).tolist(), name
    assert all(torch.equal(a, b) for a, b in zip(before, kept))
    return want


def assert_release(device, lengths, state, named, page):
    tables, shares, stack, count = state
    before = on_device(device, lengths, *state)
    got = cow.release_page_tables(*before, ints(named, device), page_tokens=page)
    new_lengths, new_shares, new_stack, new_count = ref.release(lengths, tables, shares, stack,
                                                                count, named, page)
    assert got.lengths.tolist() == new_lengths
    assert got.page_shares.tolist() == new_shares
    assert got.free_count.tolist() == [new_count]
    assert before[3].tolist() == new_stack
    assert before[0].tolist() == list(lengths) and before[2].tolist() == list(shares)
    assert np.array_equal(before[1].cpu().numpy(), tables)
    return new_lengths, (tables, new_shares, new_stack, new_count)


def assert_compact(device, lengths, state, page):
    tables, shares, _, _ = state
    before = on_device(device, lengths, *state)[:3]
    kept = [t.clone() for t in before]
    got = cow.compact_page_tables(*before, page_tokens=page)
    want = ref.compact(lengths, tables, shares, page)
    for name, g, w in zip(got._fields, got, want):
        assert g.cpu().numpy().reshape(-1).tolist() == np.asarray(w).reshape(-1).tolist(), name
    assert all(torch.equal(a, b) for a, b in zip(before, kept))
    return want


# the last two are more than one workgroup takes
SIZES = [([5], 16, 3), ([0], 64, 0), ([64, 0, 1, 63, 65, 128], 64, 9),
         ([(37 * i) % 300 for i in range(70)], 32, 90),
         ([(53 * i) % 2049 for i in range(600)], 32, 900),
         ([70000, 5, 40001], 16, 20000), ([(11 * i) % 40 for i in range(5000)], 16, 700)]


@pytest.mark.parametrize("lengths,page,spare", SIZES)
def test_a_life(device, lengths, page, spare):
    """Fork, fork the forks, release some of both, compact, release the rest:
    every page is free or held all the way, and each step is the definition's."""

    rng = np.random.default_rng(len(lengths) + page)
    state = pool(lengths, page, spare, 3)
    n = min(spare, 2 * len(lengths) + 3)
    for _ in range(2):
        parents = rng.integers(0, len(lengths), n).tolist()
        tokens = [lengths[p] if rng.random() < 0.5 else int(rng.integers(0, lengths[p] + 1))
                  for p in parents]
        n = min(n, 4000)
        parents, tokens = parents[:n], tokens[:n]
        tables, shares, stack, count = state
        if sum(t % page > 0 for t in tokens) > count:
            break
        new, rows, shares, count, *_ = assert_fork(device, lengths, state, parents, tokens, page)
        lengths = list(lengths) + new
        state = np.concatenate((tables, rows)), shares, stack, count
        ref.check(lengths, *state, page)
    named = rng.permutation(len(lengths))[:min(4096, 2 * len(lengths) // 3)].tolist()
    lengths, state = assert_release(device, lengths, state, named, page)
    ref.check(lengths, *state, page)
    tables, shares, stack, count, *_ = assert_compact(device, lengths, state, page)
    state = tables, shares, stack, count
    ref.check(lengths, *state, page)
    for at in range(0, len(lengths), 4096):
        rest = list(range(at, min(len(lengths), at + 4096)))
        lengths, state = assert_release(device, lengths, state, rest, page)
    assert state[3] == len(state[1]) and not any(state[1])


@pytest.mark.parametrize("entries,pages,n", [
    (8192, 8192, 1024), (8192 + 8, 8000, 1025), (8192, 8193, 64), (8184, 8192, 1023)])
def test_where_one_workgroup_ends(device, entries, pages, n):
    """The most entries, pages and requests that one workgroup takes, all of
    them held, and one more of each."""

    page, batch = 16, n
    columns = entries // n
    lengths = [page * columns - (i % 3) for i in range(batch)]
    held = batch * columns
    shares = [0] * pages
    order = np.random.default_rng(n).permutation(pages)[:min(pages, held)]
    tables = np.resize(order, held).reshape(batch, columns)      # wraps: shared pages
    for p, c in zip(*np.unique(tables, return_counts=True)):
        shares[p] = int(c) - 1
    free = [p for p in range(pages) if p not in set(order.tolist())]
    state = tables, shares, free + [-1] * (pages - len(free)), len(free)
    assert_fork(device, lengths, state, list(range(batch))[::-1],
                [page * (columns - 1)] * batch, page)
    assert_compact(device, lengths, state, page)
    _, left = assert_release(device, lengths, state, list(range(batch))[::-1], page)
    assert left[3] == pages and not any(left[1])


def test_fork_refused_as_a_whole(device):
    lengths, page = [40, 16, 0], 16
    state = pool(lengths, page, 2, 5)
    for parents, tokens in (([0, 3], [1, 0]), ([-1], [0]), ([0], [41]), ([1], [-1]),
                            ([0, 0, 0], [17, 18, 19]), ([2], [1])):
        assert assert_fork(device, lengths, state, parents, tokens, page)[6] == 1
    assert assert_fork(device, lengths, state, [0, 0, 2, 1], [17, 18, 0, 16], page)[6] == 0
    assert assert_fork(device, lengths, state, [], [], page)[6] == 0
    # a length past its table's columns
    tables, shares, stack, count = state
    narrow = tables[:, :2].copy(), shares, stack, count
    assert assert_fork(device, lengths, narrow, [0], [40], page)[6] == 1


def test_release_names_and_entries(device):
    """Names twice and out of range, entries that are no page, lengths past
    the table, and a list of nothing."""

    lengths, page = [100, 33, 16, 7], 16
    tables, shares, stack, count = pool(lengths, page, 4, 6)
    for named in ([], [2, 2, 1, 2], [9, -1, 3, 4], [3, 1, 0, 2]):
        assert_release(device, lengths, (tables, shares, stack, count), named, page)
    odd = tables.copy()
    odd[0, 1], odd[0, 2] = -1, len(shares) + 5
    assert_release(device, lengths, (odd, shares, stack, count), [0, 1], page)
    assert_release(device, [1 << 30, 33, -5, 7], (tables, shares, stack, count), [0, 2, 3], page)


def test_compact_of_little(device):
    """No request, nothing held, all held, and entries that are no page."""

    page = 16
    assert_compact(device, [], (np.zeros((0, 3), int), [0] * 5, None, None)[:2] + ([0] * 5, 0),
                   page)
    assert_compact(device, [0, 0], pool([0, 0], page, 7, 1), page)
    assert_compact(device, [50, 20], pool([50, 20], page, 0, 2), page)
    assert_compact(device, [16], pool([16], page, 0, 2), page)
    tables, shares, stack, count = pool([50, 20], page, 9, 4)
    tables[0, 1], tables[1, 0] = -3, 99
    assert_compact(device, [50, 20], (tables, shares, stack, count), page)


def cache(layers, pages, heads, page, width, device, seed):
    g = torch.Generator(device=device).manual_seed(seed)

    def bits(*shape):
        return torch.randint(0, 256, shape, generator=g, device=device,
                             dtype=torch.uint8).view(torch.float8_e4m3fn)

    lead = () if layers is None else (layers,)
    return [bits(*lead, pages, heads, page, width),
            torch.rand(*lead, pages, heads, generator=g, device=device),
            bits(*lead, pages, heads, width, page),
            torch.rand(*lead, pages, heads, generator=g, device=device)]


@pytest.mark.parametrize("layers,heads,page,width", [
    (None, 1, 16, 32), (1, 3, 16, 96), (3, 2, 64, 128), (2, 8, 256, 256), (4, 300, 16, 32)])
def test_copies(device, layers, heads, page, width):
    """Pages named in no order, one source twice, entries left out."""

    pages = 12
    tensors = cache(layers, pages, heads, page, width, device, 7)
    want = [t.view(torch.uint8).clone() if t.dtype is not torch.float32 else t.clone()
            for t in tensors]
    sources, targets = [3, 11, 3, -1, 5, 12, 7, 9], [0, 10, 4, 2, -1, 6, 12, 9]
    for t in want:
        pool_axis = t if layers is not None else t.unsqueeze(0)
        for s, d in ((3, 0), (11, 10), (3, 4)):
            pool_axis[:, d] = pool_axis[:, s].clone()
    cow.copy_pages(*tensors, ints(sources, device), ints(targets, device))
    for t, w in zip(tensors, want):
        assert torch.equal(t.view(w.dtype) if t.dtype is not w.dtype else t, w)
    cow.copy_pages(*tensors, ints([], device), ints([], device))


def test_copies_past_four_gigabytes(device):
    """Offsets of more than 32 bits, in the last layer and page."""

    pages, heads, page, width = 72, 32, 256, 256      # 302 MB a layer, twice
    keys = torch.zeros(15, pages, heads, page, width, dtype=torch.uint8, device=device)
    values = torch.zeros(15, pages, heads, width, page, dtype=torch.uint8, device=device)
    scales = [torch.ones(15, pages, heads, device=device) for _ in range(2)]
    keys[14, 71], values[14, 71], scales[0][14, 71] = 5, 6, 0.25
    codes = [t.view(torch.float8_e4m3fn) for t in (keys, values)]
    cow.copy_pages(codes[0], scales[0], codes[1], scales[1], ints([71], device),
                   ints([70], device))
    assert bool((keys[14, 70] == 5).all()) and bool((values[14, 70] == 6).all())
    assert bool((scales[0][14, 70] == 0.25).all()) and int(keys[:14].amax()) == 0
    assert int(keys[14, :70].amax()) == 0 and int(values[14, :70].amax()) == 0


@pytest.mark.parametrize("requests,columns,pages", [(0, 0, 0), (0, 3, 0), (2, 0, 0), (2, 0, 5),
                                                    (2, 3, 0), (3, 2, 1), (0, 3, 4)])
def test_tables_of_nothing(device, requests, columns, pages):
    """No requests, columns or pages, alone and together: empty requests are
    forked and released, and the stack is the pool."""

    page, lengths = 16, [0] * requests
    state = np.full((requests, columns), -1), [0] * pages, list(range(pages)), pages
    named = list(range(requests))
    assert assert_fork(device, lengths, state, named * 2, [0] * (2 * requests), page)[6] == 0
    assert_release(device, lengths, state, named[::-1] + named, page)
    assert_compact(device, lengths, state, page)
