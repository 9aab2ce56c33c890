"""The paged cache in 8 bits against its definitions (oracle/attention.py):
page tables and slots exactly, codes and scales bit for bit, and the attention
over them within derived bounds."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import copy_on_write_sdm_amd as cow
from attention_cases import assert_within, wide
from oracle import attention as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
PARTS = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}


def ints(values, device):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device=device)


def pool(lengths, page, columns, spare, seed):
    """Page tables of requests holding `lengths` tokens and the free stack."""

    rng = np.random.default_rng(seed)
    counts = [-(-n // page) for n in lengths]
    order = rng.permutation(sum(counts) + spare)
    tables, at = np.full((len(lengths), columns), -1), 0
    for b, n in enumerate(counts):
        tables[b, :n] = order[at:at + n]
        at += n
    free = np.full(sum(counts) + spare, -1)
    free[:spare] = order[at:]
    return tables, free


# ------------------------------------------------------------- page tables


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("lengths,added", [
    ([0], [1]), ([5], [0]), ([0, 0, 0], [0, 0, 0]), ([64, 63, 65, 0], [1, 1, 1, 1]),
    ([0, 100, 0, 7, 16, 300], [40, 0, 257, 9, 16, 1]), ([15] * 300, [2] * 300),
    (list(range(0, 700)), [(i * 7) % 5 for i in range(700)]), ([3], [5000])])
def test_extend(device, page, lengths, added):
    columns = -(-(max(lengths) + max(added)) // page) + 2
    need = sum(-(-(n + m) // page) - -(-n // page) for n, m in zip(lengths, added))
    tables, free = pool(lengths, page, columns, need + 3, 1)
    tokens = sum(added) + 5
    want = ref.extend(lengths, added, tables, free, need + 3, page, tokens)
    t = ints(tables, device)
    step = cow.extend_page_tables(ints(lengths, device), ints(added, device), t,
                                  ints(free, device), ints([need + 3], device),
                                  page_tokens=page, tokens=tokens)
    got = (t, *step)
    for name, x, y in zip(("tables", *cow.PageTableStep._fields), got, want):
        assert x.dtype == torch.int32
        assert np.array_equal(x.cpu().numpy().reshape(-1), np.asarray(y).reshape(-1)), name


@pytest.mark.parametrize("short", ["pages", "columns", "tokens", "negative", "none"])
def test_extend_refuses_whole_steps(device, short):
    lengths, added, page = [10, 30, 0], [10, 10, -1 if short == "negative" else 40], 16
    columns = 2 if short == "columns" else 4
    tables, free = pool(lengths, page, columns, 9, 2)
    need = 4 if short == "pages" else 5
    tokens = 59 if short == "tokens" else 60
    t = ints(tables, device)
    step = cow.extend_page_tables(ints(lengths, device), ints(added, device), t,
                                  ints(free, device), ints([need], device), page_tokens=page,
                                  tokens=tokens)
    assert step.overflow.item() == (short != "none")
    if short != "none":
        assert np.array_equal(t.cpu().numpy(), tables)
        assert step.lengths.tolist() == lengths and step.free_count.item() == need
        assert (step.slots == -1).all() and (step.positions == -1).all()


def test_extend_into_given_tensors(device):
    lengths, added, page = [10, 30], [10, 40], 16
    tables, free = pool(lengths, page, 8, 9, 3)
    args = (ints(lengths, device), ints(added, device), ints(tables, device),
            ints(free, device), ints([9], device))
    out = [torch.full((n,), 77, dtype=torch.int32, device=device) for n in (2, 1, 3, 50, 50, 1)]
    step = cow.extend_page_tables(*args, page_tokens=page, tokens=50, out=out)
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(step, out))
    want = ref.extend(lengths, added, tables, free, 9, page, 50)
    assert step.slots.tolist() == want[5].tolist() and step.free_count.item() == want[2]
    # the same call again gives the same: nothing it reads has changed
    again = cow.extend_page_tables(*args, page_tokens=page, tokens=50)
    assert all(torch.equal(a, b) for a, b in zip(step, again))
    for i, x in ((0, args[0]), (1, args[4])):
        bad = list(out)
        bad[i] = x
        with pytest.raises(ValueError, match="over the old"):
            cow.extend_page_tables(*args, page_tokens=page, tokens=50, out=bad)


# ------------------------------------------------------------------- write


def empty_cache(pages, heads, width, page, device, seed=0):
    """A pool whose memory holds anything at all, NaN codes too."""

    padded = cow.cache_width(width)
    g = torch.Generator().manual_seed(seed)

    def codes(*shape):
        return torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).to(device).view(
            torch.float8_e4m3fn)

    return [codes(pages, heads, page, padded),
            torch.full((pages, heads), 2.0 ** -3, device=device),
            codes(pages, heads, padded, page),
            torch.full((pages, heads), 2.0 ** -3, device=device)]


def host(cache):
    keys, ks, values, vs = cache
    return [keys.view(torch.uint8).cpu().numpy().copy(), ks.double().cpu().numpy(),
            values.view(torch.uint8).cpu().numpy().swapaxes(2, 3).copy(),
            vs.double().cpu().numpy()]


def assert_cache(cache, want):
    got = host(cache)
    for name, x, y in zip(("keys", "key scales", "values", "value scales"), got, want):
        if x.dtype == np.uint8:      # any NaN is NaN
            x, y = (np.where((t & 127) == 127, 127, t) for t in (x, y))
        assert np.array_equal(x, y), name


def write_both(cache, want, key, value, slots):
    ref.write(wide(key), slots, want[0], want[1])
    ref.write(wide(value), slots, want[2], want[3])
    cow.write_kv_cache(key, value, ints(slots, key.device), *cache)
    assert_cache(cache, want)


def inputs(tokens, heads, width, dtype, seed, device, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = scale * torch.randn(tokens, 2 * heads, width, generator=g)
    x[:, :, ::3] *= 0.02
    x = x.to(dtype).to(device)
    return x[:, :heads], x[:, heads:]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,page", [(8, 16), (32, 32), (40, 64), (64, 16), (96, 64),
                                        (128, 64), (136, 128), (256, 256)])
def test_write(device, dtype, width, page):
    """Prompts of several lengths, then single tokens that go on in their
    pages, larger and smaller than what the pages hold."""

    print(f"write width {width} page {page} {dtype}", flush=True)
    heads, lengths = 2, [3 * page + 5, 1, page, page - 1, 7]
    cache = empty_cache(16, heads, width, page, device)
    want = host(cache)
    tables, free = pool([0] * 5, page, 5, 16, 4)
    tables, held, top, _, _, slots, _ = ref.extend([0] * 5, lengths, tables, free, 16, page,
                                                   sum(lengths))
    write_both(cache, want, *inputs(sum(lengths), heads, width, dtype, 5, device), slots)
    for step, scale in enumerate((1.0, 9.0, 0.1, 300.0, 1e-3)):
        added = [1, 2, 1, 3, 0] if step % 2 else [1, 1, 1, 1, 1]
        tables, held, top, _, _, slots, short = ref.extend(held, added, tables, free, top, page,
                                                           sum(added) + 2)
        assert not short
        write_both(cache, want, *inputs(sum(added) + 2, heads, width, dtype, 6 + step, device,
                                        scale), slots)


@pytest.mark.parametrize("tokens", [1023, 1024, 1025, 1100])
def test_write_of_many_tokens(device, tokens):
    """Around the size from which a workgroup takes several tokens' runs."""

    cache = empty_cache(40, 1, 32, 32, device)
    want = host(cache)
    lengths = [tokens - 60, 0, 11, 49]
    tables, free = pool([0] * 4, 32, 40, 40, 8)
    _, _, _, _, _, slots, short = ref.extend([0] * 4, lengths, tables, free, 40, 32, tokens)
    assert not short
    write_both(cache, want, *inputs(tokens, 1, 32, torch.bfloat16, 9, device), slots)


@pytest.mark.parametrize("dtype", TYPES)
def test_write_extremes(device, dtype):
    """Zeros, the smallest and largest numbers, infinities and NaN, ties."""

    cache = empty_cache(8, 1, 32, 16, device)
    want = host(cache)
    info = torch.finfo(dtype)
    x = torch.zeros(7, 1, 32, dtype=dtype)
    x[1, 0, 0] = info.max
    x[2, 0, 0] = info.smallest_normal
    x[3, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), 2.5])
    x[4, 0, :2] = torch.tensor([448.0, 1.0])
    x[5, 0, :2] = torch.tensor([449.0 if dtype != torch.bfloat16 else 450.0, -0.0])
    # between two codes of a page whose scale is 1
    x[6, 0] = torch.tensor([256.0] + [(8 + 0.5 + i) * 2.0 for i in range(8)]
                           + [(0.5 + i) * 2.0 ** -9 for i in range(10)] + [17.0] * 13).to(dtype)
    x = x.to(device)
    write_both(cache, want, x, -x, np.arange(7) * 16)       # each token opens a page
    small = torch.full((1, 1, 32), float(info.smallest_normal), dtype=dtype, device=device)
    write_both(cache, want, small, small, np.array([7 * 16]))
    write_both(cache, want, x[1:2], x[1:2], np.array([7 * 16 + 1]))    # everything before shrinks


def test_write_leaves_slots_of_minus_one_and_outside(device):
    cache = empty_cache(4, 2, 64, 16, device)
    before = host(cache)
    key, value = inputs(3, 2, 64, torch.float32, 10, device)
    cow.write_kv_cache(key, value, ints([-1, 64, 1 << 30], device), *cache)
    assert_cache(cache, before)
    cow.write_kv_cache(key[:0], value[:0], ints([], device), *cache)
    assert_cache(cache, before)


def test_write_of_strided_rows(device):
    key, value = inputs(40, 2, 40, torch.bfloat16, 11, device)
    slots = np.arange(40) + 16
    plain, other = empty_cache(4, 2, 40, 16, device), empty_cache(4, 2, 40, 16, device)
    cow.write_kv_cache(key.contiguous(), value.contiguous(), ints(slots, device), *plain)
    room = torch.empty(40, 2, 41, device=device, dtype=torch.bfloat16)
    room[..., 1:] = value
    cow.write_kv_cache(key.transpose(0, 1).contiguous().transpose(0, 1), room[..., 1:],
                       ints(slots, device), *other)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8))
               for a, b in zip(plain, other))


# --------------------------------------------------------------- attention


def filled(lengths, heads, width, page, device, seed, spare=2):
    """A cache of random codes (none NaN) under scales of their own, whose
    unused places hold NaN codes, and its tables."""

    rng = np.random.default_rng(seed)
    columns = max([-(-n // page) for n in lengths] + [1])
    tables, _ = pool(lengths, page, columns, spare, seed)
    pages = sum(-(-n // page) for n in lengths) + spare
    padded = cow.cache_width(width)
    keys = np.full((pages, heads, page, padded), 127, dtype=np.uint8)
    values = np.full((pages, heads, padded, page), 255, dtype=np.uint8)

    def codes(*shape):
        # about normally distributed under a scale of 2^-5
        return ref.encode(np.clip(rng.standard_normal(shape) * 32, -448, 448))

    for b, length in enumerate(lengths):
        for column in range(-(-length // page)):
            n = min(page, length - column * page)
            into = tables[b, column]
            keys[into, :, :n] = 0
            values[into, :, :, :n] = 0
            keys[into, :, :n, :width] = codes(heads, n, width)
            values[into, :, :width, :n] = codes(heads, width, n)
    ks = 2.0 ** rng.integers(-7, -3, (pages, heads))
    vs = 2.0 ** rng.integers(-7, -3, (pages, heads))
    cache = [torch.from_numpy(keys).to(device).view(torch.float8_e4m3fn),
             torch.from_numpy(ks).float().to(device),
             torch.from_numpy(values).to(device).view(torch.float8_e4m3fn),
             torch.from_numpy(vs).float().to(device)]
    numbers = (ref.CODES[keys] * ks[:, :, None, None], ref.CODES[values] * vs[:, :, None, None])
    return cache, numbers, tables


def check_cached(query, cache, numbers, tables, lengths, device, **kw):
    got = cow.cached_attention(query, *cache, ints(tables, device), ints(lengths, device), **kw)
    out, weight, logit = ref.cached(wide(query), *numbers, tables, lengths, kw.get("scale"))
    assert got.shape == query.shape and got.dtype == query.dtype and got.is_contiguous()
    assert_within(got, out, weight, logit, longest=max([*lengths, 1]), values=numbers[1],
                  parts=PARTS[query.dtype])
    return got


def queries(batch, tokens, heads, width, dtype, seed, device):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(batch, tokens, heads, width, generator=g).to(dtype).to(device)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,page", [(8, 16), (32, 32), (40, 64), (64, 16), (96, 64),
                                        (128, 64), (136, 128), (192, 32), (256, 256)])
def test_cached_widths(device, dtype, width, page):
    print(f"cached width {width} page {page} {dtype}", flush=True)
    lengths = [1, 0, page, page + 1, 3 * page - 1, 70, 64, 129]
    cache, numbers, tables = filled(lengths, 2, width, page, device, width)
    check_cached(queries(8, 1, 4, width, dtype, 1, device), cache, numbers, tables, lengths,
                 device)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 9, 20])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 2), (6, 2), (17, 1)])
def test_cached_tokens_and_groups(device, dtype, tokens, heads, kv_heads):
    """Several query tokens, each seeing one more than the one before; requests
    shorter than their query rows leave rows that see nothing."""

    print(f"cached tokens {tokens} heads {heads}/{kv_heads} {dtype}", flush=True)
    lengths = [0, 1, tokens, 63, 64, 66, 200]
    cache, numbers, tables = filled(lengths, kv_heads, 32, 32, device, tokens)
    got = check_cached(queries(7, tokens, heads, 32, dtype, 2, device), cache, numbers, tables,
                       lengths, device)
    assert not got[0].any() and not got[1, :tokens - 1].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 5])
def test_cached_splits_of_the_long_axis(device, dtype, tokens):
    lengths = [5000, 0, 257, 3]
    cache, numbers, tables = filled(lengths, 1, 64, 64, device, 3)
    q = queries(4, tokens, 3, 64, dtype, 3, device)
    assert cow.attention.cached_workspace_bytes(4, tokens, 3, 1, 64, 5000) > 0
    first = check_cached(q, cache, numbers, tables, lengths, device, longest=5000)
    # bounds that are too small, and larger than the tables
    for longest in (1, 300, 2000, 1 << 29):
        check_cached(q, cache, numbers, tables, lengths, device, longest=longest)
    again = cow.cached_attention(q, *cache, ints(tables, device), ints(lengths, device),
                                 longest=5000)
    assert torch.equal(first, again)


@pytest.mark.parametrize("dtype", TYPES)
def test_cached_not_finite(device, dtype):
    """A NaN code reaches the rows that see it, in its column alone where it
    is a value; a NaN key makes a row that sees it NaN."""

    lengths, tokens = [130, 90], 6
    cache, (keys, values), tables = filled(lengths, 1, 64, 64, device, 4)
    codes = cache[2].view(torch.uint8)
    for b, position, column in ((0, 127, 5), (0, 129, 0), (0, 20, 7), (1, 86, 9)):
        into = tables[b, position // 64]
        codes[into, 0, column, position % 64] = 0x7f
        values[into, 0, column, position % 64] = np.nan
    into = tables[1, 88 // 64]
    cache[0].view(torch.uint8)[into, 0, 88 % 64, 3] = 0xff
    keys[into, 0, 88 % 64, 3] = np.nan
    got = check_cached(queries(2, tokens, 2, 64, dtype, 4, device), cache, (keys, values),
                       tables, lengths, device)
    assert torch.isnan(got[0, 2, :, 5]).sum() == 0 and torch.isnan(got[0, 3:, :, 5]).all()
    assert torch.isnan(got[0, :5, :, 0]).sum() == 0 and torch.isnan(got[0, 5, :, 0]).all()
    assert torch.isnan(got[0, :, :, 7]).all()
    assert torch.isfinite(got[1, :2]).all() and torch.isnan(got[1, 4:]).all()


def test_cached_pages_that_do_not_exist(device):
    """Table entries outside the pool, and columns that a length runs past,
    are not read; the rows that need them are the caller's error."""

    lengths = [200, 64, 64]
    cache, numbers, tables = filled(lengths, 1, 32, 64, device, 5)
    q = queries(3, 1, 1, 32, torch.float32, 5, device)
    want = cow.cached_attention(q, *cache, ints(tables, device), ints(lengths, device))
    bad = tables.copy()
    bad[1, 0], bad[2, 0] = -1, 1 << 20
    got = cow.cached_attention(q, *cache, ints(bad, device), ints([200, 64, 64], device))
    assert torch.equal(got[0], want[0])
    got = cow.cached_attention(q, *cache, ints(tables, device), ints([1 << 30, 64, -5], device))
    assert torch.equal(got[1], want[1]) and not got[2].any()


def test_cached_strides_and_scale(device):
    lengths = [100, 37]
    cache, numbers, tables = filled(lengths, 2, 40, 32, device, 6)
    fused = queries(2, 3, 8, 40, torch.bfloat16, 6, device)
    q = fused[:, :, 2:6]
    want = check_cached(q, cache, numbers, tables, lengths, device, scale=0.4)
    turned = q.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    room = torch.empty(2, 3, 4, 41, device=device, dtype=torch.bfloat16)
    room[..., 1:] = q
    for other in (q.contiguous(), turned, room[..., 1:]):
        got = cow.cached_attention(other, *cache, ints(tables, device), ints(lengths, device),
                                   scale=0.4)
        assert torch.equal(got, want)


def test_cached_on_another_stream(device):
    lengths = [4000, 37]
    cache, numbers, tables = filled(lengths, 1, 64, 64, device, 7)
    q = queries(2, 1, 4, 64, torch.float16, 7, device)
    want = cow.cached_attention(q, *cache, ints(tables, device), ints(lengths, device))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cow.cached_attention(q, *cache, ints(tables, device), ints(lengths, device))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_cached_offsets_past_32_bits(device):
    """A pool of more than 2^32 bytes of keys: the last pages are read and
    written at their own addresses."""

    heads, page, width = 8, 64, 128
    pages = (1 << 32) // (heads * page * width) + 9
    keys = torch.zeros(pages, heads, page, width, dtype=torch.uint8, device=device)
    values = torch.zeros(pages, heads, width, page, dtype=torch.uint8, device=device)
    cache = [keys.view(torch.float8_e4m3fn), torch.ones(pages, heads, device=device),
             values.view(torch.float8_e4m3fn), torch.ones(pages, heads, device=device)]
    small = empty_cache(3, heads, width, page, device)
    key, value = inputs(150, heads, width, torch.bfloat16, 12, device)
    tables = np.array([[pages - 1, pages - 3, pages - 2]])
    t = np.arange(150)
    cow.write_kv_cache(key, value, ints(tables[0, t // page] * page + t % page, device), *cache)
    cow.write_kv_cache(key, value, ints(t, device), *small)
    assert not keys[:8].any() and not values[:8].any()
    q = queries(1, 1, 16, width, torch.bfloat16, 13, device)
    got = cow.cached_attention(q, *cache, ints(tables, device), ints([150], device))
    want = cow.cached_attention(q, *small, ints([[0, 1, 2]], device), ints([150], device))
    assert torch.equal(got, want)


@pytest.mark.parametrize("batch", [33, 64, 65])
def test_cached_requests_longest_first(device, batch):
    """More workgroups than run at once, where up to 64 requests are taken by
    their length: every request is taken once, equal and empty ones too."""

    rng = np.random.default_rng(batch)
    lengths = [int(n) for n in rng.integers(0, 90, batch)]
    lengths[3:9] = [17] * 6
    lengths[10] = lengths[batch - 1] = 0
    cache, numbers, tables = filled(lengths, 8, 32, 16, device, batch)
    got = check_cached(queries(batch, 1, 8, 32, torch.float32, 1, device), cache, numbers, tables,
                       lengths, device)
    assert not got[10].any()
