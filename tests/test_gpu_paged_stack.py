"""A "BAAB" stack whose attention layers run on the paged 8-bit cache
(PagedAttention), through a lifecycle: prefill 3 requests, decode past a page,
release 1, compact, admit 2 requests with a longer prefix, decode on.

Every attention product is checked against the 64-bit definition on the
cache's own numbers, every layer's cache against the oracle's write of the same
keys and values bit for bit, and the tables and free pages against the oracle's
page tables; the SDM layers and the lifecycle are the state's own."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import copy_on_write_sdm_amd as cow
from attention_cases import assert_within, wide
from controller_cases import make_layer
from oracle import attention as ref

pytestmark = pytest.mark.gpu

LAYOUT = "BAAB"
WIDTH, SLOTS, MEMORY_HEADS, READS, WRITES = 64, 64, 2, 8, 4
HEADS, KV_HEADS, HEAD_WIDTH, PAGE, CAPACITY, PAGES = 4, 2, 16, 16, 80, 24
PARTS = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}


class Model:
    """The model's parts of the attention layers, and the checks around them."""

    def __init__(self, dtype, device):
        g = torch.Generator().manual_seed(3)
        n = (HEADS + 2 * KV_HEADS) * HEAD_WIDTH
        self.wqkv = [(torch.randn(WIDTH, n, generator=g) * WIDTH ** -0.5).to(device)
                     for _ in range(2)]
        self.wo = [(torch.randn(HEADS * HEAD_WIDTH, WIDTH, generator=g) * 0.1).to(device)
                   for _ in range(2)]
        self.dtype = dtype
        self.cache = cow.PagedKVCache(2, KV_HEADS, HEAD_WIDTH, capacity=CAPACITY, pages=PAGES,
                                      page_tokens=PAGE, device=device)
        self.block = cow.PagedAttention(self.cache, (1, 2), self.project, self.finish)
        self.rows = {}               # what project() last gave for a layer
        self.host = [self.host_copy(i) for i in range(2)]
        self.checked = 0

    def host_copy(self, layer):
        c = self.cache
        return [c.key_pages[layer].view(torch.uint8).cpu().numpy().copy(),
                c.key_scales[layer].double().cpu().numpy(),
                c.value_pages[layer].view(torch.uint8).cpu().numpy().swapaxes(2, 3).copy(),
                c.value_scales[layer].double().cpu().numpy()]

    def project(self, layer, tokens, positions):
        # something by position, so that a wrong one shows
        x = tokens + 0.1 * torch.sin(positions.float())[:, None]
        x = (x @ self.wqkv[layer - 1]).reshape(-1, HEADS + 2 * KV_HEADS, HEAD_WIDTH)
        x = x.to(self.dtype)
        q, k, v = x[:, :HEADS], x[:, HEADS:HEADS + KV_HEADS], x[:, HEADS + KV_HEADS:]
        self.rows[layer] = (q, k, v, positions)
        return q, k, v

    def finish(self, layer, tokens, mixed):
        self.check(layer, mixed)
        mixed = mixed.float().reshape(-1, HEADS * HEAD_WIDTH)
        return tokens + torch.tanh(mixed @ self.wo[layer - 1])

    def check(self, layer, mixed):
        q, k, v, positions = self.rows[layer]
        step, cache, index = self.block._step, self.cache, layer - 1
        slots = step.slots.cpu().numpy()
        assert not step.overflow.item()
        want = self.host[index]
        ref.write(wide(k), slots, want[0], want[1])
        ref.write(wide(v), slots, want[2], want[3])
        for got, expected in zip(self.host_copy(index), want):
            assert np.array_equal(got, expected)
        tables, lengths = cache.page_tables.cpu().numpy(), cache.lengths.tolist()
        assert lengths == cache.request_lengths()
        keys = ref.CODES[want[0]] * want[1][:, :, None, None]
        values = (ref.CODES[want[2]] * want[3][:, :, None, None]).swapaxes(2, 3)
        if self.prompt:
            out, weight, logit = ref.prompt(wide(q), wide(k), wide(v), step.offsets.tolist())
            assert_within(mixed, out, weight, logit, longest=max(lengths), values=wide(v))
        else:
            assert positions.tolist() == [n - 1 for n in lengths]
            out, weight, logit = ref.cached(wide(q)[:, None], keys, values, tables, lengths)
            assert_within(mixed[:, None], out, weight, logit, longest=max(lengths),
                          values=values, parts=PARTS[self.dtype])
        self.checked += 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_stack_on_a_paged_cache_through_lifecycle(device, dtype):
    g = torch.Generator().manual_seed(29)
    layers = [make_layer(WIDTH, slots=SLOTS, reads=READS, writes=WRITES, heads=MEMORY_HEADS,
                         seed=s, dtype=torch.float32) for s in (8, 9)]
    ctrls = [cow.SDMController.from_module(layer, device=device) for layer in layers]
    m0s = [(torch.randn(MEMORY_HEADS, SLOTS, WIDTH // MEMORY_HEADS, generator=g) * 0.5).to(device)
           for _ in layers]
    sdm = list(zip(ctrls, m0s))
    model = Model(dtype, device)
    cache, block = model.cache, model.block

    def prefill(batch, time):
        print(f"paged stack {dtype} prefill {batch} x {time}", flush=True)
        model.prompt = True
        x = torch.randn(batch, time, WIDTH, generator=g).to(device)
        return cow.prefill_faithful_sdm_stack(
            LAYOUT, sdm, x, attention_block=block.prefill, capacity=CAPACITY,
            sdm_growth_quantum_rows=batch * MEMORY_HEADS * WRITES * 2)[1]

    def decode(state, tokens):
        model.prompt = False
        for _ in range(tokens):
            x = torch.randn(state.batch, 1, WIDTH, generator=g).to(device)
            out = cow.decode_faithful_sdm_stack(LAYOUT, sdm, x, state,
                                                attention_decode=block.decode)
            assert torch.isfinite(out).all()

    def pages():
        return sum(-(-n // PAGE) for n in cache.request_lengths())

    def pages_are_apart():
        tables = cache.page_tables.cpu().numpy()
        mine = [p for row, n in zip(tables, cache.request_lengths())
                for p in row[:-(-n // PAGE)]]
        free = cache.free_pages[:cache.free_count.item()].tolist()
        assert cache.free == len(free) == PAGES - pages()
        assert sorted(mine + free) == list(range(PAGES))

    state = prefill(3, 14)
    assert all(t.numel() == 0 for t in (*state.dense_keys, *state.dense_values))
    assert state.storage_bytes()["dense_kv_allocated"] == 0
    decode(state, 5)                                  # across a page's end
    assert cache.request_lengths() == [19] * 3
    pages_are_apart()
    state.release([1])
    assert cache.release([1]) == 2
    with pytest.raises(ValueError, match="invalid, duplicated, or inactive"):
        cache.release([1])
    with pytest.raises(ValueError, match="removed before further decode"):
        cache.extend(1)
    state.compact()
    assert cache.compact() == [0, 2]
    pages_are_apart()
    state.admit(prefill(2, 33))
    assert cache.request_lengths() == [19, 19, 33, 33]
    decode(state, 4)
    assert cache.request_lengths() == [23, 23, 37, 37] == state.positions.tolist()
    pages_are_apart()
    used = cache.storage_bytes()
    assert used["kv_live"] == used["kv_codes"] // PAGES * pages() + (
        used["kv_scales"] // PAGES * pages())
    assert model.checked == 2 * (1 + 5 + 1 + 4)


def test_refusals(device):
    make = lambda **kw: cow.PagedKVCache(1, 2, 32, **{**dict(      # noqa: E731
        capacity=40, pages=4, page_tokens=16, device=device), **kw})
    with pytest.raises(ValueError, match="must be positive"):
        make(pages=0)
    with pytest.raises(ValueError, match="16, 32, 64, 128 or 256"):
        make(page_tokens=24)
    with pytest.raises(RuntimeError, match="no CPU path"):
        make(device="cpu")
    cache = make()
    assert cache.admit(2) == [0, 1] and cache.extend(16).slots.numel() == 32
    before = cache.page_tables.clone(), cache.lengths.clone(), cache.free
    with pytest.raises(ValueError, match="one count per request"):
        cache.extend([1])
    with pytest.raises(ValueError, match="one count per request"):
        cache.extend([1, -1])
    with pytest.raises(ValueError, match="fixed capacity"):
        cache.extend([25, 0])
    with pytest.raises(ValueError, match="exhausted: 3 needed, 2 free"):
        cache.extend([17, 1])
    for bad in ([2], [-1], [0, 0]):
        with pytest.raises(ValueError, match="invalid, duplicated"):
            cache.release(bad)
    assert torch.equal(cache.page_tables, before[0]) and torch.equal(cache.lengths, before[1])
    assert cache.free == before[2] == 2
    block = cow.PagedAttention(cache, (1,), None, None)
    with pytest.raises(ValueError, match="exhausted: 3 needed, 2 free"):
        block.prefill(1, torch.zeros(1, 40, 8, device=device))
    assert cache.requests == 2 and cache.free == 2
    assert torch.equal(cache.page_tables, before[0]) and torch.equal(cache.lengths, before[1])
    with pytest.raises(ValueError, match="not one of the attention layers"):
        block.prefill(0, torch.zeros(1, 1, 8, device=device))
    with pytest.raises(ValueError, match="do not match the KV cache"):
        block.decode(1, torch.zeros(2, 1, 8, device=device), None, None, 15)
    with pytest.raises(ValueError, match="a layer for every"):
        cow.PagedAttention(cache, (1, 3), None, None)


def test_release_of_many_requests(device):
    """More released requests than a workgroup takes at once, in list order."""

    n = 600
    cache = cow.PagedKVCache(1, 1, 8, capacity=48, pages=3 * n, page_tokens=16, device=device)
    cache.admit(n)
    counts = [(7 * i) % 49 for i in range(n)]
    cache.extend(counts)
    tables = cache.page_tables.cpu().numpy()
    left = cache.free_pages[:cache.free].tolist()
    order = np.random.default_rng(1).permutation(n)[:450].tolist()
    freed = [p for r in order for p in tables[r, :-(-counts[r] // 16)]]
    assert cache.release(order) == len(freed)
    assert cache.free_pages[:cache.free_count.item()].tolist() == left + freed
    assert cache.free == len(left) + len(freed)
    lengths = cache.lengths.tolist()
    assert all(lengths[r] == (0 if r in set(order) else counts[r]) for r in range(n))
    assert (cache.page_tables[order] == -1).all()
    kept = cache.compact()
    assert cache.lengths.tolist() == [counts[r] for r in kept]
