"""PagedKVCache's forks, releases, trims and growth, and a stack that runs on
``AttentionProjections``, ``ResidualMLP`` and rotated heads through them."""

from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

import copy_on_write_sdm_amd as cow
from attention_cases import wide
from controller_cases import make_layer
from oracle import attention as attention_ref
from oracle import pages as pages_ref
from oracle import projections as ref

pytestmark = pytest.mark.gpu

PAGE = 16


def assert_whole(cache):
    """The host's counts are the device's, and every page is free or held."""

    assert cache.free == cache.free_count.item()
    assert cache.lengths.tolist() == cache.request_lengths()
    tables = cache.page_tables.cpu().numpy()
    pages_ref.check(cache.request_lengths(), tables, cache.page_shares.tolist(),
                    cache.free_pages.tolist(), cache.free, cache.page_tokens)


def contents(cache, request):
    """The codes' values of a request's tokens in all layers."""

    n = cache.request_lengths()[request]
    at = torch.arange(n, device=cache.device)
    pages = cache.page_tables[request][at // PAGE].long()
    k = cache.key_pages.view(torch.uint8)[:, pages, :, at % PAGE].view(cache.key_pages.dtype)
    v = cache.value_pages.view(torch.uint8)[:, pages, :, :, at % PAGE].view(cache.key_pages.dtype)
    scales = cache.key_scales[:, pages], cache.value_scales[:, pages]
    # an index between slices and after them: [tokens, layers, ...] of both
    return [x.float().flatten(1) for x in (k, v)] + [s.transpose(0, 1).flatten(1)
                                                     for s in scales]


def same(a, b):
    return all(torch.equal(x[:len(y)], y[:len(x)]) for x, y in zip(a, b))


def fill(cache, added, g):
    step = cache.extend(added)
    n = step.slots.numel()
    for layer in range(cache.layers):
        k, v = (torch.randn(n, cache.heads, cache.head_width, generator=g).to(cache.device)
                for _ in range(2))
        cache.write(layer, k, v, step.slots)


def test_a_cache_through_forks_and_trims(device):
    g = torch.Generator().manual_seed(4)
    cache = cow.PagedKVCache(3, 2, 24, capacity=200, pages=60, page_tokens=PAGE, device=device)
    cache.admit(3)
    fill(cache, [37, 48, 0], g)
    parents = [contents(cache, r) for r in range(3)]
    assert cache.fork([0, 1, 0, 2]) == [3, 4, 5, 6]
    assert cache.request_lengths() == [37, 48, 0, 37, 48, 37, 0]
    assert cache.free == 60 - 6 - 2                    # two children end inside a page
    assert_whole(cache)
    for child, parent in zip((3, 4, 5, 6), (0, 1, 0, 2)):
        assert same(contents(cache, child), parents[parent])
    assert cache.fork([1, 3], [20, 16]) == [7, 8]      # of a part, and of a child
    assert cache.request_lengths()[7:] == [20, 16]
    assert_whole(cache)
    # each goes its own way from here
    before = [contents(cache, r) for r in range(9)]
    fill(cache, [5, 1, 17, 2, 30, 0, 3, 16, 1], g)
    assert_whole(cache)
    for r, old in enumerate(before):
        now = contents(cache, r)
        n = cache.request_lengths()[r]
        # codes of a page that went on can be taken to a larger scale
        kept = len(old[0]) // PAGE * PAGE
        assert len(now[0]) == n and same([x[:kept] for x in now], [x[:kept] for x in old])
    freed = cache.release([0, 4])
    assert freed == 1 + 2                              # what 0 and 4 alone held
    assert (cache.page_tables[[0, 4]] == -1).all()
    assert_whole(cache)
    assert cache.compact() == [1, 2, 3, 5, 6, 7, 8]
    kept = [contents(cache, r) for r in range(7)]
    used = 60 - cache.free
    assert cache.trim_pages(headroom_pages=3) == 60 - used - 3
    assert cache.key_pages.shape[1] == used + 3 == cache.free_pages.numel()
    assert_whole(cache)
    assert all(same(contents(cache, r), kept[r]) for r in range(7))
    assert cache.trim_pages(headroom_pages=4) == 0
    cache.grow_pages(10)
    assert cache.free == 13 and cache.value_pages.shape[1] == used + 13
    assert_whole(cache)
    fill(cache, [20] * 7, g)
    assert_whole(cache)
    assert all(same([x[:len(y) // PAGE * PAGE] for x, y in zip(contents(cache, r), kept[r])],
                    [y[:len(y) // PAGE * PAGE] for y in kept[r]]) for r in range(7))
    held = used + 13 - cache.free
    assert cache.release(list(range(7))) == held
    assert cache.free == used + 13 and not cache.page_shares.any()
    assert_whole(cache)
    assert cache.compact() == [] and cache.trim_pages() == used + 12
    cache.admit(1)
    fill(cache, 16, g)
    assert_whole(cache)


def test_a_step_is_taken_back_after_a_fork(device):
    cache = cow.PagedKVCache(1, 1, 8, capacity=64, pages=12, page_tokens=PAGE, device=device)
    cache.admit(1)
    cache.extend(40)
    cache.fork([0])
    with pytest.raises(ValueError, match="no KV cache step"):
        cache.take_back()                              # the fork has followed it
    state = cache.page_tables.clone(), cache.lengths.clone(), cache.free
    cache.extend([9, 1])
    cache.take_back()
    assert torch.equal(cache.lengths, state[1]) and cache.free == state[2]
    assert_whole(cache)
    cache.release([0])
    assert cache.compact() == [1]
    assert_whole(cache)


def test_refusals(device):
    cache = cow.PagedKVCache(1, 2, 32, capacity=40, pages=4, page_tokens=PAGE, device=device)
    cache.admit(2)
    cache.extend([40, 0])
    kept = cache.page_tables.clone(), cache.lengths.clone(), cache.free
    for bad in ([2], [-1]):
        with pytest.raises(ValueError, match="invalid or inactive"):
            cache.fork(bad)
    for tokens in ([1], [1, 2, 3], [41, 0], [0, -1], 1):
        with pytest.raises(ValueError, match="one count per request"):
            cache.fork([0, 1], tokens)
    with pytest.raises(ValueError, match="exhausted: 2 needed, 1 free"):
        cache.fork([0, 0])
    with pytest.raises(ValueError, match="cannot be negative"):
        cache.trim_pages(headroom_pages=-1)
    with pytest.raises(ValueError, match="cannot be negative"):
        cache.grow_pages(-1)
    assert torch.equal(cache.page_tables, kept[0]) and torch.equal(cache.lengths, kept[1])
    assert cache.free == kept[2] and cache.requests == 2
    assert cache.fork([]) == [] and cache.fork([0, 0], 32) == [2, 3]
    cache.release([1])
    with pytest.raises(ValueError, match="invalid or inactive"):
        cache.fork([1])
    with pytest.raises(ValueError, match="multiple of the key heads"):
        cow.AttentionProjections({}, heads=3, kv_heads=2, head_width=8)
    good = torch.zeros(32, 16), torch.zeros(16, 16)
    for wrong in (cow.AttentionLayer(good[0][:31], good[1]),
                  cow.AttentionLayer(good[0], good[1][:, :8])):
        with pytest.raises(ValueError, match="attention layer 1's"):
            cow.AttentionProjections({1: wrong}, heads=2, kv_heads=1, head_width=8)
    with pytest.raises(ValueError, match="one pair per attention layer"):
        cow.PagedAttention(cache, (1,), None, None, head_norms=[])


LAYOUT, WIDTH, SLOTS, MEMORY_HEADS = "BAAB", 64, 64, 2
HEADS, KV_HEADS, HEAD_WIDTH = 4, 2, 16


def test_a_stack_with_forked_requests(device):
    """Prefill, decode, fork every request once (in the SDM state as a copy
    that is admitted), decode, release, trim, decode.  Forked requests that
    get the same tokens answer the same, bit for bit, and every attention
    block is the definition's on the cache's own numbers."""

    g = torch.Generator().manual_seed(31)
    rand = lambda *s, by=1.0: (by * torch.randn(*s, generator=g)).to(device)     # noqa: E731
    layers = [make_layer(WIDTH, slots=SLOTS, reads=8, writes=4, heads=MEMORY_HEADS, seed=s,
                         dtype=torch.float32) for s in (8, 9)]
    sdm = [(cow.SDMController.from_module(layer, device=device),
            rand(MEMORY_HEADS, SLOTS, WIDTH // MEMORY_HEADS, by=0.5)) for layer in layers]
    norm = torch.nn.LayerNorm(WIDTH, device=device)
    rows = (HEADS + 2 * KV_HEADS) * HEAD_WIDTH
    mlps = [cow.ResidualMLP(rand(4 * WIDTH, WIDTH, by=0.1), rand(WIDTH, 4 * WIDTH, by=0.05),
                            rand(4 * WIDTH), rand(WIDTH), norm=norm) for _ in range(2)]
    weights = {at: cow.AttentionLayer(rand(rows, WIDTH, by=WIDTH ** -0.5),
                                      rand(WIDTH, HEADS * HEAD_WIDTH, by=0.1), rand(rows, by=0.1),
                                      None, norm, mlp) for at, mlp in zip((1, 2), mlps)}
    parts = cow.AttentionProjections(weights, heads=HEADS, kv_heads=KV_HEADS,
                                     head_width=HEAD_WIDTH)
    rotation = cow.HeadRotation(HEAD_WIDTH, device=device)
    norms = [(1 + rand(HEAD_WIDTH, by=0.1), 1 + rand(HEAD_WIDTH, by=0.1)) for _ in range(2)]
    cache = cow.PagedKVCache(2, KV_HEADS, HEAD_WIDTH, capacity=80, pages=40, page_tokens=PAGE,
                             device=device)
    checked = []

    def finish(layer, tokens, mixed):
        """The block's output, once more in 64 bits."""

        out = parts.finish(layer, tokens, mixed)
        w = weights[layer]
        with torch.no_grad():
            x = norm(tokens)
            want = wide(tokens) + wide(mixed).reshape(len(tokens), -1) @ wide(w.output_weight).T
            got = norm(torch.from_numpy(want).float().to(device))
        inner, _, _ = ref.linear(wide(got), wide(w.tail.up_weight), wide(w.tail.up_bias), "gelu")
        end, _, _ = ref.linear(inner, wide(w.tail.down_weight), wide(w.tail.down_bias), None, want)
        # float32 sums of at most 256 terms, magnitudes of a few units
        np.testing.assert_allclose(wide(out), end, rtol=0, atol=256 * 2.0 ** -24 * 64)
        if block._prompt:
            return out
        # the newest token's attention over the cache, from the block's input on
        index = layer - 1
        qkv, _, _ = ref.linear(wide(x), wide(w.input_weight), wide(w.input_bias))
        q = qkv.reshape(len(tokens), -1, HEAD_WIDTH)[:, :HEADS]
        positions = block._step.positions.tolist()
        q, _ = ref.rotate(q, positions, rotation.frequencies, weight=wide(norms[index][0]))
        keys = wide(cache.key_pages[index].float()) * wide(cache.key_scales[index])[..., None,
                                                                                    None]
        values = wide(cache.value_pages[index].float()) * wide(
            cache.value_scales[index])[..., None, None]
        mix, _, _ = attention_ref.cached(q[:, None], keys, values,
                                         cache.page_tables.cpu().numpy(),
                                         cache.lengths.tolist())
        # logits are sums of 16 products of magnitudes within 4 by 4
        np.testing.assert_allclose(wide(mixed), mix[:, 0], rtol=0, atol=2.0 ** -14)
        checked.append(layer)
        return out

    block = cow.PagedAttention(cache, (1, 2), parts.project, finish, rotation=rotation,
                               head_norms=norms)
    tail = lambda layer, tokens: mlps[layer // 2](tokens)                        # noqa: E731

    def decode(state, x):
        return cow.decode_faithful_sdm_stack(LAYOUT, sdm, x, state, attention_decode=block.decode,
                                             sdm_tail=tail)

    batch = 3
    _, state = cow.prefill_faithful_sdm_stack(
        LAYOUT, sdm, rand(batch, 21, WIDTH), attention_block=block.prefill, capacity=80,
        sdm_growth_quantum_rows=64, sdm_tail=tail)
    decode(state, rand(batch, 1, WIDTH))
    assert cache.fork(range(batch)) == [3, 4, 5]
    state.admit(copy.deepcopy(state))
    assert state.batch == cache.requests == 6
    for n in range(14):                                # across a page's end
        print(f"forked decode {n}", flush=True)
        x = rand(batch, 1, WIDTH)
        if n < 5:
            out = decode(state, torch.cat((x, x)))
            assert torch.equal(out[:batch], out[batch:])
        else:
            out = decode(state, torch.cat((x, rand(batch, 1, WIDTH))))
        assert torch.isfinite(out).all()
    assert_whole(cache)
    state.release([0, 4])
    cache.release([0, 4])
    state.compact()
    assert cache.compact() == [1, 2, 3, 5]
    assert cache.trim_pages(headroom_pages=4) > 0
    assert_whole(cache)
    decode(state, rand(4, 1, WIDTH))
    assert cache.request_lengths() == [37] * 4
    assert len(checked) == 2 * (1 + 14 + 1)
