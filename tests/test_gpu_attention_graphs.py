"""The attention operators in a captured graph: a token's tables, write and
attention, and a prompt, replayed on new inputs between eager work."""

from __future__ import annotations

import pytest
import torch

import copy_on_write_sdm_amd as cow
from attention_cases import packed
from test_gpu_kv_cache import filled, ints, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("longest", [300, 4000])
def test_a_token_replayed(device, longest):
    """In one launch, and with the long axis split."""

    lengths, page = [longest - 10, 63, 5], 64
    cache, _, tables = filled(lengths, 2, 64, page, device, 51, spare=8)
    used = set(tables[tables >= 0].tolist())
    free = [p for p in range(len(cache[1])) if p not in used]
    tables = ints(tables, device)
    stack = ints(free, device)
    held, count = ints(lengths, device), ints([len(free)], device)
    added = ints([1, 1, 1], device)
    q = queries(3, 1, 4, 64, torch.bfloat16, 52, device)
    k, v = (queries(3, 1, 2, 64, torch.bfloat16, s, device)[:, 0] for s in (53, 54))

    def token(state):
        tables, held, count, cache, q, k, v = state
        step = cow.extend_page_tables(held, added, tables, stack, count, page_tokens=page,
                                      tokens=3)
        cow.write_kv_cache(k, v, step.slots, *cache)
        out = cow.cached_attention(q, *cache, tables, step.lengths, longest=longest)
        held.copy_(step.lengths)
        count.copy_(step.free_count)
        return out

    def copies():
        return [tables.clone(), held.clone(), count.clone(),
                [t.view(torch.uint8).clone().view(t.dtype) for t in cache], q.clone(), k.clone(),
                v.clone()]

    eager, static = copies(), copies()
    token(copies())                     # whatever a first call sets up
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = token(static)
    for n in range(4):
        print(f"replay {n} longest {longest}", flush=True)
        for state in (eager, static):
            for i, t in enumerate(state[4:]):
                t.copy_(queries(*q.shape, torch.bfloat16, 60 + 3 * n + i, device) if i == 0 else
                        queries(3, 1, 2, 64, torch.bfloat16, 60 + 3 * n + i, device)[:, 0])
        want = token(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip(eager[:3], static[:3]))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8))
                   for a, b in zip(eager[3], static[3]))
    assert static[1].tolist() == [n + 4 for n in lengths]


@pytest.mark.parametrize("dtype,width,lengths", [
    (torch.bfloat16, 128, [70, 0, 300]), (torch.float32, 32, [512, 9]),
    (torch.float16, 64, [900, 20])])
def test_a_prompt_replayed(device, dtype, width, lengths):
    q, k, v, offsets = packed(lengths, 4, 2, width, dtype, 55, device)
    cow.prompt_attention(q, k, v, offsets, longest=max(lengths))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cow.prompt_attention(q, k, v, offsets, longest=max(lengths))
    for n in range(3):
        print(f"replay {n} {dtype}", flush=True)
        for t, other in zip((q, k, v), packed(lengths, 4, 2, width, dtype, 56 + n, device)):
            t.copy_(other)
        want = cow.prompt_attention(q, k, v, offsets, longest=max(lengths))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
