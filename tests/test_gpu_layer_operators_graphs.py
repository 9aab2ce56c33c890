"""The operators around the attention in captured graphs, replayed on new inputs
between eager work, on streams of their own and two at a time."""

from __future__ import annotations

import pytest
import torch

import copy_on_write_sdm_amd as cow
from test_gpu_pages import cache, ints, pool

pytestmark = pytest.mark.gpu

# (rows, inner, outer, type): few rows, a split axis, small, odd, middle and the largest tiles
SIZES = [(5, 264, 96, torch.float32), (70, 4096, 130, torch.bfloat16),
         (70, 4096, 130, torch.float32), (90, 72, 64, torch.float16), (33, 37, 65, torch.bfloat16),
         (700, 200, 900, torch.float32), (4100, 136, 4100, torch.bfloat16),
         (2910, 7848, 1420, torch.float16)]


def linear_inputs(size, seed, device):
    rows, inner, outer, dtype = size
    g = torch.Generator(device=device).manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g, device=device).to(dtype)     # noqa: E731
    return make(rows, inner), make(outer, inner), make(outer), make(rows, outer)


def linear(x, weight, bias, residual):
    return [cow.linear(x, weight, bias, activation="gelu", residual=residual)]


def head_inputs(seed, device):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(300, 12, 64, generator=g, device=device).to(torch.bfloat16)
    at = torch.randint(0, 1 << 20, (300,), generator=g, device=device, dtype=torch.int32)
    weight = torch.randn(64, generator=g, device=device).to(torch.bfloat16)
    return x, at, weight


def heads_call(rotation):
    def call(x, at, weight):
        return list(cow.rotate_heads(x[:, :8], x[:, 8:10], at, rotation, query_norm=weight,
                                     key_norm=weight))
    return call


def page_inputs(seed, device, many):
    """A pool in use, who is forked and who is released."""

    page = 16
    lengths = [(seed * 31 + 37 * i) % (2000 if many else 100) for i in range(200 if many else 9)]
    tables, shares, stack, count = pool(lengths, page, 4000 if many else 40, seed,
                                        columns=126 if many else 8)
    pages = 30000 if many else 128
    shares += [0] * (pages - len(shares))
    stack += [-1] * (pages - len(stack))
    g = torch.Generator().manual_seed(seed)
    n = 150 if many else 6
    parents = torch.randint(0, len(lengths), (n,), generator=g).tolist()
    named = torch.randperm(len(lengths), generator=g)[:n].tolist()
    return [ints(lengths, device), ints(tables, device), ints(shares, device),
            ints(stack, device), ints([count], device), ints(parents, device),
            ints([lengths[p] for p in parents], device), ints(named, device),
            *cache(2, 128, 2, page, 32, device, seed)]


def page_call(lengths, tables, shares, stack, count, parents, tokens, named, *tensors):
    """Requests forked, some of those before released, the rest moved together."""

    fork = cow.fork_page_tables(lengths, tables, shares, stack, count, parents, tokens,
                                page_tokens=16)
    cow.copy_pages(*tensors, fork.sources, fork.targets)
    both = torch.cat((lengths, fork.lengths)), torch.cat((tables, fork.page_tables))
    left = cow.release_page_tables(*both, fork.page_shares, stack, fork.free_count, named,
                                   page_tokens=16)
    moves = cow.compact_page_tables(left.lengths, both[1], left.page_shares, page_tokens=16)
    cow.copy_pages(*tensors, moves.sources, moves.targets)
    return [*fork, *left, *moves, stack, *tensors]


def calls(device):
    rotation = cow.HeadRotation(64, device=device)
    return ([(f"linear {s}", linear, lambda seed, s=s: linear_inputs(s, seed, device))
             for s in SIZES]
            + [("heads", heads_call(rotation), lambda seed: head_inputs(seed, device))]
            + [(f"pages {many}", page_call, lambda seed, m=many: page_inputs(seed, device, m))
               for many in (False, True)])


def bits(t):
    return t.view(torch.uint8) if t.dtype is torch.float8_e4m3fn else t


def same(a, b):
    return len(a) == len(b) and all(torch.equal(bits(x), bits(y)) for x, y in zip(a, b))


def test_replays(device):
    for name, call, make in calls(device):
        static = [t.clone() for t in make(1)]
        call(*[t.clone() for t in static])             # whatever a first call sets up
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = call(*static)
        for n in range(3):
            print(f"{name} replay {n}", flush=True)
            inputs = make(2 + n)
            for t, new in zip(static, inputs):
                bits(t).copy_(bits(new))
            want = call(*inputs)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert same(out, want), (name, n)
        del graph


def test_two_graphs_share_nothing(device):
    """Captured in one memory pool, replayed in turn."""

    size = SIZES[1]
    graphs, outs, wants, pool_id = [], [], [], None
    for seed in (1, 2):
        inputs = linear_inputs(size, seed, device)
        wants.append(linear(*inputs)[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool_id):
            outs.append((inputs, linear(*inputs)[0]))
        pool_id = pool_id or graph.pool()
        graphs.append(graph)
    for n in (0, 1, 1, 0):
        graphs[n].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[n][1], wants[n])


def test_two_streams_at_once(device):
    streams = [torch.cuda.Stream() for _ in range(2)]
    for name, call, make in calls(device):
        print(f"{name} on two streams", flush=True)
        inputs = [make(11), make(12)]
        wants = [call(*[t.clone() for t in i]) for i in inputs]
        copies = [[[t.clone() for t in i] for _ in range(4)] for i in inputs]
        torch.cuda.synchronize()
        got = [[], []]
        for n in range(4):
            for s, stream in enumerate(streams):
                with torch.cuda.stream(stream):
                    got[s].append(call(*copies[s][n]))
        torch.cuda.synchronize()
        for s in range(2):
            assert all(same(g, wants[s]) for g in got[s]), (name, s)
