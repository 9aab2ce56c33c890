"""Steps of the paged cache that are refused or fail: the cache stands where the
decode state does, and the step run again gives what it gives undisturbed."""

from __future__ import annotations

import pytest
import torch

import copy_on_write_sdm_amd as cow
from controller_cases import make_layer

pytestmark = pytest.mark.gpu

WIDTH, SLOTS, MEMORY_HEADS, READS, WRITES = 64, 64, 2, 8, 4
HEADS, KV_HEADS, HEAD_WIDTH, PAGE, CAPACITY = 4, 2, 16, 16, 80


class Failure(Exception):
    pass


class Run:
    """A stack with attention layers on a paged cache, whose parts can be told
    to fail once."""

    def __init__(self, layout, device, *, pages=24):
        g = torch.Generator().manual_seed(3)
        self.layout, self.device, self.g = layout, device, g
        self.layers = tuple(i for i, kind in enumerate(layout) if kind == "A")
        n = (HEADS + 2 * KV_HEADS) * HEAD_WIDTH
        self.wqkv = {i: (torch.randn(WIDTH, n, generator=g) * WIDTH ** -0.5).to(device)
                     for i in self.layers}
        self.wo = {i: (torch.randn(HEADS * HEAD_WIDTH, WIDTH, generator=g) * 0.1).to(device)
                   for i in self.layers}
        self.sdm = []
        for i in range(layout.count("B")):
            layer = make_layer(WIDTH, slots=SLOTS, reads=READS, writes=WRITES,
                               heads=MEMORY_HEADS, seed=8 + i, dtype=torch.float32)
            m0 = torch.randn(MEMORY_HEADS, SLOTS, WIDTH // MEMORY_HEADS, generator=g) * 0.5
            self.sdm.append((cow.SDMController.from_module(layer, device=device), m0.to(device)))
        self.cache = cow.PagedKVCache(len(self.layers), KV_HEADS, HEAD_WIDTH, capacity=CAPACITY,
                                      pages=pages, page_tokens=PAGE, device=device)
        self.block = cow.PagedAttention(self.cache, self.layers, self.project, self.finish)
        self.fail = None             # (part, layer)
        self.ran = []

    def part(self, name, layer):
        self.ran.append((name, layer))
        if self.fail == (name, layer):
            self.fail = None
            raise Failure(name)

    def project(self, layer, tokens, positions):
        self.part("project", layer)
        x = tokens + 0.1 * torch.sin(positions.float())[:, None]
        x = (x @ self.wqkv[layer]).reshape(-1, HEADS + 2 * KV_HEADS, HEAD_WIDTH).bfloat16()
        if self.fail == ("type", layer):          # refused by the operators
            self.fail = None
            return x[:, :HEADS], x[:, HEADS:HEADS + KV_HEADS].float(), x[:, HEADS + KV_HEADS:]
        return x[:, :HEADS], x[:, HEADS:HEADS + KV_HEADS], x[:, HEADS + KV_HEADS:]

    def finish(self, layer, tokens, mixed):
        self.part("finish", layer)
        return tokens + torch.tanh(mixed.float().reshape(-1, HEADS * HEAD_WIDTH) @ self.wo[layer])

    def tail(self, layer, tokens):
        self.part("tail", layer)
        return tokens

    def tokens(self, batch, time):
        return torch.randn(batch, time, WIDTH, generator=self.g).to(self.device)

    def prefill(self, x):
        return cow.prefill_faithful_sdm_stack(
            self.layout, self.sdm, x, attention_block=self.block.prefill, capacity=CAPACITY,
            sdm_tail=self.tail,
            sdm_growth_quantum_rows=max(1, len(x)) * MEMORY_HEADS * WRITES * 2)

    def decode(self, x, state):
        return cow.decode_faithful_sdm_stack(self.layout, self.sdm, x, state, sdm_tail=self.tail,
                                             attention_decode=self.block.decode)

    def standing(self):
        """What a step must not leave changed."""

        c = self.cache
        held = [-(-n // PAGE) for n in c.request_lengths()]
        return (c.request_lengths(), c.lengths.tolist(), c.free, c.free_count.item(),
                c.free_pages[:c.free].tolist(), c.requests,
                [row[:n] for row, n in zip(c.page_tables.tolist(), held)])

    def codes(self):
        """Each request's codes and scales up to its length."""

        c, out = self.cache, []
        for row, n in zip(c.page_tables.tolist(), c.request_lengths()):
            for column in range(-(-n // PAGE)):
                p, m = row[column], min(PAGE, n - column * PAGE)
                out += [c.key_pages.view(torch.uint8)[:, p, :, :m],
                        c.value_pages.view(torch.uint8)[:, p, :, :, :m],
                        c.key_scales[:, p], c.value_scales[:, p]]
        return out


FAILURES = [("project", 0), ("type", 0), ("finish", 0), ("project", 1), ("type", 1), ("finish", 1)]


@pytest.mark.parametrize("part,layer", FAILURES)
@pytest.mark.parametrize("ragged", [False, True])
def test_a_token_that_fails_can_be_run_again(device, part, layer, ragged):
    """At tokens that open pages and tokens that go on in them; positions
    shared, and one for each request."""

    print(f"token fails in {part} {layer} ragged {ragged}", flush=True)
    runs = [Run("AAB", device) for _ in range(2)]
    outs = []
    for disturbed, run in enumerate(runs):
        _, state = run.prefill(run.tokens(2, 14))
        if ragged:
            state.admit(run.prefill(run.tokens(2, 31))[1])
            assert state.positions is not None
        out = []
        for step in range(5):
            x = run.tokens(state.batch, 1)
            if disturbed and step in (1, 2, 3):
                before, run.fail = run.standing(), (part, layer)
                with pytest.raises(TypeError if part == "type" else Failure):
                    run.decode(x, state)
                assert run.standing() == before
            out.append(run.decode(x, state))
        assert run.cache.request_lengths() == [19, 19] + [36, 36] * ragged
        outs.append(out)
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert all(torch.equal(a, b) for a, b in zip(*(run.codes() for run in runs)))


@pytest.mark.parametrize("ragged", [False, True])
def test_a_token_that_fails_past_the_attention_layers(device, ragged):
    run = Run("AAB", device)
    _, state = run.prefill(run.tokens(2, 16))
    if ragged:
        state.admit(run.prefill(run.tokens(1, 20))[1])
    before, run.fail = run.standing(), ("tail", 2)
    with pytest.raises(Failure):
        run.decode(run.tokens(state.batch, 1), state)
    assert run.standing() == before
    assert torch.isfinite(run.decode(run.tokens(state.batch, 1), state)).all()
    assert run.cache.request_lengths() == [17, 17] + [21] * ragged


@pytest.mark.parametrize("part,layer", FAILURES + [("tail", 2)])
def test_a_prompt_that_fails_can_be_run_again(device, part, layer):
    print(f"prompt fails in {part} {layer}", flush=True)
    runs = [Run("AAB", device) for _ in range(2)]
    outs = []
    for disturbed, run in enumerate(runs):
        out, state = run.prefill(run.tokens(2, 14))
        run.decode(run.tokens(2, 1), state)
        x = run.tokens(3, 18)
        if disturbed:
            before, run.fail = run.standing(), (part, layer)
            with pytest.raises(TypeError if part == "type" else Failure):
                run.prefill(x)
            assert run.standing() == before
        more, incoming = run.prefill(x)
        state.admit(incoming)
        outs.append([out, more, run.decode(run.tokens(5, 1), state)])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert all(torch.equal(a, b) for a, b in zip(*(run.codes() for run in runs)))


def test_a_step_without_room_is_refused_before_any_layer(device):
    """The SDM layer above the first attention layer has not run either."""

    run = Run("BA", device, pages=2)
    _, state = run.prefill(run.tokens(2, 16))
    before, memory = run.standing(), state.sdm_states[0].materialize_dense()
    run.ran.clear()
    with pytest.raises(ValueError, match="exhausted: 2 needed, 0 free"):
        run.decode(run.tokens(2, 1), state)
    with pytest.raises(ValueError, match="exhausted: 1 needed, 0 free"):
        run.prefill(run.tokens(1, 3))
    assert not run.ran and run.standing() == before and state.position == 16
    assert torch.equal(state.sdm_states[0].materialize_dense(), memory)


def test_a_layout_without_one_of_the_attention_layers(device):
    run = Run("ABA", device)
    before = run.standing()
    run.layout = "AB"
    with pytest.raises(ValueError, match="layer 2 is not in the layout"):
        cow.prefill_faithful_sdm_stack("AB", run.sdm, run.tokens(2, 5), capacity=CAPACITY,
                                       attention_block=run.block.prefill)
    assert run.standing() == before


def test_positions_of_each_request_are_compared(device):
    run = Run("A", device)
    _, state = run.prefill(run.tokens(2, 5))
    state.admit(run.prefill(run.tokens(1, 9))[1])
    before = run.standing()
    x = run.tokens(3, 1)
    for off in ([5, 5, 8], [6, 6, 10], [5, 5]):
        at = torch.tensor(off, device=device)
        with pytest.raises(ValueError, match="do not match the KV cache"):
            run.block.decode(0, x, None, None, at)
    assert run.standing() == before
    run.block.decode(0, x, None, None, state.positions)
    assert run.cache.request_lengths() == [6, 6, 10]


def test_layers_called_by_themselves(device):
    """Without the stack the first layer opens the step; one that has not come
    to its end is refused and can be taken back."""

    run = Run("AA", device)
    x, y = run.tokens(2, 16), run.tokens(2, 1)
    with pytest.raises(ValueError, match="layer 1 is not the next"):
        run.block.prefill(1, x)
    run.block.prefill(0, x)
    for again in (lambda: run.block.prefill(0, x), lambda: run.block.decode(0, y, None, None, 16),
                  lambda: run.block.decode(1, y, None, None, 16)):
        with pytest.raises(ValueError, match="is not the next of its step"):
            again()
    with pytest.raises(ValueError, match="has not run attention layer 1"):
        run.prefill(x)
    run.block.abort()
    assert run.cache.requests == 0 and run.cache.free == 24
    _, state = run.prefill(x)
    want = run.block.decode(0, y, None, None, 16)
    with pytest.raises(ValueError, match="has not run attention layer 1"):
        run.decode(y, state)
    run.block.abort()
    run.block.abort()                              # nothing more to take back
    assert run.cache.request_lengths() == [16, 16]
    assert torch.equal(run.block.decode(0, y, None, None, 16), want)
    run.block.decode(1, want, None, None, 16)
    assert run.cache.request_lengths() == [17, 17] == run.cache.lengths.tolist()


def test_take_back(device):
    cache = cow.PagedKVCache(1, 1, 16, capacity=64, pages=8, page_tokens=16, device=device)
    with pytest.raises(ValueError, match="no KV cache step"):
        cache.take_back()
    cache.admit(2)
    cache.extend([15, 16])
    first = cache.extend([2, 1])
    assert cache.free == 4
    cache.take_back()
    assert cache.lengths.tolist() == [15, 16] == cache.request_lengths()
    assert cache.free == cache.free_count.item() == 6
    with pytest.raises(ValueError, match="no KV cache step"):
        cache.take_back()
    again = cache.extend([2, 1])
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    for change in (lambda: cache.release([0]), cache.compact, lambda: cache.admit(1)):
        change()
        with pytest.raises(ValueError, match="no KV cache step"):
            cache.take_back()
    assert cache.request_lengths() == [17, 0]
    cache.extend([0, 5])
    cache.take_back()
    assert cache.request_lengths() == [17, 0] and cache.free == 6


def test_layers_whose_weights_require_a_gradient(device):
    """As in the stack, no gradient is recorded."""

    run = Run("A", device)
    run.wqkv[0].requires_grad_(), run.wo[0].requires_grad_()
    out = run.block.prefill(0, run.tokens(2, 5))[0]
    assert not out.requires_grad
    assert not run.block.decode(0, out[:, -1:], None, None, 5).requires_grad
