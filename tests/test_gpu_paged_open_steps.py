"""Changes of a cache's pool between the layers of a step: what would move or
copy pages that the step has yet to write is refused, and the step goes on, or
is taken back, as if nothing had been asked."""

from __future__ import annotations

import pytest
import torch

from test_gpu_paged_lifecycle import assert_whole
from test_gpu_paged_steps import Run

pytestmark = pytest.mark.gpu

CHANGES = {"fork": lambda c: c.fork([0]), "fork_none": lambda c: c.fork([]),
           "trim": lambda c: c.trim_pages(), "trim_to_all": lambda c: c.trim_pages(
               headroom_pages=1 << 20),
           "grow": lambda c: c.grow_pages(3), "grow_none": lambda c: c.grow_pages(0)}


def refused(run, change):
    before = run.standing(), run.cache.key_pages.data_ptr()
    with pytest.raises(ValueError, match="has not run attention layer 1"):
        CHANGES[change](run.cache)
    assert (run.standing(), run.cache.key_pages.data_ptr()) == before


@pytest.mark.parametrize("change", CHANGES)
def test_between_the_layers_of_a_step(device, change):
    run, plain = Run("AA", device), Run("AA", device)
    x, y = run.tokens(2, 16), run.tokens(2, 1)
    out = run.block.prefill(0, x)[0]
    refused(run, change)
    out = run.block.prefill(1, out)[0]
    assert torch.equal(out, plain.block.prefill(1, plain.block.prefill(0, x)[0])[0])
    out = run.block.decode(0, y, None, None, 16)
    refused(run, change)
    out = run.block.decode(1, out, None, None, 16)
    assert torch.equal(out, plain.block.decode(1, plain.block.decode(0, y, None, None, 16), None,
                                               None, 16))
    assert all(torch.equal(a, b) for a, b in zip(run.codes(), plain.codes()))
    # the step is whole
    CHANGES[change](run.cache)
    assert_whole(run.cache)


@pytest.mark.parametrize("change", CHANGES)
def test_an_open_step_is_taken_back_after_a_refusal(device, change):
    run = Run("AA", device)
    x = run.tokens(2, 16)
    run.block.prefill(1, run.block.prefill(0, x)[0])
    before = run.standing()
    run.block.decode(0, run.tokens(2, 1), None, None, 16)
    refused(run, change)
    run.block.abort()
    assert run.standing() == before
    CHANGES[change](run.cache)                      # and no step is open any more
    assert_whole(run.cache)


def test_within_the_stack(device):
    """A callable of the stack that asks for it: the whole step is taken back."""

    run = Run("AA", device)
    _, state = run.prefill(run.tokens(2, 16))
    before, project = run.standing(), run.block.project

    def forking(layer, tokens, positions):
        if layer == 1:
            run.cache.fork([0])
        return project(layer, tokens, positions)

    run.block.project = forking
    with pytest.raises(ValueError, match="has not run attention layer 1"):
        run.decode(run.tokens(2, 1), state)
    assert run.standing() == before
    run.block.project = project
    run.decode(run.tokens(2, 1), state)
    assert run.cache.fork([0]) == [2]


@pytest.mark.parametrize("change", CHANGES)
def test_within_the_stack_past_the_attention_layers(device, change):
    run = Run("AB", device)
    _, state = run.prefill(run.tokens(2, 16))
    before, tail = run.standing(), run.tail

    def changing(layer, tokens):
        CHANGES[change](run.cache)

    run.tail = changing
    with pytest.raises(ValueError, match="within a step"):
        run.decode(run.tokens(2, 1), state)
    assert run.standing() == before
    run.tail = tail
    run.decode(run.tokens(2, 1), state)
    CHANGES[change](run.cache)
    assert_whole(run.cache)


def test_a_block_that_is_gone_holds_nothing_open(device):
    run = Run("AA", device)
    run.block.prefill(0, run.tokens(2, 16))
    refused(run, "fork")
    run.block = None
    assert run.cache.fork([1]) == [2]
    assert_whole(run.cache)
