"""The attention operators have no backward pass: inputs that require a gradient
are refused, not answered without one.  Refused first of all, so no GPU is
needed."""

from __future__ import annotations

import pytest
import torch

import copy_on_write_sdm_amd as cow
from test_attention_host import cache, ints


@pytest.mark.parametrize("which", ["query", "key", "value"])
def test_inputs_that_require_a_gradient(which):
    q, k = torch.zeros(5, 4, 64), torch.zeros(5, 2, 64)
    inputs = dict(query=q, key=k, value=k.clone())
    inputs[which] = inputs[which].clone().requires_grad_()

    def prompt():
        cow.prompt_attention(**inputs, offsets=ints(2))

    def write():
        cow.write_kv_cache(inputs["key"], inputs["value"], ints(5), *cache())

    def cached():
        cow.cached_attention(inputs["query"][None], *cache(), ints(1, 2), ints(1))

    calls = {"query": (prompt, cached)}.get(which, (prompt, write))
    for call in calls:
        with pytest.raises(RuntimeError, match="no backward pass"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            call()
