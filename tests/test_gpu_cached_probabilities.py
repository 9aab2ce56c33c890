"""Attention over the paged cache, its probabilities: what carries them keeps
more than the bits of a 16-bit query."""

from __future__ import annotations

import pytest
import torch

import copy_on_write_sdm_amd as cow
from attention_cases import assert_within, wide
from oracle import attention as ref
from test_gpu_kv_cache import TYPES, filled, ints, queries

pytestmark = pytest.mark.gpu

# numbers of bfloat16 that carry a probability
PARTS = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 2}


def check(query, cache, numbers, tables, lengths, device, **kw):
    got = cow.cached_attention(query, *cache, ints(tables, device), ints(lengths, device), **kw)
    out, weight, logit = ref.cached(wide(query), *numbers, tables, lengths)
    assert_within(got, out, weight, logit, longest=max([*lengths, 1]), values=numbers[1],
                  parts=PARTS[query.dtype])
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,longest", [(1, 700), (5, 700), (1, 5000)])
def test_probabilities_keep_more_than_a_queries_bits(device, dtype, tokens, longest):
    """Values of both signs cancel, so that a probability's rounding would show
    beside the output's own."""

    lengths = [longest, 300, 64]
    cache, numbers, tables = filled(lengths, 2, 64, 64, device, 21)
    check(queries(3, tokens, 4, 64, dtype, 22, device), cache, numbers, tables, lengths, device)
