"""Attention over a paged cache some of whose pages are missing."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import copy_on_write_sdm_amd as cow
from attention_cases import assert_within, wide
from oracle import attention as ref
from test_gpu_kv_cache import PARTS, TYPES, filled, ints, queries

pytestmark = pytest.mark.gpu


def seen_of(query, keys, values, tables, lengths, page):
    """The definition over the tokens whose pages exist."""

    batch, tokens, heads, width = query.shape
    group = heads // keys.shape[1]
    out, weight, logit = np.zeros(query.shape), np.zeros(query.shape), np.zeros(query.shape[:3])
    for b, length in enumerate(lengths):
        at = np.arange(length)
        pages = tables[b, at // page]
        at, pages = at[pages >= 0], pages[pages >= 0]
        for h in range(heads):
            k = keys[pages, h // group, at % page, :width]
            v = values[pages, h // group, :width, at % page]
            for i in range(tokens):
                n = int((at <= length - tokens + i).sum())
                out[b, i, h], weight[b, i, h], logit[b, i, h] = ref.attend_row(
                    query[b, i, h], k[:n], v[:n], width ** -0.5)
    return out, weight, logit


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 3])
@pytest.mark.parametrize("longest", [200, 5000])
def test_missing_pages_are_left_out(device, dtype, tokens, longest):
    """Rows none of whose pages exist are zero, the others go by what there
    is: in one launch and with the long axis split."""

    print(f"missing pages {dtype} {tokens} {longest}", flush=True)
    lengths = [longest, 64, 130, 128, 40]
    cache, numbers, tables = filled(lengths, 1, 64, 64, device, 31)
    split = cow.attention.cached_workspace_bytes(5, tokens, 2, 1, 64, longest)
    assert (split > 0) == (longest == 5000)
    tables[0, :len(tables[0]) // 2] = -1        # the first splits have nothing
    tables[1, 0] = -1
    tables[2, 1] = -1
    tables[3, 0], tables[3, 1] = -1, -1
    sent = tables.copy()
    sent[3, 1] = 1 << 20                        # outside the pool
    q = queries(5, tokens, 2, 64, dtype, 32, device)
    got = cow.cached_attention(q, *cache, ints(sent, device), ints(lengths, device))
    out, weight, logit = seen_of(wide(q), *numbers, tables, lengths, 64)
    assert_within(got, out, weight, logit, longest=longest, values=numbers[1], parts=PARTS[dtype])
    assert not got[1].any() and not got[3].any()


@pytest.mark.parametrize("longest", [200, 5000])
def test_rows_whose_logits_are_all_minus_infinity_are_not_zero(device, longest):
    """Such a row sees its tokens: its softmax is 0 / 0."""

    lengths = [longest, 3]
    cache, numbers, tables = filled(lengths, 1, 32, 64, device, 33)
    keys = cache[0].view(torch.uint8)
    keys[..., 0] = 0x38                         # one, for every token
    q = queries(2, 1, 1, 32, torch.float32, 34, device)
    q[1] = 0.0
    q[1, 0, 0, 0] = float("-inf")
    got = cow.cached_attention(q, *cache, ints(tables, device), ints(lengths, device))
    assert torch.isfinite(got[0]).all() and torch.isnan(got[1]).all()
    # a NaN key that a row sees, with nothing else
    keys[tables[1, 0], 0, :3, 1] = 0x7f
    q[1] = 1.0
    got = cow.cached_attention(q, *cache, ints(tables, device), ints(lengths, device))
    assert torch.isfinite(got[0]).all() and torch.isnan(got[1]).all()
