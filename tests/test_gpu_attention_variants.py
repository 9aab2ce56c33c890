"""The attention kernels' variants against the definition, each at sizes whose
launch takes it: split keys and whole rows in the prompts, and the splits of a
long cache at every width."""

from __future__ import annotations

import pytest
import torch

import copy_on_write_sdm_amd as cow
from attention_cases import packed
from test_gpu_kv_cache import TYPES, check_cached, filled, queries
from test_gpu_prompt_attention import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [40, 64])
def test_split_keys_at_width_64(device, dtype, width):
    """Few rows of many keys: lengths whose last turn is one tile, two, or
    ends inside either, and values that are not finite."""

    for length in (512, 577, 640, 705):
        print(f"split keys {length} width {width} {dtype}", flush=True)
        q, k, v, offsets = packed([length, 3], 1, 1, width, dtype, length, device)
        check(q, k, v, offsets, cow.prompt_attention(q, k, v, offsets, longest=length))
    v[300, 0, 1], v[650, 0, 2], v[651, 0, 2] = float("nan"), float("inf"), float("-inf")
    check(q, k, v, offsets, cow.prompt_attention(q, k, v, offsets, longest=705))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [32, 64, 72, 96, 128, 136, 192, 256])
def test_whole_rows_at_every_width(device, dtype, width):
    """More workgroups than those that split keys take, and rows too short for
    it; a workgroup that takes several blocks of rows."""

    print(f"whole rows width {width} {dtype}", flush=True)
    q, k, v, offsets = packed([300, 1, 200, 131], 80, 1, width, dtype, width, device)
    v[70, 0, 1], v[320, 0, 3] = float("nan"), float("inf")
    for longest in (300, 64):
        got = cow.prompt_attention(q, k, v, offsets, longest=longest)
        for some in (slice(0, 1), slice(79, 80)):
            check(q[:, some], k, v, offsets, got[:, some].contiguous())
    short, k, v, offsets = packed([50, 3], 2, 1, width, dtype, width, device)
    check(short, k, v, offsets, cow.prompt_attention(short, k, v, offsets, longest=50))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [8, 32, 72, 96, 128, 136, 192, 256])
@pytest.mark.parametrize("tokens", [1, 3])
def test_splits_of_the_long_axis_at_every_width(device, dtype, width, tokens):
    print(f"splits width {width} tokens {tokens} {dtype}", flush=True)
    lengths = [4500, 0, 1100, 2]
    cache, numbers, tables = filled(lengths, 1, width, 64, device, width)
    q = queries(4, tokens, 3, width, dtype, width, device)
    for longest in (4500, 2200):
        assert cow.attention.cached_workspace_bytes(4, tokens, 3, 1, width, longest) > 0
        check_cached(q, cache, numbers, tables, lengths, device, longest=longest)
