"""prompt_attention with more blocks of rows than a launch has workgroups for."""

from __future__ import annotations

import pytest
import torch

import copy_on_write_sdm_amd as cow
from attention_cases import packed
from test_gpu_prompt_attention import TYPES, check

pytestmark = pytest.mark.gpu


def test_longest_left_out_of_many_sequences(device):
    """512 prompts of 128 rows and 64 heads: as many workgroups as all rows
    could need for every sequence and head are more than a launch holds, so a
    workgroup takes several blocks, most of which are empty."""

    q, k, v, offsets = packed([128] * 512, 64, 8, 8, torch.bfloat16, 42, device)
    got = cow.prompt_attention(q, k, v, offsets)
    assert torch.equal(got, cow.prompt_attention(q, k, v, offsets, longest=128))
    some = slice(128 * 300, 128 * 301)
    check(q[some], k[some], v[some], offsets[:2], got[some])


@pytest.mark.parametrize("dtype", TYPES)
def test_one_long_sequence_among_many(device, dtype):
    """More sequences than the launch has workgroups for every block of the
    longest."""

    print(f"one long of many {dtype}", flush=True)
    lengths = [3] * 900 + [1500] + [2] * 900
    q, k, v, offsets = packed(lengths, 64, 1, 8, dtype, 43, device)
    got = cow.prompt_attention(q, k, v, offsets)
    for first, n in ((0, 3), (2700, 1500), (4200, 2)):
        rows = slice(first, first + n)
        ends = torch.tensor([0, n], dtype=torch.int32, device=device)
        check(q[rows, :1], k[rows], v[rows], ends, got[rows, :1].contiguous())
        one = cow.prompt_attention(q[rows, 60:], k[rows], v[rows], ends, longest=64)
        assert torch.equal(got[rows, 60:], one)
