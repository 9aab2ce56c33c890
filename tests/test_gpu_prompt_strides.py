"""prompt_attention on rows that lie far apart."""

from __future__ import annotations

import pytest
import torch

import copy_on_write_sdm_amd as cow
from attention_cases import packed
from test_gpu_prompt_attention import TYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_far_apart(device, dtype):
    """Rows further apart than a buffer address reaches."""

    q, k, v, offsets = packed([3], 2, 1, 32, dtype, 41, device)
    want = cow.prompt_attention(q, k, v, offsets)
    room = torch.zeros(3, (1 << 23) + 8, dtype=dtype, device=device)
    far = [room[:, 64 * i:64 * i + t[0].numel()].view(t.shape).copy_(t)
           for i, t in enumerate((q, k, v))]
    assert all(t.stride(0) > 1 << 23 for t in far)
    for i in range(3):
        some = [q, k, v]
        some[i] = far[i]
        assert torch.equal(cow.prompt_attention(*some, offsets), want)
    assert torch.equal(cow.prompt_attention(*far, offsets), want)
