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


@pytest.mark.parametrize("dtype", TYPES)
def test_one_row_with_any_stride(device, dtype):
    """The strides of an axis of one element say nothing."""

    q, k, v, offsets = packed([1], 1, 1, 40, dtype, 44, device)
    want = cow.prompt_attention(q, k, v, offsets)
    for stride in (41, 1, (1 << 23) + 8):
        room = torch.zeros(1 << 24, dtype=dtype, device=device)
        odd = [room[64 * i:].as_strided((1, 1, 40), (stride, stride, 1)).copy_(t)
               for i, t in enumerate((q, k, v))]
        assert torch.equal(cow.prompt_attention(*odd, offsets), want)
        caches = []
        for pair in ((k, v), odd[1:]):
            cache = [torch.zeros(2, 1, 16, 64, dtype=torch.uint8, device=device),
                     torch.ones(2, 1, device=device),
                     torch.zeros(2, 1, 64, 16, dtype=torch.uint8, device=device),
                     torch.ones(2, 1, device=device)]
            caches.append([t.view(torch.float8_e4m3fn) if t.dtype == torch.uint8 else t
                           for t in cache])
            cow.write_kv_cache(*pair, torch.zeros(1, dtype=torch.int32, device=device),
                               *caches[-1])
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8))
                   for a, b in zip(*caches))
        table, one = torch.zeros(1, 1, dtype=torch.int32, device=device), torch.ones(
            1, dtype=torch.int32, device=device)
        assert torch.equal(cow.cached_attention(odd[0][None], *caches[0], table, one),
                           cow.cached_attention(q[None], *caches[0], table, one))
