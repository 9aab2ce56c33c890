"""prompt_attention against its definition in 64 bits (oracle/attention.py):
the three types, head widths and groupings, lengths around the kernels' tiles,
empty sequences, rows of no sequence, strides, values that are not finite in
places a row does not see, and a longest length given too small."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import copy_on_write_sdm_amd as cow
from attention_cases import assert_within, packed, wide
from oracle import attention as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def check(q, k, v, offsets, got, scale=None):
    ends = offsets.tolist()
    out, weight, logit = ref.prompt(wide(q), wide(k), wide(v), ends, scale)
    longest = max([b - a for a, b in zip(ends, ends[1:])] + [1])
    assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
    assert_within(got, out, weight, logit, longest=longest, values=wide(v))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [8, 32, 40, 64, 80, 96, 128, 136, 192, 256])
def test_widths(device, dtype, width):
    print(f"prompt width {width} {dtype}", flush=True)
    q, k, v, offsets = packed([70, 1, 0, 131], 2, 1, width, dtype, width, device)
    check(q, k, v, offsets, cow.prompt_attention(q, k, v, offsets, longest=131))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (6, 2), (8, 8), (16, 8), (5, 1)])
def test_groups(device, dtype, heads, kv_heads):
    print(f"prompt heads {heads} over {kv_heads} {dtype}", flush=True)
    q, k, v, offsets = packed([33, 95], heads, kv_heads, 64, dtype, heads, device)
    check(q, k, v, offsets, cow.prompt_attention(q, k, v, offsets, longest=95))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255,
                                    256, 257, 300])
def test_lengths(device, dtype, length):
    print(f"prompt length {length} {dtype}", flush=True)
    q, k, v, offsets = packed([length, length], 1, 1, 128, dtype, length, device)
    check(q, k, v, offsets, cow.prompt_attention(q, k, v, offsets, longest=length))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("longest", [None, 1, 64, 200, 100_000])
def test_longest_is_a_hint(device, dtype, longest):
    q, k, v, offsets = packed([3, 200, 40], 2, 2, 32, dtype, 5, device)
    check(q, k, v, offsets, cow.prompt_attention(q, k, v, offsets, longest=longest))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_sequences_share_key_heads_over_eight(device, dtype):
    q, k, v, offsets = packed([5, 0, 19, 64, 1, 0, 40, 66], 8, 4, 64, dtype, 6, device)
    check(q, k, v, offsets, cow.prompt_attention(q, k, v, offsets, longest=66))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_no_sequence_are_zero(device, dtype):
    q, k, v, offsets = packed([17, 40], 4, 2, 64, dtype, 7, device, gap=9)
    torch.full((66_000,), float("nan"), device=device)      # what the allocator may hand out next
    got = cow.prompt_attention(q, k, v, offsets, longest=40)
    check(q, k, v, offsets, got)
    assert not got[:9].any() and not got[-9:].any()
    empty = torch.zeros(1, dtype=torch.int32, device=device)
    assert not cow.prompt_attention(q, k, v, empty).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_to_do(device, dtype):
    q, k, v, offsets = packed([0, 0], 4, 2, 64, dtype, 7, device)
    assert cow.prompt_attention(q, k, v, offsets).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(device, dtype):
    lengths, heads, width = [20, 45], 4, 40
    q, k, v, offsets = packed(lengths, heads, 2, width, dtype, 8, device)
    want = cow.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), offsets)
    assert torch.equal(cow.prompt_attention(q, k, v, offsets), want)
    # head-major tensors, and rows that do not start on 16 bytes
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(cow.prompt_attention(*turned, offsets), want)
    odd = []
    for t in (q, k, v):
        room = torch.empty(t.shape[0], t.shape[1], width + 1, device=device, dtype=dtype)
        room[..., 1:] = t
        odd.append(room[..., 1:])
    assert torch.equal(cow.prompt_attention(*odd, offsets), want)
    shifted = []
    for t in (q, k, v):
        room = torch.empty(t.numel() + 1, device=device, dtype=dtype)
        shifted.append(room[1:].view(t.shape).copy_(t))
    assert torch.equal(cow.prompt_attention(*shifted, offsets), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [32, 128])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(device, dtype, width):
    lengths = [150, 70]
    q, k, v, offsets = packed(lengths, 2, 1, width, dtype, 9, device)
    nan, inf = float("nan"), float("inf")
    for row, col, x in ((40, 3, nan), (41, 3, inf), (63, 5, inf), (64, 7, -inf), (90, 5, -inf),
                        (149, 0, nan), (150, 1, inf), (219, 2, nan)):
        v[row, 0, col] = x
    got = cow.prompt_attention(q, k, v, offsets, longest=150)
    check(q, k, v, offsets, got)
    # rows before the first such value, and of the other sequence, are as without them
    clean = torch.where(torch.isfinite(v), v, 0.0)
    want = cow.prompt_attention(q, k, clean, offsets, longest=150)
    assert torch.equal(got[:40], want[:40])
    assert torch.equal(got[..., 8:], want[..., 8:])


@pytest.mark.parametrize("dtype", TYPES)
def test_keys_that_are_not_finite_reach_only_rows_that_see_them(device, dtype):
    q, k, v, offsets = packed([100, 30], 2, 1, 64, dtype, 10, device)
    k[70, 0, 4] = float("nan")
    k[101, 0, 4] = float("inf")
    got = cow.prompt_attention(q, k, v, offsets)
    k2 = k.clone()
    k2[70, 0, 4] = k2[101, 0, 4] = 0.0
    want = cow.prompt_attention(q, k2, v, offsets)
    assert torch.equal(got[:70], want[:70]) and torch.equal(got[100], want[100])
    assert torch.isnan(got[70:100]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_large_logits_and_scale(device, dtype):
    q, k, v, offsets = packed([80], 2, 2, 64, dtype, 11, device)
    for scale in (0.5, 3.0, 1e-6):
        check(q, k, v, offsets, cow.prompt_attention(q, k, v, offsets, scale=scale), scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_whose_maximum_rises_late(device, dtype):
    """Every later key's logit is larger than all before it, by little and
    by much: the running maximum moves all along the row."""

    for step in (0.05, 1.0):
        q, k, v, offsets = packed([200], 1, 1, 32, dtype, 12, device)
        q.fill_(1.0)
        k.copy_((torch.arange(200, device=device) * step / 32)[:, None, None].expand(200, 1, 32))
        check(q, k, v, offsets, cow.prompt_attention(q, k, v, offsets, scale=1.0), 1.0)


def test_another_stream(device):
    q, k, v, offsets = packed([64, 200], 4, 2, 64, torch.bfloat16, 13, device)
    want = cow.prompt_attention(q, k, v, offsets)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cow.prompt_attention(q, k, v, offsets)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_repeats_are_the_same_bits(device):
    q, k, v, offsets = packed([257, 600, 64], 8, 8, 64, torch.float16, 14, device)
    first = cow.prompt_attention(q, k, v, offsets)
    assert all(torch.equal(cow.prompt_attention(q, k, v, offsets), first) for _ in range(3))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [32, 96, 128])
def test_few_rows_of_many_keys(device, dtype, width):
    """Grids that leave the chip empty, where two waves share a row's keys:
    lengths whose last turn is one tile, two, or ends inside either, values
    that are not finite, and the same rows of a larger grid."""

    for length in (512, 577, 640, 705):
        print(f"few rows {length} width {width} {dtype}", flush=True)
        q, k, v, offsets = packed([length, 3], 1, 1, width, dtype, length, device)
        check(q, k, v, offsets, cow.prompt_attention(q, k, v, offsets, longest=length))
    v[300, 0, 1], v[650, 0, 2], v[651, 0, 2] = float("nan"), float("inf"), float("-inf")
    check(q, k, v, offsets, cow.prompt_attention(q, k, v, offsets, longest=705))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_workgroups(device, dtype):
    """More than four rounds of workgroups, whose order is another, and heads
    over eight, five and one key heads."""

    for heads, kv_heads in ((16, 8), (20, 5), (16, 1)):
        print(f"many workgroups {heads} over {kv_heads} {dtype}", flush=True)
        q, k, v, offsets = packed([130, 1, 0] * 60, heads, kv_heads, 8, dtype, heads, device)
        got = cow.prompt_attention(q, k, v, offsets, longest=130)
        some = slice(0, 131 * 2)
        out, weight, logit = ref.prompt(wide(q[some]), wide(k[some]), wide(v[some]),
                                        offsets[:7].tolist())
        assert_within(got[some], out, weight, logit, longest=130, values=wide(v))
        # the other sequences of 130 rows alone
        for at in (5, 59):
            rows = slice(131 * at, 131 * at + 130)
            alone = torch.tensor([0, 130], dtype=torch.int32, device=device)
            one = cow.prompt_attention(q[rows], k[rows], v[rows], alone)
            assert torch.equal(got[rows], one)
