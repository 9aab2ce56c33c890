"""Argument errors of the operators around the attention (projections, head
rotation, cache pages), from Python and at the C entries: refused before any
launch, so no GPU is needed; and their oracles against closed forms."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import copy_on_write_sdm_amd as cow
from copy_on_write_sdm_amd import _native as nat
from oracle import pages as pages_ref
from oracle import projections as ref

FAKE = 0x1000                # never dereferenced: every call fails first


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def refuser(call, good):
    def refused(error, match, **kw):
        with pytest.raises(error, match=match):
            call(**{**good, **kw})
    return refused


def test_linear_refusals():
    x, w = torch.zeros(5, 16), torch.zeros(7, 16)
    refused = refuser(cow.linear, dict(x=x, weight=w))
    refused(RuntimeError, "no CPU path")
    refused(ValueError, "the activation must be", activation="tanh")
    refused(ValueError, r"x \[...,K\] and weight \[N,K\]", weight=w[:, :8])
    refused(ValueError, r"x \[...,K\] and weight \[N,K\]", weight=w[0])
    refused(ValueError, "bias must be", bias=torch.zeros(6))
    refused(ValueError, "residual must be", residual=torch.zeros(5, 6))
    refused(ValueError, "residual must be", x=x[None], residual=torch.zeros(5, 7))
    refused(ValueError, "at most 1048576", x=torch.zeros(1).expand(2, 1 << 21),
            weight=torch.zeros(1).expand(3, 1 << 21))
    refused(TypeError, "float32, float16 or bfloat16", x=x.double(), weight=w.double())
    refused(TypeError, "share one type", weight=w.half())
    refused(TypeError, "share one type", bias=torch.zeros(7, dtype=torch.bfloat16))
    for name, t in (("x", x), ("weight", w), ("bias", torch.zeros(7)),
                    ("residual", torch.zeros(5, 7))):
        refused(RuntimeError, "no backward pass", **{name: t.clone().requires_grad_()})
    with torch.no_grad():
        refused(RuntimeError, "no CPU path", x=x.clone().requires_grad_())


def test_rotation_refusals():
    q, k, at = torch.zeros(5, 4, 32), torch.zeros(5, 2, 32), ints(5)
    rotation = cow.HeadRotation(32, device="cpu")
    refused = refuser(cow.rotate_heads, dict(query=q, key=k, positions=at, rotation=rotation))
    refused(RuntimeError, "no CPU path")
    refused(ValueError, r"query \[T,heads,D\]", query=q[0])
    refused(ValueError, r"query \[T,heads,D\]", key=k[:4])
    refused(ValueError, "differ in width", key=k[..., :24])
    refused(ValueError, "a head each", key=k[:, :0])
    refused(ValueError, "multiple of 8", query=q[..., :12], key=k[..., :12])
    refused(ValueError, "at most 256", query=torch.zeros(5, 1, 264), key=torch.zeros(5, 1, 264))
    refused(ValueError, "rotated in 32", query=q[..., :24], key=k[..., :24])
    refused(ValueError, "eps", eps=-1.0)
    refused(ValueError, "eps", eps=math.nan)
    refused(TypeError, "share one type", key=k.half())
    refused(TypeError, "float32, float16 or bfloat16", query=q.double(), key=k.double())
    refused(ValueError, r"weight must be \[D\]", query_norm=torch.zeros(31))
    refused(ValueError, r"weight must be \[D\]", key_norm=torch.zeros(64)[::2])
    refused(TypeError, "share one type", key_norm=torch.zeros(32, dtype=torch.float16))
    refused(RuntimeError, "no backward pass", query=q.clone().requires_grad_())
    refused(RuntimeError, "no backward pass", key_norm=torch.zeros(32).requires_grad_())
    for width in (0, 12, 264, -8):
        with pytest.raises(ValueError, match="multiple of 8"):
            cow.HeadRotation(width, device="cpu")
    for base in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="base must be positive"):
            cow.HeadRotation(32, base=base, device="cpu")
    for wrong in ([1.0] * 15, [math.inf] * 16, torch.zeros(17)):
        with pytest.raises(ValueError, match="16 finite frequencies"):
            cow.HeadRotation(32, frequencies=wrong, device="cpu")


def test_turns_are_the_frequencies():
    """2^-64ths of a turn, to the nearest."""

    frequencies = [1.0, math.pi, 1e-5, -2.0]
    rotation = cow.HeadRotation(8, frequencies=frequencies, device="cpu")
    for f, turns in zip(frequencies, rotation.turns.tolist()):
        got = turns / 2 ** 64 % 1.0
        assert abs(got - f / (2 * math.pi) % 1.0) < 1e-16 * 4
    assert cow.HeadRotation(16, base=100.0, device="cpu").frequencies == tuple(
        100.0 ** (-j / 8) for j in range(8))


def good_tables():
    return dict(lengths=ints(3), page_tables=ints(3, 2), page_shares=ints(4))


def test_page_table_refusals():
    stack = dict(free_pages=ints(4), free_count=ints(1))
    calls = [(cow.fork_page_tables, dict(**good_tables(), **stack, parents=ints(2),
                                         tokens=ints(2), page_tokens=16)),
             (cow.release_page_tables, dict(**good_tables(), **stack, requests=ints(2),
                                            page_tokens=16)),
             (cow.compact_page_tables, dict(**good_tables(), page_tokens=16))]
    for call, good in calls:
        refused = refuser(call, good)
        refused(RuntimeError, "no CPU path")
        refused(ValueError, "page tables take", page_tables=ints(3))
        refused(ValueError, "page tables take", page_shares=ints(4, 1))
    from copy_on_write_sdm_amd import pages

    check = lambda **kw: pages._check_tables(**{**good_tables(), "page_tokens": 16, **kw})  # noqa
    real, pages._need_device = pages._need_device, lambda *a: None
    try:
        assert check() == (3, 2, 4, -1)
        for match, kw in (("a row for every request", dict(page_tables=ints(2, 2))),
                          ("contiguous int32", dict(lengths=torch.zeros(3))),
                          ("contiguous int32", dict(page_shares=ints(8)[::2])),
                          ("16, 32, 64, 128 or 256", dict(page_tokens=24))):
            with pytest.raises(ValueError, match=match):
                check(**kw)
        fork, release = (refuser(c, g) for c, g in calls[:2])
        fork(ValueError, "one parent and token count each", tokens=ints(3))
        fork(ValueError, "one parent and token count each", parents=ints(2, 1), tokens=ints(2, 1))
        fork(ValueError, "at most 4096", parents=ints(4097), tokens=ints(4097))
        fork(ValueError, "free pages must be 4", free_pages=ints(5))
        release(ValueError, "must be a vector", requests=ints(2, 1))
        release(ValueError, "at most 4096", requests=ints(4097))
        release(ValueError, "contiguous int32", requests=torch.zeros(2, dtype=torch.int64))
    finally:
        pages._need_device = real


def cache(layers=None, pages=2, heads=2, page=16, width=64):
    lead = () if layers is None else (layers,)
    codes = torch.float8_e4m3fn
    return dict(key_pages=torch.zeros(*lead, pages, heads, page, width, dtype=codes),
                key_scales=torch.ones(*lead, pages, heads),
                value_pages=torch.zeros(*lead, pages, heads, width, page, dtype=codes),
                value_scales=torch.ones(*lead, pages, heads), sources=ints(1), targets=ints(1))


def test_copy_refusals():
    from copy_on_write_sdm_amd import pages

    refuser(cow.copy_pages, cache())(RuntimeError, "no CPU path")
    real, pages._need_device = pages._need_device, lambda *a: None
    try:
        for good in (cache(), cache(layers=3)):
            refused = refuser(cow.copy_pages, good)
            refused(ValueError, "do not align", value_pages=good["key_pages"])
            refused(ValueError, "do not align", key_scales=good["key_scales"][..., :1])
            refused(TypeError, "float8_e4m3fn", key_pages=good["key_pages"].float())
            refused(ValueError, "contiguous",
                    key_scales=torch.ones(*reversed(good["key_scales"].shape)).permute(
                        *reversed(range(good["key_scales"].ndim)))
                    if good["key_scales"].ndim == 3 else torch.ones(2, 2).t().contiguous().t())
            refused(ValueError, "one source and target each", targets=ints(2))
            refused(ValueError, "contiguous int32", sources=torch.zeros(1))
        refuser(cow.copy_pages, cache(page=24))(ValueError, "16, 32, 64, 128 or 256")
        refuser(cow.copy_pages, cache(width=80))(ValueError, "192 or 256 wide")
        refuser(cow.copy_pages, cache())(ValueError, "of all layers",
                                         key_pages=ints(2, 2, 2).view(torch.int8))
    finally:
        pages._need_device = real


def test_c_entries_refuse_without_launching():
    lib = nat.lib()

    def error():
        return lib.cowsdm_last_error_string()

    def each(call, struct, cases):
        for field, value, code, text in cases:
            kept = getattr(struct, field)
            setattr(struct, field, value)
            assert call(struct, None) == code, (field, error())
            assert text in error(), (field, error())
            setattr(struct, field, kept)

    a = nat.Linear(FAKE, FAKE, None, None, FAKE, 16, 16, 0, 3, 16, 8, 0, 0)
    run = lambda a, stream: lib.cowsdm_linear(a, None, 0, stream)     # noqa: E731
    assert run(None, None) == -1
    each(run, a, (
        ("rows", -1, -1, b"negative size"), ("inner", -1, -1, b"negative size"),
        ("float_type", 3, -1, b"float type"), ("activation", 5, -1, b"activation"),
        ("activation", -1, -1, b"activation"), ("x_row", -16, -1, b"negative stride"),
        ("inner", (1 << 20) + 1, -2, b"2^20"), ("weight_row", 1 << 21, -2, b"2^20"),
        ("rows", 1 << 31, -2, b"too large"), ("outer", 1 << 31, -2, b"too large"),
        ("x", None, -1, b"null"), ("weight", None, -1, b"null"), ("out", None, -1, b"null")))
    a.rows = 0
    assert run(a, None) == 0
    size = lib.cowsdm_linear_workspace_bytes
    assert size(0, 16, 16, 0) == 0 and size(64, 128, 384, 0) == 0 and size(-1, 16, 16, 0) == -1
    assert size(1 << 31, 16, 16, 0) == -1 and size(16, 16, 1 << 31, 0) == -1

    h = nat.RotateHeads(FAKE, FAKE, 128, 32, 64, 32, FAKE, FAKE, None, None, FAKE, FAKE, 3, 4, 2,
                        32, 32, 0, 0, 1e-6)
    assert lib.cowsdm_rotate_heads(None, None) == -1
    each(lib.cowsdm_rotate_heads, h, (
        ("rows", -1, -1, b"bad size"), ("heads", -1, -1, b"bad size"),
        ("width", 12, -1, b"multiple of 8"), ("width", 264, -2, b"at most 256"),
        ("rotated", 12, -1, b"multiple of 8"), ("rotated", 40, -1, b"at most the width"),
        ("float_type", -1, -1, b"float type"), ("eps", -1.0, -1, b"eps"),
        ("eps", math.nan, -1, b"eps"), ("rows", 1 << 40, -2, b"too large"),
        ("heads", 1 << 20, -2, b"too large"), ("query", None, -1, b"null"),
        ("key_out", None, -1, b"null"), ("positions", None, -1, b"null"),
        ("turns", None, -1, b"null"), ("query", FAKE + 4, -1, b"aligned"),
        ("key_head", 2, -1, b"aligned"), ("query_row", -128, -1, b"aligned")))
    h.rows = 0
    assert lib.cowsdm_rotate_heads(h, None) == 0

    size = lib.cowsdm_page_tables_release_workspace_bytes
    assert size(10, 4, 3) >= 4 * (10 + 3) and size(-1, 4, 3) == -1 and size(10, 4, 5000) == -1
    size = lib.cowsdm_page_tables_compact_workspace_bytes
    assert size(10) >= 40 and size(-1) == -1 and size(1 << 40) == -1

    def fork(requests=3, columns=2, pages=4, children=2, page=16, lengths=FAKE, shares=FAKE,
             parents=FAKE, count=FAKE):
        return lib.cowsdm_page_tables_fork(lengths, FAKE, requests, columns, shares, FAKE, pages,
                                           count, parents, FAKE, children, page, *[FAKE] * 7, None)

    def release(requests=3, columns=2, pages=4, n=2, page=16, lengths=FAKE, shares=FAKE,
                named=FAKE, count=FAKE, workspace=FAKE, room=1 << 20):
        return lib.cowsdm_page_tables_release(lengths, FAKE, requests, columns, shares, FAKE,
                                              pages, count, named, n, page, FAKE, FAKE, FAKE,
                                              workspace, room, None)

    def compact(requests=3, columns=2, pages=4, page=16, lengths=FAKE, shares=FAKE,
                workspace=FAKE, room=1 << 20):
        return lib.cowsdm_page_tables_compact(lengths, FAKE, requests, columns, shares, pages,
                                              page, *[FAKE] * 6, workspace, room, None)

    for call in (fork, release, compact):
        for kw, code, text in ((dict(page=24), -1, b"page tokens"),
                               (dict(requests=-1), -1, b"negative size"),
                               (dict(pages=-1), -1, b"negative size"),
                               (dict(requests=1 << 31), -2, b"too large"),
                               (dict(pages=1 << 28), -2, b"2^31 tokens"),
                               (dict(columns=1 << 28), -2, b"2^31 tokens"),
                               (dict(requests=4000, columns=1 << 20), -2, b"2^31 table entries"),
                               (dict(lengths=None), -1, b"null"),
                               (dict(shares=None), -1, b"null")):
            assert call(**kw) == code and text in error(), (call.__name__, kw, error())
    assert fork(children=4097) == -2 and fork(parents=None) == -1 and fork(count=None) == -1
    assert release(n=4097) == -2 and release(named=None) == -1 and release(count=None) == -1
    for call in (release, compact):
        assert call(workspace=None) == -1 and b"workspace" in error()
        assert call(room=8) == -1 and b"workspace" in error()

    c = nat.KVCache(4, 2, 16, 64, FAKE, FAKE, FAKE, FAKE)
    copy = lib.cowsdm_pages_copy
    assert copy(None, 1, FAKE, FAKE, 2, None) == -1
    for field, value, code, text in (
            ("page_tokens", 24, -1, b"page tokens"), ("width", 80, -1, b"cache width"),
            ("width", 288, -1, b"cache width"), ("heads", 0, -1, b"bad size"),
            ("heads", 1 << 20, -2, b"heads"), ("pages", 1 << 28, -2, b"2^31"),
            ("key_codes", None, -1, b"null"), ("value_scales", None, -1, b"null"),
            ("value_codes", FAKE + 8, -1, b"aligned")):
        kept = getattr(c, field)
        setattr(c, field, value)
        assert copy(c, 1, FAKE, FAKE, 2, None) == code, (field, error())
        assert text in error(), (field, error())
        setattr(c, field, kept)
    assert copy(c, -1, FAKE, FAKE, 2, None) == -1 and copy(c, 1, None, FAKE, 2, None) == -1
    assert copy(c, 1, FAKE, FAKE, 1 << 30, None) == -2
    assert copy(c, 1, None, None, 0, None) == 0 and copy(c, 0, FAKE, FAKE, 2, None) == 0


def test_oracle_rotations_are_rotations():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, 2, 16))
    frequencies = cow.HeadRotation(16, device="cpu").frequencies
    for interleaved in (False, True):
        near, _ = ref.rotate(x, [0, 1, 5, 100], frequencies, interleaved=interleaved)
        np.testing.assert_allclose(near[0], x[0], atol=1e-15)
        np.testing.assert_allclose((near ** 2).sum(-1), (x ** 2).sum(-1), rtol=1e-12)
        # products of two rows go by the difference of their positions
        a, _ = ref.rotate(np.stack([x[0], x[1]]), [10, 13], frequencies, interleaved=interleaved)
        b, _ = ref.rotate(np.stack([x[0], x[1]]), [1010, 1013], frequencies,
                          interleaved=interleaved)
        np.testing.assert_allclose((a[0] * a[1]).sum(-1), (b[0] * b[1]).sum(-1), rtol=1e-9)
    plain = complex(*ref.point(7, 0.3))
    assert abs(plain - complex(math.cos(2.1), math.sin(2.1))) < 1e-15
    normed, _ = ref.rotate(x, [0] * 4, (), weight=np.ones(16), eps=0.0)
    np.testing.assert_allclose((normed ** 2).mean(-1), 1.0, rtol=1e-12)


def test_oracle_activations():
    y = np.linspace(-8, 8, 41)
    for name, f in (("relu", torch.relu), ("gelu", torch.nn.functional.gelu),
                    ("silu", torch.nn.functional.silu),
                    ("gelu_tanh", lambda t: torch.nn.functional.gelu(t, approximate="tanh"))):
        np.testing.assert_allclose(ref.activated(y, name), f(torch.from_numpy(y)).numpy(),
                                   atol=1e-14)


def test_oracle_pages_by_hand():
    tables = np.array([[4, 2, -1], [0, -1, -1]])
    lengths, shares, stack = [20, 16], [0] * 6, [5, 1, 3, -1, -1, -1]
    new, rows, shares, count, sources, targets, bad = pages_ref.fork(
        lengths, tables, shares, stack, 3, [0, 0, 1], [20, 16, 3], 16)
    assert (new, bad, count) == ([20, 16, 3], 0, 1)
    assert rows.tolist() == [[4, 3, -1], [4, -1, -1], [1, -1, -1]]
    assert shares == [0, 0, 0, 0, 2, 0]
    assert (sources, targets) == ([2, -1, 0], [3, -1, 1])
    tables, lengths = np.concatenate((tables, rows)), lengths + new
    pages_ref.check(lengths, tables, shares, stack, count, 16)
    lengths, shares, stack, count = pages_ref.release(lengths, tables, shares, stack, count,
                                                      [2, 0, 2, 9], 16)
    assert (lengths, shares, count) == ([0, 16, 0, 16, 3], [0] * 6, 3)
    assert stack[:3] == [5, 3, 2]
    out, shares, stack, count, sources, targets = pages_ref.compact(lengths, tables, shares, 16)
    assert out.tolist() == [[-1] * 3, [0, -1, -1], [-1] * 3, [2, -1, -1], [1, -1, -1]]
    assert (stack, count) == ([5, 4, 3, -1, -1, -1], 3)
    assert (sources, targets) == ([4, -1, -1], [2, -1, -1])
