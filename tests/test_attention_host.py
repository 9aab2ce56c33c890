"""Argument errors of the attention operators, from Python and at the C
entries: refused before any launch, so no GPU is needed; and the oracle's
codes against torch's."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import copy_on_write_sdm_amd as cow
from copy_on_write_sdm_amd import _native as nat
from copy_on_write_sdm_amd import attention
from oracle import attention as ref


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def cache(pages=2, heads=2, page=16, width=64):
    return [torch.zeros(pages, heads, page, width, dtype=torch.float8_e4m3fn),
            torch.ones(pages, heads),
            torch.zeros(pages, heads, width, page, dtype=torch.float8_e4m3fn),
            torch.ones(pages, heads)]


def test_cache_width():
    assert [cow.cache_width(w) for w in (8, 32, 40, 64, 72, 96, 104, 128, 136, 192, 200, 256)] == [
        32, 32, 64, 64, 96, 96, 128, 128, 192, 192, 256, 256]
    for width in (0, -8, 4, 33, 264):
        with pytest.raises(ValueError, match="multiple of 8"):
            cow.cache_width(width)


def test_prompt_refusals():
    q, k = torch.zeros(5, 4, 64), torch.zeros(5, 2, 64)
    good = dict(query=q, key=k, value=k, offsets=ints(2))

    def refused(error, match, **kw):
        with pytest.raises(error, match=match):
            cow.prompt_attention(**{**good, **kw})

    refused(RuntimeError, "no CPU path")
    refused(ValueError, r"query \[T,heads,D\]", query=q[0])
    refused(ValueError, r"query \[T,heads,D\]", value=k[:, :1])
    refused(ValueError, "do not align", query=q[:4])
    refused(ValueError, "multiple of the key heads", query=q[:, :3])
    refused(ValueError, "multiple of the key heads", key=k[:, :0], value=k[:, :0])
    refused(ValueError, "multiple of 8", query=q[..., :12], key=k[..., :12], value=k[..., :12])
    refused(TypeError, "float32, float16 or bfloat16", query=q.double())
    refused(TypeError, "share one type", key=k.half())


def test_cached_refusals():
    q = torch.zeros(3, 1, 4, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        cow.cached_attention(q, *cache(), ints(3, 2), ints(3))
    with pytest.raises(ValueError, match=r"query \[B,n,heads,D\]"):
        cow.cached_attention(q[0], *cache(), ints(3, 2), ints(3))
    with pytest.raises(RuntimeError, match="no CPU path"):
        cow.write_kv_cache(q[0], q[0], ints(1), *cache())
    with pytest.raises(ValueError, match=r"key and value \[T,heads,D\]"):
        cow.write_kv_cache(q[0], q[0, :, :2], ints(1), *cache())
    with pytest.raises(RuntimeError, match="no CPU path"):
        cow.extend_page_tables(ints(3), ints(3), ints(3, 2), ints(4), ints(1), page_tokens=16,
                               tokens=1)
    with pytest.raises(ValueError, match="page_tables"):
        cow.extend_page_tables(ints(3), ints(3), ints(3), ints(4), ints(1), page_tokens=16,
                               tokens=1)


def test_cache_checks():
    device = -1              # what a CPU tensor gives
    view = attention._cache(*cache(), 64, device)
    assert (view.pages, view.heads, view.page_tokens, view.width) == (2, 2, 16, 64)

    def refused(error, match, tensors, width=64):
        with pytest.raises(error, match=match):
            attention._cache(*tensors, width, device)

    refused(ValueError, "is 96 wide", cache(), 72)
    refused(ValueError, "16, 32, 64, 128 or 256", cache(page=24))
    for i, match in ((1, "do not align"), (2, "do not align"), (3, "do not align")):
        bad = cache()
        bad[i] = bad[i][:1]
        refused(ValueError, match, bad)
    bad = cache()
    bad[0] = bad[0].to(torch.float32)
    refused(TypeError, "float8_e4m3fn", bad)
    bad = cache()
    bad[2] = torch.zeros(2, 2, 16, 64, dtype=torch.float8_e4m3fn).transpose(2, 3)
    refused(ValueError, "contiguous", bad)


def test_rows_are_copied_only_where_they_cannot_be_loaded():
    x = torch.zeros(6, 8, 64, dtype=torch.bfloat16)
    for kept in (x, x[:, 2:4], x.transpose(0, 1), x[..., 8:24]):
        tensor, address, strides = attention._rows(kept, 8)
        assert tensor is kept and address == kept.data_ptr() and strides == kept.stride()
    for copied in (x[..., 1:9], x[..., ::2], torch.zeros(6, 8, 65)[..., :64]):
        tensor, address, strides = attention._rows(copied, 8)
        assert address == tensor.data_ptr() != copied.data_ptr() and tensor.is_contiguous()
        assert strides == tensor.stride() and torch.equal(tensor, copied)


def test_c_entries_refuse_without_launching():
    lib = nat.lib()
    fake = 0x1000           # never dereferenced: every call fails first

    def error():
        return lib.cowsdm_last_error_string()

    a = nat.PromptAttention(fake, fake, fake, 64, 64, 64, 64, 64, 64, fake, fake, 4, 1, 4, 1, 1,
                            64, 0, 0.1)
    assert lib.cowsdm_prompt_attention(None, None) == -1
    for field, value, code, text in (
            ("rows", -1, -1, b"bad size"), ("heads", 0, -1, b"bad size"),
            ("kv_heads", 2, -1, b"multiple of key heads"), ("width", 12, -1, b"multiple of 8"),
            ("width", 264, -2, b"at most 256"), ("float_type", 3, -1, b"float type"),
            ("scale", 0.0, -1, b"scale"), ("scale", float("nan"), -1, b"scale"),
            ("scale", float("inf"), -1, b"scale"), ("sequences", 0, -1, b"without a sequence"),
            ("query", None, -1, b"null"), ("offsets", None, -1, b"null"),
            ("key_row", 65, -1, b"multiples of 16 bytes"),
            ("value_head", -64, -1, b"multiples of 16 bytes"),
            ("key", fake + 4, -1, b"aligned"), ("key_row", 1 << 24, -2, b"too large")):
        kept = getattr(a, field)
        setattr(a, field, value)
        assert lib.cowsdm_prompt_attention(a, None) == code, field
        assert text in error(), (field, error())
        setattr(a, field, kept)
    a.rows = 0
    assert lib.cowsdm_prompt_attention(a, None) == 0

    c = nat.KVCache(4, 1, 16, 64, fake, fake, fake, fake)
    q = nat.CachedQuery(fake, 64, 64, 64, fake, fake, fake, 2, 1, 1, 64, 3, 48, 0, 0.1)
    run = lambda: lib.cowsdm_cached_attention(c, q, None, 0, None)     # noqa: E731
    assert lib.cowsdm_cached_attention(None, q, None, 0, None) == -1
    assert lib.cowsdm_cached_attention(c, None, None, 0, None) == -1
    for at, field, value, code, text in (
            (c, "page_tokens", 8, -1, b"page tokens"), (c, "page_tokens", 48, -1, b"page tokens"),
            (c, "page_tokens", 512, -1, b"page tokens"), (c, "width", 80, -1, b"cache width"),
            (c, "pages", 1 << 30, -2, b"2^31"), (c, "key_scales", None, -1, b"null cache"),
            (c, "pages", 0, -1, b"no pages"), (c, "heads", 3, -1, b"multiple of the cache's"),
            (q, "width", 72, -1, b"head width"), (q, "width", 20, -1, b"head width"),
            (q, "tokens", -1, -1, b"bad size"), (q, "longest", 1 << 31, -2, b"too large"),
            (q, "columns", 1 << 31, -2, b"too large"), (q, "float_type", -1, -1, b"float type"),
            (q, "scale", -1.0, -1, b"scale"), (q, "lengths", None, -1, b"null"),
            (q, "query_head", 4, 0, b""), (q, "query_head", 2, -1, b"aligned"),
            (q, "longest", 5000, -1, b"workspace")):
        kept = getattr(at, field)
        setattr(at, field, value)
        if code == 0:
            q.requests = 0          # a good call, with nothing to run
        assert run() == code, (field, error())
        assert code == 0 or text in error(), (field, error())
        q.requests = 2
        setattr(at, field, kept)

    write = lib.cowsdm_kv_write
    assert write(c, fake, 64, 64, fake, 64, 64, 0, 64, fake, 0, None) == 0
    assert write(None, fake, 64, 64, fake, 64, 64, 0, 64, fake, 3, None) == -1
    assert write(c, fake, 64, 64, None, 64, 64, 0, 64, fake, 3, None) == -1
    assert write(c, fake, 66, 64, fake, 64, 64, 0, 64, fake, 3, None) == -1
    assert b"aligned" in error()
    assert write(c, fake, 64, 64, fake, 64, 64, 5, 64, fake, 3, None) == -1
    assert write(c, fake, 64, 64, fake, 64, 64, 0, 64, fake, -3, None) == -1

    extend = lib.cowsdm_page_tables_extend
    rest = [fake] * 6 + [None]
    assert extend(fake, fake, 4097, fake, 2, fake, 4, fake, 16, 4, *rest) == -2
    assert b"4096 requests" in error()
    assert extend(fake, fake, 4, fake, 2, fake, 4, fake, 20, 4, *rest) == -1
    assert extend(fake, fake, 4, fake, -2, fake, 4, fake, 16, 4, *rest) == -1
    assert extend(fake, fake, 4, None, 2, fake, 4, fake, 16, 4, *rest) == -1
    assert extend(fake, fake, 4, fake, 2, fake, 1 << 28, fake, 16, 4, *rest) == -2
    release = lib.cowsdm_pages_release
    assert release(fake, fake, 4, 2, fake, 0, fake, 4, fake, 16, None) == 0
    assert release(fake, fake, 4, 2, None, 2, fake, 4, fake, 16, None) == -1
    assert release(fake, fake, 4, 2, fake, 2, fake, 4, fake, 17, None) == -1

    size = lib.cowsdm_cached_attention_workspace_bytes
    assert size(64, 1, 32, 8, 128, 200) == 0
    assert size(1, 1, 4, 4, 32, 4096) > 0
    assert size(1, 1, 4, 3, 32, 4096) == -1 and size(1, 1, 4, 4, 33, 4096) == -1


def test_oracle_codes_are_the_formats():
    numbers = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(np.isnan(ref.CODES), np.isnan(numbers))
    assert np.array_equal(ref.CODES[~np.isnan(numbers)], numbers[~np.isnan(numbers)])
    rng = np.random.default_rng(1)
    x = np.concatenate([ref._TIES, -ref._TIES, ref._POSITIVE, 448 * rng.uniform(-1, 1, 5000),
                        2.0 ** -7 * rng.standard_normal(5000)]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ref.encode(x), want)
    assert ref.power_scale(448.0) == 1.0 and ref.power_scale(448.1) == 2.0
    assert ref.power_scale(224.0) == 0.5 and ref.power_scale(0.0) == 2.0 ** -100


def test_oracle_attention_is_softmax():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(9, h, 8, generator=g, dtype=torch.float64) for h in (4, 2, 2))
    out, weight, _ = ref.prompt(q.numpy(), k.numpy(), v.numpy(), [0, 4, 4, 9])
    for a, b in ((0, 4), (4, 9)):
        logits = torch.einsum("qhd,khd->hqk", q[a:b], k[a:b].repeat_interleave(2, 1)) / 8 ** 0.5
        logits = logits.masked_fill(torch.ones(b - a, b - a).triu(1).bool(), float("-inf"))
        want = torch.einsum("hqk,khd->qhd", logits.softmax(-1), v[a:b].repeat_interleave(2, 1))
        np.testing.assert_allclose(out[a:b], want.numpy(), rtol=1e-12, atol=1e-14)
    assert (weight >= np.abs(out) - 1e-12).all()
