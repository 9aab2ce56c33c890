"""Limits of the attention entries, refused before any launch: no GPU needed."""

from __future__ import annotations

import torch

from copy_on_write_sdm_amd import _native as nat
from copy_on_write_sdm_amd import attention


def test_prompts_of_more_pairs_than_a_launch_holds():
    """A launch counts its threads in 32 bits: 2^24 workgroups of 256 are too
    many, however short the sequences."""

    lib = nat.lib()
    fake = 0x1000           # never dereferenced: the call fails first
    for heads, sequences in ((1 << 12, 1 << 12), (1 << 20, 1 << 30), (1, 1 << 24)):
        a = nat.PromptAttention(fake, fake, fake, 64, 64, 64, 64, 64, 64, fake, fake, 4,
                                sequences, 1, heads, 1, 64, 0, 0.1)
        assert lib.cowsdm_prompt_attention(a, None) == -2
        assert b"pairs" in lib.cowsdm_last_error_string()


def test_strides_of_axes_of_one_element_say_nothing():
    """torch calls a tensor contiguous whatever they are."""

    for t in (torch.zeros(1, 1, 65)[..., :64], torch.zeros(1, 3, 1, 64)[..., ::2],
              torch.zeros(70).as_strided((1, 1, 64), (1, 3, 1))):
        _, _, strides = attention._rows(t, 4)
        assert strides == torch.empty(t.shape).stride()


def test_cache_codes_that_cannot_be_loaded():
    """Codes are loaded 16 bytes at a time, from the cache's own address on."""

    lib = nat.lib()
    fake = 0x1000
    q = nat.CachedQuery(fake, 64, 64, 64, fake, fake, fake, 2, 1, 1, 64, 3, 48, 0, 0.1)
    for field in ("key_codes", "value_codes"):
        for off in (1, 8, 15):
            c = nat.KVCache(4, 1, 16, 64, fake, fake, fake, fake)
            setattr(c, field, fake + off)
            q.requests = 0              # nothing to run, were it not refused
            assert lib.cowsdm_cached_attention(c, q, None, 0, None) == -1
            assert b"codes must be 16-byte aligned" in lib.cowsdm_last_error_string()
            assert lib.cowsdm_kv_write(c, fake, 64, 64, fake, 64, 64, 0, 64, fake, 0, None) == -1
            assert b"codes must be 16-byte aligned" in lib.cowsdm_last_error_string()


def test_writes_and_queries_of_more_than_a_launch_holds():
    lib = nat.lib()
    fake = 0x1000
    c = nat.KVCache(4, 1, 16, 64, fake, fake, fake, fake)
    for tokens in (1 << 30, (1 << 31) - 1):
        assert lib.cowsdm_kv_write(c, fake, 64, 64, fake, 64, 64, 0, 64, fake, tokens, None) == -2
        assert b"2^30" in lib.cowsdm_last_error_string()
    # 65,535 query tokens of 65,535 heads over one key head: 2^28 tiles of rows
    q = nat.CachedQuery(fake, 64, 64, 64, fake, fake, fake, 1, 65535, 65535, 64, 3, 48, 0, 0.1)
    assert lib.cowsdm_cached_attention(c, q, None, 0, None) == -2
    assert b"query rows" in lib.cowsdm_last_error_string()
