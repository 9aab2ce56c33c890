"""Calls of the operators around the attention that are larger than a launch,
or that ask for what they do not compute: refused before any launch, so no GPU
is needed."""

from __future__ import annotations

import pytest

from copy_on_write_sdm_amd import _native as nat

FAKE = 0x1000                # never dereferenced: every call fails first


@pytest.mark.parametrize("rows,heads,kv_heads,width,code", [
    (1 << 24, 32, 8, 128, 2),              # a token a workgroup
    (1 << 25, 16, 4, 128, 2),              # two
    ((1 << 24) * 3 - 1, 32, 8, 128, 0), ((1 << 24) * 3 - 1, 8, 8, 96, 1)])
def test_heads_of_more_threads_than_a_launch_counts(rows, heads, kv_heads, width, code):
    """A launch counts its threads in 32 bits: workgroups of 256 threads, one
    to three tokens each."""

    lib, row = nat.lib(), (heads + kv_heads) * width
    a = nat.RotateHeads(FAKE, FAKE, row, width, row, width, FAKE, FAKE, None, None, FAKE, FAKE,
                        rows, heads, kv_heads, width, width, 0, code, 1e-6)
    assert lib.cowsdm_rotate_heads(a, None) == nat.ELIMIT
    assert b"too large" in lib.cowsdm_last_error_string()
