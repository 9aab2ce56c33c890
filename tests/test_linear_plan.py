"""What a product of given sizes runs: its form and splits, at the C entry.  No
GPU is needed."""

from __future__ import annotations

import pytest

from copy_on_write_sdm_amd import _native as nat

FAKE = 0x1000                # never dereferenced: every call fails first


def plan(rows, inner, outer, float_type, aligned=True):
    """(rows and columns of a tile, splits, workspace bytes)."""

    p = nat.LinearPlan()
    rc = nat.lib().cowsdm_linear_plan(rows, inner, outer, float_type, aligned, p)
    assert rc == 0, nat.lib().cowsdm_last_error_string()
    return (p.tile_rows, p.tile_columns), p.splits, p.workspace_bytes


SIZES = [(r, i, o) for r in (1, 8, 64, 65, 300, 2048) for i in (1, 7, 64, 2048, 4096, 8191)
         for o in (1, 64, 1024, 6144)]


@pytest.mark.parametrize("float_type", [0, 1, 2])
def test_plans_by_alignment(float_type):
    """Rows that do not start on 16 bytes, by their width or by their address,
    run in tiles of 64 by 64 with splits of their own; the workspace that a
    call whose alignment is not told asks for holds either plan's sums."""

    unit = 8 if float_type else 4
    for rows, inner, outer in SIZES:
        odd, aligned = (plan(rows, inner, outer, float_type, a) for a in (False, True))
        assert odd[0] == (64, 64)
        if inner % unit:
            assert aligned == odd
        for _, splits, size in (odd, aligned):
            assert 1 <= splits <= 16
            assert size == (0 if splits == 1 else splits * rows * ((outer + 3) // 4 * 16))
            steps = -(-inner * (16 // unit) // 128)
            assert splits == 1 or (splits - 1) * -(-steps // splits) < steps   # none is empty
        assert nat.lib().cowsdm_linear_workspace_bytes(rows, inner, outer, float_type) == max(
            odd[2], aligned[2])
    # few groups of rows that are not aligned share the summed axis out
    for rows, inner, outer in ((1, 4096, 1024), (1, 4096, 6144), (8, 2048, 2048)):
        assert plan(rows, inner, outer, float_type)[0] == (16, 16)
        assert plan(rows, inner, outer, float_type, False)[1] > 4


def test_calls_get_the_plan_of_their_alignment():
    """A call without the workspace that its own plan needs is refused: by the
    address of either operand and by either stride."""

    lib = nat.lib()
    need = plan(8, 2048, 2048, 2, False)[2]
    assert need and not plan(8, 2048, 2048, 2)[2]
    text = f"workspace of {need} bytes".encode()
    for x, w, x_row, w_row in ((FAKE + 2, FAKE, 2048, 2048), (FAKE, FAKE + 8, 2048, 2048),
                               (FAKE, FAKE, 2049, 2048), (FAKE, FAKE, 2048, 2052)):
        a = nat.Linear(x, w, None, None, FAKE, x_row, w_row, 0, 8, 2048, 2048, 2, 0)
        assert lib.cowsdm_linear(a, None, 0, None) == -1
        assert text in lib.cowsdm_last_error_string()
        assert lib.cowsdm_linear(a, FAKE, need - 16, None) == -1
        assert text in lib.cowsdm_last_error_string()
        assert lib.cowsdm_linear(a, FAKE + 8, need, None) == -1
        assert b"aligned" in lib.cowsdm_last_error_string()


def test_refusals():
    lib, p = nat.lib(), nat.LinearPlan()
    for args, code, text in (((-1, 8, 8, 0), -1, b"negative"), ((8, -1, 8, 0), -1, b"negative"),
                             ((8, 8, -1, 0), -1, b"negative"), ((8, 8, 8, 3), -1, b"float type"),
                             ((8, (1 << 20) + 1, 8, 0), -2, b"too large"),
                             ((1 << 31, 8, 8, 0), -2, b"too large"),
                             ((8, 8, 1 << 31, 0), -2, b"too large")):
        assert lib.cowsdm_linear_plan(*args, 1, p) == code and text in (
            lib.cowsdm_last_error_string())
    assert lib.cowsdm_linear_plan(8, 8, 8, 0, 1, None) == -1
    for rows, inner, outer in ((0, 8, 8), (8, 8, 0)):
        assert plan(rows, inner, outer, 0) == ((0, 0), 0, 0)
    for aligned in (True, False):
        assert plan(3, 0, 5, 0, aligned)[1:] == (1, 0)
