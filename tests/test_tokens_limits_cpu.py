"""Sizes that the packed-token operators ask of their caller."""

from __future__ import annotations

import ctypes

import pytest

from ctmr_b200 import _lib


def _workspace(rows, segments, rank, inner=4096, outer=4096):
    d = _lib.AdapterLinearDesc(0x1000, inner, _lib.DTYPE_BF16, rows, inner, outer, 0x2000, inner, None, 0, 0x4000, 0x5000,
                               0x6000, 2, rank, 0x7000, 0x8000, segments, 0x9000, outer)
    return _lib.LIB.ctmr_adapter_linear_workspace_size(ctypes.byref(d))


@pytest.mark.parametrize(("inner", "outer"), [(4096, 4096), (512, 1536)])
@pytest.mark.parametrize("rank", [16, 64, 128])
@pytest.mark.parametrize("segments", [1000, 4096, 8000])
def test_short_segments_do_not_take_a_large_tile_each(segments, rank, inner, outer):
    """One-row segments own a block of the workspace each: of 64 rows at most, not of a CTA pair's 256."""
    blocks = segments + segments // 16
    assert 0 < _workspace(segments, segments, rank, inner, outer) <= blocks * 64 * rank * 2


@pytest.mark.parametrize("rank", [8, 24, 128])
def test_long_segments_take_little_more_than_their_rows(rank):
    pad = (rank + 15) // 16 * 16
    assert _workspace(8192, 8, rank) <= (8192 + 8 * 256) * pad * 2
