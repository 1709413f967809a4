"""What the 8-bit row operators of the C ABI refuse about their outputs' rows: status codes, no CUDA call."""

from __future__ import annotations

import itertools

import pytest
from test_eight_bit_cpu import INVALID, LIB, OK, _norm, _quantize

from ctmr_b200 import _lib

# A descriptor with rows that reaches every check, refused at its last one if at no other.
REFUSED_LAST = dict(sum=0x4000, y=0x4000)


@pytest.mark.parametrize("change", [
    dict(y_token_stride=0),                                  # an expanded tensor
    dict(y_token_stride=255),
    dict(sum_token_stride=0),
    dict(sum_token_stride=128),
    dict(scale_token_stride=0),
    dict(scale_group_stride=0),
    dict(scale_group_stride=9),                              # 10 tokens, one element apart
    dict(sum=0x4000),                                        # y
])
def test_norm_refuses_rows_over_one_another(change):
    assert LIB.ctmr_rms_norm(_norm(**change), None) == INVALID


@pytest.mark.parametrize("change", [
    dict(values_stride=0), dict(values_stride=255), dict(scale_row_stride=0), dict(scale_group_stride=9),
    dict(scale_row_stride=2, scale_group_stride=2)])
def test_quantize_refuses_rows_over_one_another(change):
    assert LIB.ctmr_quantize_rows(_quantize(**change), None) == INVALID


def _overlap(na, a, nb, b, width):
    at = sorted(i * a + j * b for i in range(na) for j in range(nb))
    return any(y - x < width for x, y in zip(at, at[1:]))


def test_norm_of_heads_in_every_layout():
    """Small layouts of (tokens, heads) rows, in either order or between one another, against a count of places."""
    last = b"two tensors"
    seen = [0, 0]
    for tokens, heads, width in itertools.product((1, 2, 3, 5), (1, 2, 4), (1, 3)):
        for a, b in itertools.product(range(0, 16), repeat=2):
            d = _norm(tokens=tokens, heads=heads, channels=width, scale=None, y_token_stride=a, y_head_stride=b,
                      sum_token_stride=width * heads, sum_head_stride=width, **REFUSED_LAST)
            assert LIB.ctmr_rms_norm(d, None) == INVALID
            overlap = last not in LIB.ctmr_last_error()
            assert overlap == _overlap(tokens, a, heads, b, width)
            seen[overlap] += 1
    assert min(seen) > 500


def test_norm_of_the_longest_strides():
    d = _norm(tokens=2 ** 30, heads=1, scale=None, y_token_stride=2 ** 38 - 1, **REFUSED_LAST)
    assert LIB.ctmr_rms_norm(d, None) == INVALID and b"two tensors" in LIB.ctmr_last_error()
    d = _norm(tokens=2 ** 15, heads=2 ** 15, scale=None, y_token_stride=2 ** 38 - 1, y_head_stride=2 ** 38 - 257,
              sum_token_stride=2 ** 30, sum_head_stride=256, **REFUSED_LAST)
    assert LIB.ctmr_rms_norm(d, None) == INVALID and b"two tensors" in LIB.ctmr_last_error()


def test_no_rows_have_no_overlap():
    assert LIB.ctmr_rms_norm(_norm(tokens=0, y_token_stride=0), None) == OK
    assert LIB.ctmr_quantize_rows(_quantize(rows=0, values_stride=0), None) == OK
    assert _lib.LIB is LIB
