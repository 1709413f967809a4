"""What the 8-bit row operators refuse about outputs, numbers and weights, without a CUDA call."""

from __future__ import annotations

import ctypes
import itertools
from types import SimpleNamespace

import pytest
import torch
from test_eight_bit_cpu import INVALID, LIB, OK, _norm, _quantize

from ctmr_b200 import _lib, ops, packed

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


@pytest.mark.parametrize("value", [1e300, -3.5e38, float("nan"), float("inf")])
def test_weights_past_fp32_are_refused(value):
    weight = torch.ones((3, 5), dtype=torch.float64)
    weight[1, 2] = value
    with pytest.raises(ValueError):
        ops.scale_weight(weight)


def test_weights_of_every_type():
    """A weight is taken in fp32: the largest numbers, e4m3's own, and none but zeros."""
    big = torch.tensor([[3.4e38, 1.0, -3.4e38]], dtype=torch.float64)
    got = ops.scale_weight(big)
    assert got.scale.item() == 2.0 ** 120 and torch.equal(got.values.float(), torch.tensor([[256.0, 0.0, -256.0]]))
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    codes = codes[codes.float().isfinite()].view(2, 127)
    got = ops.scale_weight(codes)
    assert got.scale.item() == 1.0 and torch.equal(got.values.float(), codes.float())
    assert (ops.scale_weight(torch.zeros((2, 300), dtype=torch.float16)).scale == 2.0 ** -100).all()


@pytest.mark.parametrize(("field", "value"), [("tokens", 2 ** 31), ("channels", 2 ** 40), ("eps", "1"),
                                              ("x_token_stride", 2 ** 63), ("heads", 1.5)])
def test_numbers_that_a_descriptor_does_not_hold_are_refused(field, value):
    fields = [0.5 if t is ctypes.c_float else 3 for _, t in _lib.RmsNormDesc._fields_]
    fields[[n for n, _ in _lib.RmsNormDesc._fields_].index(field)] = value
    with pytest.raises(ValueError, match="RmsNormDesc"):
        _lib.pack_rms_norm(*fields)


def test_an_eps_past_fp32_is_refused():
    """It is packed as an infinity, which the entry refuses."""
    fields = [getattr(_norm()._obj, n) or 0 for n, _ in _lib.RmsNormDesc._fields_]
    names = [n for n, _ in _lib.RmsNormDesc._fields_]
    fields[names.index("eps")] = 1e39
    assert LIB.ctmr_rms_norm(_lib.pack_rms_norm(*fields), None) == INVALID and b"eps" in LIB.ctmr_last_error()


@pytest.mark.parametrize("root", [SimpleNamespace(), SimpleNamespace(_dynamo=None),
                                  SimpleNamespace(_dynamo=SimpleNamespace(guards=SimpleNamespace()))])
def test_outputs_are_allocated_where_torch_lacks_its_direct_entry(root, monkeypatch):
    got = {}
    monkeypatch.setattr(torch, "empty_strided", lambda size, stride, **kw: got.update(size=size, stride=stride, **kw))
    ops._allocator(root)((2, 3), (4, 1), torch.float32)
    assert got == dict(size=(2, 3), stride=(4, 1), dtype=torch.float32, device="cuda")


@pytest.mark.parametrize("heads", [0, -2, 3])
def test_blocks_of_no_heads_are_refused(heads):
    with pytest.raises(ValueError, match="heads"):
        packed.packed_transformer_tokens(torch.zeros((8, 64)), SimpleNamespace(starts=[0, 8]), [], heads=heads)
