"""Argument checks of the 8-bit row operators of the C ABI: status codes, no CUDA call."""

from __future__ import annotations

import ctypes

import pytest

from ctmr_b200 import _lib

LIB = _lib.LIB
INVALID, UNSUPPORTED, OK = _lib.CTMR_ERR_INVALID, _lib.CTMR_ERR_UNSUPPORTED, _lib.CTMR_OK


def _changed(d, kw):
    for k, v in kw.items():
        assert hasattr(d, k)
        setattr(d, k, v)
    return ctypes.byref(d)


@pytest.mark.parametrize(("pack", "desc"), [
    (_lib.pack_rms_norm, _lib.RmsNormDesc), (_lib.pack_quantize_rows, _lib.QuantizeRowsDesc),
    (_lib.pack_scaled_linear, _lib.ScaledLinearDesc)])
def test_packed_descriptors_are_the_structures(pack, desc):
    values = [0.5 if t is ctypes.c_float else 3 + 2 * i for i, (_, t) in enumerate(desc._fields_)]
    assert pack(*values) == bytes(desc(*values))


def _norm(**kw):
    return _changed(_lib.RmsNormDesc(0x1000, 0x2000, 0x3000, _lib.DTYPE_BF16, _lib.DTYPE_F32, 10, 1, 256, 256, 0, 256, 0,
                                     1e-6, 0x4000, 256, 0, 0x5000, 256, 0, 0x6000, 1, 10), kw)


@pytest.mark.parametrize(("change", "status"), [
    (dict(dtype=3), INVALID),
    (dict(weight_dtype=_lib.DTYPE_F16), INVALID),
    (dict(tokens=-1), INVALID),
    (dict(heads=0), INVALID),
    (dict(channels=0), INVALID),
    (dict(channels=32769), UNSUPPORTED),
    (dict(tokens=2 ** 30, heads=2, scale=None), UNSUPPORTED),
    (dict(eps=0.0), INVALID),
    (dict(eps=-1.0), INVALID),
    (dict(eps=float("inf")), INVALID),
    (dict(eps=float("nan")), INVALID),
    (dict(heads=2), UNSUPPORTED),                       # 8-bit rows have no heads
    (dict(x=None), INVALID),
    (dict(y=None), INVALID),
    (dict(x=0x1001), INVALID),
    (dict(residual=0x2001), INVALID),
    (dict(weight=0x3002), INVALID),
    (dict(sum=0x5001), INVALID),
    (dict(scale=0x6002), INVALID),
    (dict(scale=None, y=0x4001), INVALID),
    (dict(x_token_stride=-256), INVALID),
    (dict(scale_group_stride=-1), INVALID),
    (dict(y_token_stride=1 << 38), INVALID),
    (dict(tokens=0, x=None, y=None), OK),
])
def test_norm_validation(change, status):
    assert LIB.ctmr_rms_norm(_norm(**change), None) == status
    assert LIB.ctmr_rms_norm(None, None) == INVALID


def _quantize(**kw):
    return _changed(_lib.QuantizeRowsDesc(0x1000, _lib.DTYPE_F16, 10, 256, 1, 512, 0x2000, 256, 0x3000, 1, 10), kw)


@pytest.mark.parametrize(("change", "status"), [
    (dict(dtype=3), INVALID),
    (dict(rows=-1), INVALID),
    (dict(channels=0), INVALID),
    (dict(channels=2 ** 30), UNSUPPORTED),
    (dict(x=None), INVALID),
    (dict(values=None), INVALID),
    (dict(scale=None), INVALID),
    (dict(x=0x1001), INVALID),
    (dict(scale=0x3002), INVALID),
    (dict(x_stride=-1), INVALID),
    (dict(values_stride=-1), INVALID),
    (dict(scale_row_stride=-1), INVALID),
    (dict(rows=0, x=None), OK),
])
def test_quantize_validation(change, status):
    assert LIB.ctmr_quantize_rows(_quantize(**change), None) == status
    assert LIB.ctmr_quantize_rows(None, None) == INVALID


def _linear(**kw):
    return _changed(_lib.ScaledLinearDesc(0x1000, 256, 0x2000, 1, 10, 10, 250, 300, 0x3000, 256, 0x4000, 2, 1, 0x5000,
                                          _lib.DTYPE_F32, 0x6000, _lib.DTYPE_BF16, 300), kw)


@pytest.mark.parametrize(("change", "status"), [
    (dict(y_dtype=3), INVALID),
    (dict(bias_dtype=_lib.DTYPE_F16), INVALID),
    (dict(rows=-1), INVALID),
    (dict(in_features=0), INVALID),
    (dict(out_features=0), INVALID),
    (dict(rows=2 ** 30), UNSUPPORTED),
    (dict(x_stride=248), INVALID),
    (dict(x_stride=264), INVALID),
    (dict(weight_stride=240), INVALID),
    (dict(y_stride=299), INVALID),
    (dict(x_scale_row_stride=-1), INVALID),
    (dict(weight_scale_block_stride=-1), INVALID),
    (dict(x=0x1008), INVALID),
    (dict(weight=0x3008), INVALID),
    (dict(x=None), INVALID),
    (dict(x_scale=None), INVALID),
    (dict(weight_scale=None), INVALID),
    (dict(y=None), INVALID),
    (dict(y=0x6001), INVALID),
    (dict(bias=0x5002), INVALID),
    (dict(x_scale=0x2002), INVALID),
    (dict(rows=0, x=None), OK),
])
def test_linear_validation(change, status):
    assert LIB.ctmr_scaled_linear(_linear(**change), None) == status
    assert LIB.ctmr_scaled_linear(None, None) == INVALID
