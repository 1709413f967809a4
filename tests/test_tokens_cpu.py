"""Argument checks of the packed-token entry points of the C ABI: status codes, no CUDA call."""

from __future__ import annotations

import ctypes

import pytest

from ctmr_b200 import _lib

LIB = _lib.LIB


def _rotary(**kw):
    d = _lib.RotaryDesc(0x1000, 0x2000, _lib.DTYPE_F16, 10, 2, 16, 32, 16, 32, 16, 0x3000, 0, 2, 0x4000, 2)
    d.section[0], d.section[1] = 3, 4
    sections = kw.pop("section", None)
    for i, n in enumerate(sections or ()):
        d.section[i] = n
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize(("change", "status"), [
    (dict(dtype=3), _lib.CTMR_ERR_INVALID),
    (dict(tokens=-1), _lib.CTMR_ERR_INVALID),
    (dict(heads=0), _lib.CTMR_ERR_INVALID),
    (dict(head_dim=5000), _lib.CTMR_ERR_UNSUPPORTED),
    (dict(axes=0), _lib.CTMR_ERR_INVALID),
    (dict(axes=9), _lib.CTMR_ERR_INVALID),
    (dict(section=(4, 5)), _lib.CTMR_ERR_INVALID),   # 9 pairs in a head of 16
    (dict(section=(0, 0)), _lib.CTMR_ERR_INVALID),
    (dict(section=(-1, 4)), _lib.CTMR_ERR_INVALID),
    (dict(x=None), _lib.CTMR_ERR_INVALID),
    (dict(x=0x1001), _lib.CTMR_ERR_INVALID),
    (dict(x_token_stride=-2), _lib.CTMR_ERR_INVALID),
    (dict(inv_freq=None), _lib.CTMR_ERR_INVALID),
    (dict(tokens=0, x=None), _lib.CTMR_OK),
])
def test_rotary_validation(change, status):
    assert LIB.ctmr_rotary_axes(ctypes.byref(_rotary(**change)), None) == status
    assert LIB.ctmr_rotary_axes(None, None) == _lib.CTMR_ERR_INVALID


def _linear(**kw):
    d = _lib.AdapterLinearDesc(0x1000, 64, _lib.DTYPE_BF16, 10, 64, 48, 0x2000, 64, 0x3000, _lib.DTYPE_F32, 0x4000, 0x5000,
                               0x6000, 2, 16, 0x7000, 0x8000, 3, 0x9000, 48)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize(("change", "status"), [
    (dict(dtype=_lib.DTYPE_F32), _lib.CTMR_ERR_INVALID),
    (dict(rows=-1), _lib.CTMR_ERR_INVALID),
    (dict(in_features=60), _lib.CTMR_ERR_UNSUPPORTED),
    (dict(x=None), _lib.CTMR_ERR_INVALID),
    (dict(x=0x1008), _lib.CTMR_ERR_INVALID),
    (dict(x_stride=56), _lib.CTMR_ERR_INVALID),
    (dict(weight_stride=68), _lib.CTMR_ERR_INVALID),
    (dict(y_stride=47), _lib.CTMR_ERR_INVALID),
    (dict(bias_dtype=_lib.DTYPE_F16), _lib.CTMR_ERR_INVALID),
    (dict(segments=-1), _lib.CTMR_ERR_INVALID),
    (dict(rank=12), _lib.CTMR_ERR_UNSUPPORTED),
    (dict(rank=136), _lib.CTMR_ERR_UNSUPPORTED),
    (dict(adapters=0), _lib.CTMR_ERR_INVALID),
    (dict(up=0x5004), _lib.CTMR_ERR_INVALID),
    (dict(index=None), _lib.CTMR_ERR_INVALID),
    (dict(), _lib.CTMR_ERR_WORKSPACE),
    (dict(rows=0, x=None, y=None), _lib.CTMR_OK),
])
def test_adapter_linear_validation(change, status):
    d = _linear(**change)
    assert LIB.ctmr_adapter_linear(ctypes.byref(d), None, 0, None) == status
    if status not in (_lib.CTMR_OK, _lib.CTMR_ERR_WORKSPACE):
        assert LIB.ctmr_last_error()
        assert LIB.ctmr_adapter_linear_workspace_size(ctypes.byref(d)) == 0


def _attention(**kw):
    d = _lib.AttentionDesc(q=0x1000, k=0x2000, v=0x3000, out=0x4000, dtype=_lib.DTYPE_F16, documents=2, q_tokens=10,
                           k_tokens=20, heads=4, kv_heads=2, head_dim=64, scale=0.125, q_offsets=0x5000, k_offsets=0x6000)
    for name, heads in (("q", 4), ("k", 2), ("v", 2), ("out", 4)):
        setattr(d, name + "_token_stride", heads * 64)
        setattr(d, name + "_head_stride", 64)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize(("change", "status"), [
    (dict(dtype=_lib.DTYPE_F32), _lib.CTMR_ERR_INVALID),
    (dict(documents=0), _lib.CTMR_ERR_INVALID),
    (dict(k_tokens=-1), _lib.CTMR_ERR_INVALID),
    (dict(kv_heads=3), _lib.CTMR_ERR_INVALID),
    (dict(head_dim=60), _lib.CTMR_ERR_UNSUPPORTED),
    (dict(head_dim=136), _lib.CTMR_ERR_UNSUPPORTED),
    (dict(k_offsets=None), _lib.CTMR_ERR_INVALID),
    (dict(k_lengths=0x7000), _lib.CTMR_ERR_INVALID),
    (dict(prefix=0x7000), _lib.CTMR_ERR_INVALID),
    (dict(scale=0.0), _lib.CTMR_ERR_INVALID),
    (dict(scale=float("inf")), _lib.CTMR_ERR_INVALID),
    (dict(cap=-1.0), _lib.CTMR_ERR_INVALID),
    (dict(cap=float("nan")), _lib.CTMR_ERR_INVALID),
    (dict(max_q=-1), _lib.CTMR_ERR_INVALID),
    (dict(q=None), _lib.CTMR_ERR_INVALID),
    (dict(v=None), _lib.CTMR_ERR_INVALID),
    (dict(k=0x2008), _lib.CTMR_ERR_INVALID),
    (dict(v_token_stride=132), _lib.CTMR_ERR_INVALID),
    (dict(q_offsets=None, k_offsets=None, documents=1 << 20, q_tokens=1 << 20), _lib.CTMR_ERR_UNSUPPORTED),
    (dict(q_tokens=0), _lib.CTMR_OK),
])
def test_attention_validation(change, status):
    d = _attention(**change)
    assert LIB.ctmr_attention(ctypes.byref(d), None) == status
    if status != _lib.CTMR_OK:
        assert LIB.ctmr_last_error()
