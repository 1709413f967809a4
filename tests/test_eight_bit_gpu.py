"""The 8-bit row operators (``rms_norm``, ``quantize_rows``, ``scaled_linear``) against plain implementations in 64 bits.

Tolerances follow from the roundings. With u the half-ulp of the output's type (bf16 2^-8, fp16 2^-11, fp32 2^-24):

* norm without 8 bits: one rounding of y, and the fp32 roundings of the sum, the factor and two products:
  ``u |y| + 2^-21 |y|``; the sum is one fp32 addition rounded to the type, bit for bit;
* 8-bit values: the nearest e4m3 of the 64-bit value over the group's scale, half a step of the value's binade. Where
  the residual's addition rounds in fp32 the mean square carries its relative error, at most 2^-23, the factor
  half of that: ``step / 2 + 2^-24 |v|``; without a residual 64 bits' own error, ``step / 2 + 2^-40 |v|``. Scales are
  equal (no input's largest magnitude lies that near to 448 times a power of two, but where it is meant to).
* product: one rounding of y, and fp32 sums of n products: ``u |y| + 2^-23 sqrt(n) sum |x||w|``.
fp16 results below the smallest normal number round in steps of 2^-24, so 2^-25 is always allowed.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = [torch.bfloat16, torch.float16, torch.float32]
E4M3 = torch.float8_e4m3fn


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def _within(got, ref, tol):
    got = got.double()
    assert got.shape == ref.shape
    assert torch.isfinite(got).all()
    over = ((got - ref).abs() - tol).max().item() if got.numel() else 0.0
    assert over <= 0.0, f"{over:.3e} over the tolerance; error {(got - ref).abs().max().item():.3e}"


def _no_device_error():
    from ctmr_b200 import _lib

    assert _lib.device_error(clear=True) == 0


def _groups(v):
    return torch.nn.functional.pad(v, (0, -v.shape[1] % 128)).unflatten(1, (-1, 128))


def _scale_of(v):
    """Scales of 64-bit rows: the least 2^k, k >= -100, that brings the largest magnitude to 448 or below."""
    fraction, exponent = torch.frexp(_groups(v).abs().amax(dim=2))
    k = torch.where(fraction == 0, -100, (exponent - 9 + (fraction > 0.875)).clamp(min=-100))
    return torch.ldexp(torch.ones_like(fraction), k)


def _check_rows(got, v, slack=2.0 ** -40):
    """`got` are the ScaledRows of the 64-bit rows `v`."""
    values, scale = got
    assert values.dtype == E4M3 and scale.dtype == torch.float32 and values.shape == v.shape
    ref = _scale_of(v)
    assert torch.equal(scale.double(), ref)
    u = v / ref.repeat_interleave(128, dim=1)[:, :v.shape[1]]
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3.0)
    _within(values, u, step / 2 + slack * u.abs())


def _norm_ref(x, residual, weight, eps):
    h = x.double() if residual is None else x.double() + residual.double()
    y = h / torch.sqrt(h.square().mean(dim=-1, keepdim=True) + eps)
    return y if weight is None else y * weight.double()


def _check_norm(x, weight, residual, eps, quantize, **kw):
    from ctmr_b200 import ops

    ref = _norm_ref(x, residual, weight, eps)
    total = None if residual is None else (x.float() + residual.float()).to(x.dtype)
    y = ops.rms_norm(x, weight, residual=residual, eps=eps, quantize=quantize, **kw)
    if residual is not None:
        y, h = y
        assert torch.equal(h, total)
    if quantize:
        assert x.shape[0] <= 1 or y.values.stride(0) % 16 == 0
        _check_rows(y, ref, 2.0 ** -40 if residual is None else 2.0 ** -24)
    else:
        assert y.dtype == x.dtype
        _within(y, ref, (U[x.dtype] + 2.0 ** -21) * ref.abs() + 2.0 ** -25)
    _no_device_error()


# ---------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(("rows", "channels"), [
    (1, 1), (3, 7), (5, 8), (2, 127), (9, 128), (130, 129), (31, 256), (33, 260), (17, 512), (8, 1000), (7, 1024),
    (5, 1025), (3, 1032), (40, 4096), (1, 5000), (2, 8200), (3, 16384), (2, 16390), (2, 32768), (1, 32761)])
def test_norm(rows, channels, dtype, quantize):
    gen = _gen(rows * 40000 + channels)
    x = _randn(gen, rows, channels, dtype=dtype, std=3.0)
    weight = 1.0 + _randn(gen, channels, std=0.2)
    _check_norm(x, weight, _randn(gen, rows, channels, dtype=dtype), 1e-6, quantize)
    _check_norm(x, weight.to(dtype), None, 1e-5, quantize)
    _check_norm(x, None, None, 1e-3, quantize)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_norm_slices_and_in_place(dtype, shift):
    """Columns of wider tensors, aligned or not; the sum over x or over the residual; y over x."""
    from ctmr_b200 import ops

    gen = _gen(5 + shift)
    rows, channels = 37, 640
    weight = 1.0 + _randn(gen, channels, std=0.2)
    for quantize in (False, True):
        for over in ("x", "residual", "y"):
            if over == "y" and quantize:
                continue
            wide = _randn(gen, rows, channels + 24, dtype=dtype)
            other = _randn(gen, rows, 2 * channels, dtype=dtype)
            x, residual = wide[:, shift:shift + channels], other[:, :channels]
            around = wide.clone()
            ref = _norm_ref(x, residual, weight, 1e-6)
            total = (x.float() + residual.float()).to(dtype)
            kw = dict(out=x) if over == "y" else dict(sum_out=x if over == "x" else residual)
            y, h = ops.rms_norm(x, weight, residual=residual, quantize=quantize, **kw)
            assert torch.equal(h, total)
            assert (y if over == "y" else h).data_ptr() == (residual if over == "residual" else x).data_ptr()
            if quantize:
                _check_rows(y, ref, 2.0 ** -24)
            else:
                _within(y, ref, (U[dtype] + 2.0 ** -21) * ref.abs() + 2.0 ** -25)
            outside = torch.ones(channels + 24, dtype=torch.bool, device="cuda")
            outside[shift:shift + channels] = False
            assert torch.equal(wide[:, outside], around[:, outside])
    _no_device_error()


@pytest.mark.parametrize(("heads", "dim"), [(4, 64), (3, 72), (8, 128), (1, 40), (2, 2048), (5, 33)])
def test_norm_of_heads(heads, dim):
    """The query and key heads of a fused projection, in place."""
    from ctmr_b200 import ops

    gen = _gen(heads * dim)
    qkv = _randn(gen, 50, 3 * heads, dim, dtype=torch.bfloat16)
    before, weight = qkv.clone(), 1.0 + _randn(gen, dim, std=0.2)
    view = qkv[:, :2 * heads]
    ref = _norm_ref(view, None, weight, 1e-6)
    assert ops.rms_norm(view, weight, out=view) is view
    _within(view, ref, (2.0 ** -8 + 2.0 ** -21) * ref.abs())
    assert torch.equal(qkv[:, 2 * heads:], before[:, 2 * heads:])
    x, residual = before[:, heads:2 * heads], before[:, :heads]
    _check_norm(x, weight, residual, 1e-6, False)


def test_norm_zero_rows_large_small_and_not_finite():
    from ctmr_b200 import ops

    gen = _gen(11)
    x = _randn(gen, 9, 384, dtype=torch.float32)
    x[1] = 0.0
    x[2] *= 1e30     # squares past 32 bits
    x[3] *= 1e-30    # below eps: v = x / sqrt(eps)
    x[5, 200] = float("inf")
    x[7, 3] = float("nan")
    for quantize in (False, True):
        y = ops.rms_norm(x, quantize=quantize)
        ref = _norm_ref(x, None, None, 1e-6)
        keep = [0, 1, 2, 3, 4, 6, 8]
        if quantize:
            _check_rows(ops.ScaledRows(y.values[keep], y.scale[keep]), ref[keep])
            got = y.float()
        else:
            _within(y[keep], ref[keep], 2.0 ** -20 * ref[keep].abs())
            got = y
        # An infinity's own group is NaN (infinity times zero), the rest of its row zero; a NaN's row is NaN.
        assert torch.isnan(got[5, 200]) and (got[5, :128] == 0).all() and (got[5, 256:] == 0).all()
        assert torch.isnan(got[5, 128:256]).all() == quantize
        assert torch.isnan(got[7]).all()
    _no_device_error()


def test_norm_of_no_rows():
    from ctmr_b200 import ops

    x = torch.empty((0, 256), dtype=torch.bfloat16, device="cuda")
    assert ops.rms_norm(x).shape == (0, 256)
    y, h = ops.rms_norm(x, residual=x, quantize=True)
    assert y.values.shape == (0, 256) and y.scale.shape == (0, 2) and h.shape == (0, 256)
    assert ops.quantize_rows(x, gate=True).values.shape == (0, 128)


# ---------------------------------------------------------------------------------------------- quantiser
def _gate_ref(x):
    a, b = x.double().chunk(2, dim=1)
    return a / (1.0 + torch.exp(-a)) * b


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(("rows", "channels"), [
    (1, 1), (3, 7), (5, 8), (2, 127), (9, 128), (700, 129), (617, 256), (33, 260), (1, 4096), (8, 1000), (300, 11264),
    (4000, 136), (2, 100000)])
def test_quantize(rows, channels, dtype, gate):
    from ctmr_b200 import ops

    gen = _gen(rows * 40000 + channels)
    x = _randn(gen, rows, channels * (2 if gate else 1), dtype=dtype, std=4.0)
    _check_rows(ops.quantize_rows(x, gate=gate), _gate_ref(x) if gate else x.double())
    wide = _randn(gen, rows, x.shape[1] + 5, dtype=dtype, std=0.1)
    x = wide[:, 3:3 + x.shape[1]]
    _check_rows(ops.quantize_rows(x, gate=gate), _gate_ref(x) if gate else x.double())
    _no_device_error()


def test_quantize_ties_and_borders():
    """Every e4m3 value, the ties between them (to even) and the numbers beside the ties; groups whose largest
    magnitude is 448 times a power of two, and the next number above."""
    from ctmr_b200 import ops

    codes = torch.arange(127, dtype=torch.uint8, device="cuda").view(E4M3).float()  # 0 .. 448
    ties = (codes[1:] + codes[:-1]) / 2
    x = torch.cat([codes, ties, ties * (1 + 2.0 ** -23), ties * (1 - 2.0 ** -23)])
    x = torch.cat([x, -x])
    x = torch.nn.functional.pad(x, (0, -x.numel() % 127)).view(-1, 127)
    x = torch.cat([x, torch.full((x.shape[0], 1), 448.0, device="cuda")], dim=1)
    got = ops.quantize_rows(x)
    assert (got.scale == 1).all()
    assert torch.equal(got.values.view(torch.uint8), x.to(E4M3).view(torch.uint8))
    for k in (-90, -20, 0, 60):
        top = torch.tensor([448.0, 448.0 * (1 + 2.0 ** -23), 448.0 * (1 - 2.0 ** -24), 449.0], device="cuda") * 2.0 ** k
        rows = torch.zeros((4, 128), device="cuda")
        rows[:, 77] = top
        assert ops.quantize_rows(rows).scale.flatten().tolist() == [2.0 ** k, 2.0 ** (k + 1), 2.0 ** k, 2.0 ** (k + 1)]
    _no_device_error()


def test_gate_borders():
    """Gated values that lie on a tie or on a scale's border but for their last bits: 64 bits decide."""
    from ctmr_b200 import ops

    gen = _gen(3)
    a = _randn(gen, 64, 128, std=2.0)
    silu = a.double() / (1 + torch.exp(-a.double()))
    # b brings silu(a) b as near to (odd / 16) or to 448 as 32 bits allow.
    target = (torch.randint(8, 16, a.shape, generator=gen, device="cuda") * 2 + 1).double() / 16
    b = (target / silu).float()
    a[:, 5], b[:, 5] = 30.0, 448.0 / 30.0
    x = torch.cat([a, b], dim=1)
    x[::2, 128 + 5] = torch.nextafter(x[::2, 128 + 5], torch.tensor(0.0, device="cuda"))
    _check_rows(ops.quantize_rows(x, gate=True), _gate_ref(x))


def test_quantize_extremes_and_not_finite():
    from ctmr_b200 import ops

    x = _randn(_gen(1), 6, 300, dtype=torch.bfloat16)
    x[0] = 0.0
    x[1] *= 1e37
    x[2] *= 1e-37   # below the least scale: zeros
    x[3, 130] = float("-inf")
    x[4, 299] = float("nan")
    got = ops.quantize_rows(x)
    keep = torch.tensor([0, 1, 2, 5], device="cuda")
    _check_rows(ops.ScaledRows(got.values[keep], got.scale[keep]), x[keep].double())
    back = got.float()
    assert (back[0] == 0).all() and torch.isfinite(back[1]).all()
    assert torch.isnan(back[3, 128:256]).all() and torch.isfinite(back[3, :128]).all() and torch.isfinite(back[3, 256:]).all()
    assert torch.isnan(back[4, 256:]).all() and torch.isfinite(back[4, :256]).all()
    a = torch.tensor([-200.0, -90.0, -88.0, -30.0, 0.0, 30.0, 90.0, 3e38] * 16, device="cuda")
    pair = torch.cat([a, torch.full_like(a, 0.5)])[None]
    _check_rows(ops.quantize_rows(pair, gate=True), _gate_ref(pair))
    pair[0, 7] = 1.0  # the small ones decide the scale
    pair = torch.where(pair[:, :128].repeat(1, 2).abs() > 1e30, 0.0, pair)
    _check_rows(ops.quantize_rows(pair, gate=True), _gate_ref(pair))


# ---------------------------------------------------------------------------------------------- product
def _rows8(gen, rows, channels, std=1.0):
    """8-bit rows with scales of any value, not only powers of two."""
    from ctmr_b200 import ops

    x = ops.quantize_rows(_randn(gen, rows, channels, std=std))
    return ops.ScaledRows(x.values, x.scale * (0.5 + torch.rand(x.scale.shape, generator=gen, device="cuda")))


def _weight8(gen, out, inner):
    from ctmr_b200 import ops

    w = ops.scale_weight(_randn(gen, out, inner, std=inner ** -0.5))
    return ops.ScaledWeight(w.values, w.scale * (0.5 + torch.rand(w.scale.shape, generator=gen, device="cuda")))


def _spread(scale, dim, n):
    return scale.double().repeat_interleave(128, dim=dim).narrow(dim, 0, n)


def _linear_ref(x, weight, bias):
    """(y, sum |x||w|) in 64 bits."""
    out, inner = weight.values.shape
    a = x.values.double() * _spread(x.scale, 1, inner)
    w = weight.values.double() * _spread(_spread(weight.scale, 0, out), 1, inner)
    y = a @ w.T
    return (y if bias is None else y + bias.double()), a.abs() @ w.abs().T


def _check_linear(got, x, weight, bias):
    ref, size = _linear_ref(x, weight, bias)
    inner = weight.values.shape[1]
    _within(got, ref, U[got.dtype] * ref.abs() + 2.0 ** -23 * inner ** 0.5 * size + 2.0 ** -25)
    _no_device_error()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(("rows", "inner", "outer"), [
    (1, 1, 1), (1, 64, 7), (3, 100, 128), (1, 4096, 1000), (16, 128, 129), (17, 1024, 256), (32, 4096, 512),
    (33, 1000, 1000), (64, 2000, 130), (65, 640, 384), (100, 129, 77), (128, 512, 1536), (129, 2048, 4096),
    (300, 256, 2000), (617, 512, 1536), (1000, 4096, 512), (2049, 1032, 520), (1300, 333, 4097), (5000, 128, 256),
    (4096, 2048, 2048), (1, 20000, 300)])
def test_linear(rows, inner, outer, dtype):
    from ctmr_b200 import ops

    gen = _gen(rows * 7 + inner + outer)
    x, w = _rows8(gen, rows, inner), _weight8(gen, outer, inner)
    bias = _randn(gen, outer, std=0.5)
    _check_linear(ops.scaled_linear(x, w, out_dtype=dtype), x, w, None)
    _check_linear(ops.scaled_linear(x, w, bias, out_dtype=dtype), x, w, bias)
    _check_linear(ops.scaled_linear(x, w, bias.to(dtype), out_dtype=dtype), x, w, bias.to(dtype))


@pytest.mark.parametrize("rows", [5, 90, 700])
def test_linear_strides(rows):
    """Rows, weights and outputs inside wider tensors, scales in either order; what lies around stays."""
    from ctmr_b200 import ops

    gen = _gen(rows)
    inner, outer = 384, 650
    x, w = _rows8(gen, rows, inner + 128), _weight8(gen, outer + 128, inner + 256)
    part = ops.ScaledRows(x.values[:, 128:], x.scale[:, 1:].contiguous())
    wide = ops.ScaledWeight(w.values[128:, 128:128 + inner], w.scale[1:, 1:4].t().contiguous().t())
    for dtype in TYPES:
        room = torch.full((rows, outer + 9), 7.0, dtype=dtype, device="cuda")
        out = room[:, 3:3 + outer]
        assert ops.scaled_linear(part, wide, out=out) is out
        _check_linear(out, part, wide, None)
        assert (room[:, :3] == 7).all() and (room[:, 3 + outer:] == 7).all()


@pytest.mark.parametrize("rows", [3, 700])
def test_linear_one_scale_for_all(rows):
    """A scale for a whole tensor, or for a whole row, expanded."""
    from ctmr_b200 import ops

    gen = _gen(rows)
    x, w = _rows8(gen, rows, 640), _weight8(gen, 300, 640)
    x = ops.ScaledRows(x.values, x.scale[:, :1].expand(rows, 5))
    w = ops.ScaledWeight(w.values, w.scale[:1, :1].expand(3, 5))
    _check_linear(ops.scaled_linear(x, w, out_dtype=torch.float32), x, w, None)


def test_calls_on_two_streams_at_once():
    """Each call by itself: nothing is shared between them."""
    from ctmr_b200 import ops

    gen = _gen(21)
    cases = [(_randn(gen, 600, 2048, dtype=torch.bfloat16), _weight8(gen, 1000, 2048)) for _ in range(2)]

    def chain(x, w):
        y, h = ops.rms_norm(x, residual=x, quantize=True)
        return ops.scaled_linear(y, w), ops.scaled_linear(ops.ScaledRows(y.values[:9], y.scale[:9]), w), h

    alone = [chain(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        both = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                both.append(chain(*c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p, q in zip(alone, both) for a, b in zip(p, q))
    _no_device_error()


@pytest.mark.parametrize("rows", [1, 40, 200, 1500])
def test_linear_not_finite(rows):
    """A NaN or an infinity in a row or in an output's weights stays there; rows' padding is never read."""
    from ctmr_b200 import ops

    gen = _gen(rows)
    inner, outer = 520, 300
    x, w = _rows8(gen, rows, inner), _weight8(gen, outer, inner)
    good = ops.scaled_linear(x, w, out_dtype=torch.float32)
    room = torch.full((rows, 528), 0x7f, dtype=torch.uint8, device="cuda")  # NaN in the padding
    room[:, :inner] = x.values.view(torch.uint8)
    assert torch.equal(ops.scaled_linear(ops.ScaledRows(room.view(E4M3)[:, :inner], x.scale), w, out_dtype=torch.float32), good)
    scale = x.scale.clone()
    scale[rows // 2, 1] = float("nan")
    got = ops.scaled_linear(ops.ScaledRows(x.values, scale), w, out_dtype=torch.float32)
    assert torch.isnan(got[rows // 2]).all()
    keep = torch.arange(rows, device="cuda") != rows // 2
    assert torch.equal(got[keep], good[keep])
    room = torch.zeros((outer, 528), dtype=torch.uint8, device="cuda")
    room[:, :inner] = w.values.view(torch.uint8)
    room[77, 400] = 0x7f
    got = ops.scaled_linear(x, ops.ScaledWeight(room.view(E4M3)[:, :inner], w.scale), out_dtype=torch.float32)
    assert torch.isnan(got[:, 77]).all()
    keep = torch.arange(outer, device="cuda") != 77
    assert torch.equal(got[:, keep], good[:, keep])
    _no_device_error()


def test_linear_same_bits_again():
    """The order of the sums is the same in every call."""
    from ctmr_b200 import ops

    for rows, inner, outer in ((1, 8192, 512), (48, 4096, 1024), (700, 2048, 768)):
        gen = _gen(rows)
        x, w = _rows8(gen, rows, inner), _weight8(gen, outer, inner)
        first = ops.scaled_linear(x, w, out_dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(ops.scaled_linear(x, w, out_dtype=torch.float32), first)


def test_scale_weight():
    from ctmr_b200 import ops

    gen = _gen(4)
    for out, inner in ((1, 1), (128, 128), (300, 200), (129, 1000)):
        weight = _randn(gen, out, inner, dtype=torch.bfloat16)
        got = ops.scale_weight(weight)
        assert got.values.shape == (out, inner) and (out == 1 or got.values.stride(0) % 16 == 0)
        top = weight.double().abs()[:128, :128].max()
        assert torch.frexp(got.scale)[0].eq(0.5).all()  # powers of two
        assert top <= 448 * got.scale[0, 0] and top > 224 * got.scale[0, 0]
        _within(got.float(), weight.double(), 2.0 ** -4 * weight.double().abs() + 2.0 ** -10 * got.scale.max().double())
    assert (ops.scale_weight(torch.zeros((3, 5), device="cuda")).float() == 0).all()
    for bad in (torch.zeros(5), torch.zeros((2, 2), dtype=torch.int32), torch.full((2, 2), float("inf"))):
        with pytest.raises(ValueError):
            ops.scale_weight(bad)


# ---------------------------------------------------------------------------------------------- all
def test_rows_past_32_bits():
    """Rows whose elements lie more than 2^31 apart."""
    from ctmr_b200 import ops

    pitch = 2 ** 31 + 64
    room = torch.empty(pitch + 1024, dtype=torch.float16, device="cuda")
    x = room.as_strided((2, 512), (pitch, 1))
    x.copy_(_randn(_gen(2), 2, 512))
    _check_norm(x, None, None, 1e-6, True)
    _check_norm(x, None, None, 1e-6, False)
    _check_rows(ops.quantize_rows(x), x.double())
    _check_rows(ops.quantize_rows(x, gate=True), _gate_ref(x))


@pytest.mark.parametrize(("rows", "inner", "outer", "pitch"), [(3, 256, 5, 2 ** 30 + 16), (700, 256, 2000, 2 ** 22)])
def test_linear_past_32_bits(rows, inner, outer, pitch):
    """Rows of x and of y, and their scales, more than 2^31 elements from the first, in either form."""
    from ctmr_b200 import ops

    gen = _gen(rows)
    x, w = _rows8(gen, rows, inner), _weight8(gen, outer, inner)
    far = torch.empty((rows - 1) * pitch + inner, dtype=torch.uint8, device="cuda").view(E4M3).as_strided((rows, inner), (pitch, 1))
    far.copy_(x.values)
    out = torch.empty((rows - 1) * pitch + outer, dtype=torch.float16, device="cuda").as_strided((rows, outer), (pitch, 1))
    scale = torch.empty((rows - 1) * pitch + 2, dtype=torch.float32, device="cuda").as_strided((rows, 2), (pitch, 1))
    scale.copy_(x.scale)
    x = ops.ScaledRows(far, scale)
    ops.scaled_linear(x, w, out=out)
    _check_linear(out, x, w, None)


def test_norm_with_the_least_eps():
    """Rows near or at zero, where the mean square and eps lie below 32 bits' normal numbers."""
    from ctmr_b200 import ops

    x = _randn(_gen(4), 6, 512, std=1e-21)
    x[2] = 0.0
    for eps in (1e-38, 1e-40, 1e-44):
        eps = torch.tensor(eps, dtype=torch.float32).item()
        ref = _norm_ref(x, None, None, eps)
        _within(ops.rms_norm(x, eps=eps), ref, 2.0 ** -20 * ref.abs())
        _check_rows(ops.rms_norm(x, eps=eps, quantize=True), ref)


def test_graphs_and_streams():
    """Captured and replayed on other inputs, and called on a stream of its own, with the eager call's bits."""
    from ctmr_b200 import ops

    gen = _gen(8)
    x, residual = _randn(gen, 70, 1536, dtype=torch.bfloat16), _randn(gen, 70, 1536, dtype=torch.bfloat16)
    weight = 1.0 + _randn(gen, 1536, std=0.2)
    w, many = _weight8(gen, 3000, 1536), _rows8(gen, 1000, 1536)

    def both():
        y, h = ops.rms_norm(x, weight, residual=residual, quantize=True)
        z = ops.quantize_rows(h, gate=True)
        return y.values.view(torch.uint8), y.scale, h, z.values.view(torch.uint8), z.scale, ops.scaled_linear(y, w), \
            ops.scaled_linear(ops.ScaledRows(y.values[:5], y.scale[:5]), w), ops.scaled_linear(many, w)

    both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kept = both()
    for seed in (1, 2):
        x.copy_(_randn(_gen(seed), 70, 1536))
        graph.replay()
        eager = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, eager))
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        apart = both()
    other.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(apart, eager))
    _no_device_error()


def test_refusals():
    from ctmr_b200 import ops

    x = torch.zeros((4, 256), dtype=torch.bfloat16, device="cuda")
    bad = [
        lambda: ops.rms_norm(x.cpu()),
        lambda: ops.rms_norm(x.double()),
        lambda: ops.rms_norm(x[0]),
        lambda: ops.rms_norm(x[:, ::2]),
        lambda: ops.rms_norm(x, torch.ones(255, device="cuda")),
        lambda: ops.rms_norm(x, torch.ones(256, device="cuda", dtype=torch.float16)),
        lambda: ops.rms_norm(x, torch.ones(256)),
        lambda: ops.rms_norm(x, residual=x.float()),
        lambda: ops.rms_norm(x, residual=x[:2]),
        lambda: ops.rms_norm(x, sum_out=torch.empty_like(x)),
        lambda: ops.rms_norm(x, eps=0.0),
        lambda: ops.rms_norm(x, eps=float("nan")),
        lambda: ops.rms_norm(x, residual=x, out=x, sum_out=x),
        lambda: ops.rms_norm(x, quantize=True, out=torch.empty_like(x)),
        lambda: ops.rms_norm(x.view(4, 2, 128), quantize=True),
        lambda: ops.rms_norm(torch.zeros((1, 32769), device="cuda")),
        lambda: ops.rms_norm(torch.zeros((2, 0), device="cuda")),
        lambda: ops.quantize_rows(x.view(4, 2, 128)),
        lambda: ops.quantize_rows(x.to(torch.int8)),
        lambda: ops.quantize_rows(x.t()),
        lambda: ops.quantize_rows(x[:, :255], gate=True),
        lambda: ops.quantize_rows(x.cpu()),
    ]
    a, w = ops.quantize_rows(x), ops.scale_weight(torch.ones((300, 256), device="cuda"))
    bad += [
        lambda: ops.scaled_linear(ops.ScaledRows(x, a.scale), w),
        lambda: ops.scaled_linear(ops.ScaledRows(a.values.cpu(), a.scale), w),
        lambda: ops.scaled_linear(ops.ScaledRows(a.values, a.scale[:3]), w),
        lambda: ops.scaled_linear(ops.ScaledRows(a.values, a.scale.double()), w),
        lambda: ops.scaled_linear(ops.ScaledRows(a.values[:, :128], a.scale[:, :1]), w),
        lambda: ops.scaled_linear(ops.ScaledRows(a.values[:, 8:136], a.scale), ops.scale_weight(torch.ones((3, 128), device="cuda"))),
        lambda: ops.scaled_linear(ops.ScaledRows(a.values[:, 8:136], a.scale[:, :1]),
                                  ops.scale_weight(torch.ones((3, 128), device="cuda"))),  # not 16-byte aligned
        lambda: ops.scaled_linear(a, ops.ScaledWeight(w.values, w.scale[:2])),
        lambda: ops.scaled_linear(a, ops.ScaledWeight(w.values, w.scale.cpu())),
        lambda: ops.scaled_linear(a, w, out_dtype=torch.float64),
        lambda: ops.scaled_linear(a, w, torch.ones(299, device="cuda")),
        lambda: ops.scaled_linear(a, w, torch.ones(300, device="cuda", dtype=torch.float16)),
        lambda: ops.scaled_linear(a, w, out=torch.empty((4, 299), device="cuda")),
        lambda: ops.scaled_linear(a, w, out=torch.empty((300, 4), device="cuda").t()),
        lambda: ops.scaled_linear(ops.ScaledRows(torch.zeros((4, 250), device="cuda").to(E4M3), a.scale),
                                  ops.scale_weight(torch.ones((3, 250), device="cuda"))),  # rows 250 bytes apart
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    _no_device_error()
