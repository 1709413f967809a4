"""The 8-bit row operators at the edges of what they accept and in every form that their launchers choose, against plain
implementations in 64 bits.

Tolerances. Norms and 8-bit rows as in test_eight_bit_gpu, the bytes those of the 64-bit formula everywhere:
``step / 2 + 2^-40 |v|``.

Products, in the 2-norm: sums in TMEM take four instructions a block of 128 inputs, each off by at most 2^-23 of the
running sum (a truncation), and after b of B blocks the sum in registers is rounded by 2^-24 of itself. With operands of
random signs a running sum grows as the square root of its terms and the errors of different blocks are independent, so
the squares add up: (B / 2) 2^-48 from the registers and (1 + 2 + 3 + 4) / 4 * 2^-46 from TMEM:
``2^-24 sqrt(B / 2 + 10) ||y||``. fp32's bias addition adds 2^-24 |y| at most. A single row or column: twice that.
"""

from __future__ import annotations

import pytest
import torch
from test_eight_bit_gpu import (TYPES, U, _check_rows, _gate_ref, _gen, _linear_ref, _no_device_error, _norm_ref, _randn,
                                _rows8, _weight8, _within)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- quantiser
@pytest.mark.parametrize("dtype", TYPES)
def test_gates_of_very_negative_values(dtype):
    """silu(a) far below 32 bits' normal numbers, times a b that brings the product back."""
    from ctmr_b200 import ops

    gen = _gen(31)
    a = torch.tensor([-79.0, -85.5, -86.0, -87.0, -87.25, -87.5, -88.0, -88.75, -90.0, -100.0, -103.0, -104.0, -120.0, -140.0,
                      -160.0, -170.0, -200.0, -700.0, -800.0, -60000.0], device="cuda")
    top = torch.finfo(dtype).max
    for size in (1.0, 3.0, 100.0, 60000.0, 1e10, 1e20, 1e30, 3e38):
        if size > top:
            continue
        # whole groups of one a, then a mixed one, then one among ordinary values
        groups = a[:, None].expand(-1, 128).clone()
        mixed = a[torch.randint(a.numel(), (2, 128), generator=gen, device="cuda")]
        mixed[1, 3:] = _randn(gen, 125)
        groups = torch.cat([groups, mixed])
        b = size * (0.5 + 0.5 * torch.rand(groups.shape, generator=gen, device="cuda"))
        b = b * torch.where(torch.rand(b.shape, generator=gen, device="cuda") < 0.5, -1.0, 1.0)
        b[-1, 3:] = _randn(gen, 125)
        for x in (torch.cat([groups, b], dim=1), torch.cat([groups[:, 1:], b[:, 1:]], dim=1)):  # 16-byte accesses, and not
            x = x.to(dtype)
            _check_rows(ops.quantize_rows(x, gate=True), _gate_ref(x))
    _no_device_error()


@pytest.mark.parametrize("low", [-88.0, -20.0])
def test_gates_beside_ties_over_the_whole_range(low):
    """silu(a) b as near to ties between e4m3 values as b's 32 bits allow, for a of every size: the interval that sends a
    value to 64 bits has to hold what 32 bits get wrong anywhere."""
    from ctmr_b200 import ops

    gen = _gen(34)
    for _ in range(4):
        a = low + (30.0 - low) * torch.rand((4000, 256), generator=gen, device="cuda")
        a = torch.where(a.abs() < 1e-3, 1.0, a)
        target = (torch.randint(8, 16, a.shape, generator=gen, device="cuda") * 2 + 1).double() / 16
        b = (target * (1.0 + torch.exp(-a.double())) / a.double()).float()
        x = torch.cat([a, b], dim=1)
        _check_rows(ops.quantize_rows(x, gate=True), _gate_ref(x))
    _no_device_error()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gates_below_the_normal_numbers(dtype):
    """Subnormal a or b, times a large other half."""
    from ctmr_b200 import ops

    gen = _gen(32)
    small, large = _randn(gen, 2000, 128, std=1e-40), _randn(gen, 2000, 128, std=1e30)
    for x in (torch.cat([small, large], dim=1), torch.cat([large.abs(), small], dim=1)):
        x = x.to(dtype)
        _check_rows(ops.quantize_rows(x, gate=True), _gate_ref(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gates_past_32_bits(dtype):
    """Products above fp32's largest number, as far as a scale reaches (448 * 2^127); NaN beyond, and where a or b is
    not finite."""
    from ctmr_b200 import ops

    gen = _gen(33)
    a = 1e20 * (0.5 + 0.5 * torch.rand((40, 600), generator=gen, device="cuda"))
    b = torch.exp2(torch.linspace(40.0, 66.0, 40, device="cuda"))[:, None] * _randn(gen, 40, 600).clamp(-4, 4)
    b[::3, 10:] = _randn(gen, 14, 590)  # one or a few such values in a group
    x = torch.cat([a, b], dim=1).to(dtype)
    assert 3.5e38 < _gate_ref(x).abs().max() < 448 * 2.0 ** 127
    _check_rows(ops.quantize_rows(x, gate=True), _gate_ref(x))
    x[3, 130], x[3, 730] = 1e30, 1e30     # 1e60
    x[4, 260], x[4, 860] = -90.0, float("inf")
    x[5, 599] = -float("inf")             # an infinity over an infinity
    x[6, 0], x[6, 1] = -90.0, float("nan")
    got = ops.quantize_rows(x, gate=True)
    keep = [r for r in range(40) if r not in (3, 4, 5, 6)]
    _check_rows(ops.ScaledRows(got.values[keep], got.scale[keep]), _gate_ref(x)[keep])
    back = got.float()
    for row, group in ((3, 1), (4, 2), (5, 4), (6, 0)):
        bad = torch.isnan(back[row])
        assert bad[group * 128:(group + 1) * 128].all() and bad.sum() == min(128, 600 - group * 128)
        assert torch.isnan(got.scale[row]).sum() == 1


# ---------------------------------------------------------------------------------------------- norm
def _check(x, weight, residual, quantize, eps=1e-6, **kw):
    from ctmr_b200 import ops

    ref = _norm_ref(x, residual, weight, eps)
    total = None if residual is None else (x.float() + residual.float()).to(x.dtype)
    y = ops.rms_norm(x, weight, residual=residual, eps=eps, quantize=quantize, **kw)
    if residual is not None:
        y, h = y
        assert torch.equal(h, total)
    if quantize:
        _check_rows(y, ref)
    else:
        _within(y, ref, (U[x.dtype] + 2.0 ** -21) * ref.abs() + 2.0 ** -25)
    _no_device_error()


def _resident(channels):
    """Blocks of a row that are resident at once: 512 threads to an SM, 32 to 512 channels of the row each warp."""
    threads = ((channels + 127) // 128 + 3) // 4 * 32
    return torch.cuda.get_device_properties(0).multi_processor_count * (512 // threads)


# Blocks that go on from row to row (over several turns, the last one not full; with few rows of an odd width), two groups
# of channels to eight lanes of a warp, and a block to each row.
FORMS = [(2048, "3 turns"), (4096, "3 turns"), (1001, "1.5 turns"), (1000, "warps"), (1024, "warps"), (4097, "2 turns"),
         (4224, "2 turns")]


def _rows(channels, form):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    if form == "warps":
        return 16 * sms + 301
    return int(float(form.split()[0]) * _resident(channels)) + 77 * (form != "1.5 turns")


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(("channels", "form"), FORMS)
def test_norm_of_many_rows(channels, form, dtype, quantize):
    gen = _gen(channels)
    rows = _rows(channels, form)
    x, residual = _randn(gen, rows, channels, dtype=dtype, std=3.0), _randn(gen, rows, channels, dtype=dtype)
    weight = 1.0 + _randn(gen, channels, std=0.2)
    _check(x, weight, residual, quantize)
    _check(x, weight.to(dtype), None, quantize)
    _check(x, None, None, quantize)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("over", ["x", "residual", "y"])
def test_norm_of_many_rows_in_place(dtype, over):
    """The next row's loads are ahead of this row's stores: they are another row's."""
    gen = _gen(41)
    rows, channels = _rows(2048, "3 turns"), 2048
    weight = 1.0 + _randn(gen, channels, std=0.2)
    for quantize in (False, True):
        if over == "y" and quantize:
            continue
        x, residual = _randn(gen, rows, channels, dtype=dtype), _randn(gen, rows, channels, dtype=dtype)
        # (the reference is taken before the call)
        _check(x, weight, residual, quantize, **(dict(out=x) if over == "y" else dict(sum_out=x if over == "x" else residual)))


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_many_heads(dtype):
    """Heads of a fused projection, more than are resident at once, in both orders of rows."""
    from ctmr_b200 import ops

    gen = _gen(42)
    dim, heads = 2048, 5
    tokens = _resident(dim) * 2 // heads + 13
    weight = 1.0 + _randn(gen, dim, std=0.2)
    wide = _randn(gen, tokens, heads + 2, dim, dtype=dtype)
    before = wide.clone()
    view = wide[:, 1:1 + heads]
    ref = _norm_ref(view, None, weight, 1e-6)
    assert ops.rms_norm(view, weight, out=view) is view
    _within(view, ref, (U[dtype] + 2.0 ** -21) * ref.abs() + 2.0 ** -25)
    assert torch.equal(wide[:, :1], before[:, :1]) and torch.equal(wide[:, 1 + heads:], before[:, 1 + heads:])
    x, residual = _randn(gen, heads, tokens, dim, dtype=dtype).transpose(0, 1), before[:, :heads]
    _check(x, weight, residual, False)


def _near_ties(h, width, eps):
    """Weights that bring h / sqrt(mean(h^2) + eps) as near to ties between e4m3 values as 32 bits allow."""
    y = h / torch.sqrt(h.square().mean() + eps)
    return (((torch.arange(width, device="cuda") % 8 * 2 + 17) / 16).double() / torch.where(y == 0, 1.0, y)).float()


@pytest.mark.parametrize("channels", [128, 512, 1001, 2048, 9000])
def test_norm_keeps_what_the_sum_in_32_bits_cuts_off(channels):
    """fp32: a residual that the 32-bit sum loses, the same way in every channel: 64 bits of x + residual decide."""
    gen = _gen(51)
    eps = 2.0 ** -20  # (a number of fp32: it decides some of these rows alone)

    def check(x, residual):
        weight = _near_ties(x[0].double() + residual[0].double(), channels, eps)
        _check(x.expand(3, -1).contiguous(), weight, residual.expand(3, -1).contiguous(), True, eps)

    x = 1 + torch.randint(120, (1, channels), generator=gen, device="cuda") / 128
    for factor in (1.0, -1.0, 2.0 ** 60, 2.0 ** 120, 2.0 ** -18):
        check(x * abs(factor), torch.full_like(x, factor * 0.7 * 2.0 ** -24))
    # one such channel among ordinary ones, and the two tensors the other way round
    residual = _randn(gen, 1, channels)
    residual[0, channels // 3] = 2.0 ** -24
    check(x, residual)
    check(residual, x)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_not_finite_sums(dtype):
    """An infinity's own group is NaN, the rest of its row zero, whichever tensor it is in; a NaN's row is NaN."""
    from ctmr_b200 import ops

    gen = _gen(52)
    x, residual = _randn(gen, 6, 700, dtype=dtype), _randn(gen, 6, 700, dtype=dtype)
    good = ops.rms_norm(x, residual=residual, quantize=True)[0].float()
    x[1, 300], residual[2, 300], x[3, 5], residual[3, 5] = float("inf"), -float("inf"), float("inf"), 1.0
    x[4, 9] = float("nan")
    got = ops.rms_norm(x, residual=residual, quantize=True)[0].float()
    for row, start in ((1, 256), (2, 256), (3, 0)):
        inside = torch.zeros(700, dtype=torch.bool, device="cuda")
        inside[start:start + 128] = True
        assert torch.isnan(got[row, inside]).all() and (got[row, ~inside] == 0).all()
    assert torch.isnan(got[4]).all()
    assert torch.equal(got[[0, 5]], good[[0, 5]])


@pytest.mark.parametrize("channels", [128, 512, 1001, 2048, 9000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_of_16_bit_rows_is_of_the_sum_in_32_bits(dtype, channels):
    from ctmr_b200 import ops

    gen = _gen(53)
    eps = 2.0 ** -20
    x = (1 + torch.randint(120, (1, channels), generator=gen, device="cuda") / 128).to(dtype)
    one = _randn(gen, 1, channels, dtype=dtype)
    one[0, channels // 3] = 2.0 ** -24
    for residual in (torch.full_like(x, 2.0 ** -24), torch.full_like(x, -(2.0 ** -24)), one):
        h = (x.float() + residual.float()).double()
        weight = _near_ties(h[0], channels, eps)
        y, total = ops.rms_norm(x.expand(3, -1), weight, residual=residual.expand(3, -1), eps=eps, quantize=True)
        assert torch.equal(total, h.to(dtype).expand(3, -1))
        _check_rows(y, _norm_ref(h.expand(3, -1), None, weight, eps))


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("channels", [96, 512, 2048])
def test_norm_of_rows_near_the_largest_number(channels, dtype, quantize):
    """One over the root is below 32 bits' normal numbers, off by up to 2^-22: bytes are right but within 2^-20 of a tie."""
    from ctmr_b200 import ops

    x = ((torch.rand((3, channels), generator=_gen(61), device="cuda") * 2 - 1) * 3.3e38).to(dtype)
    ref = _norm_ref(x, None, None, 1e-6)
    y = ops.rms_norm(x, quantize=quantize)
    if quantize:
        _check_rows(y, ref, 2.0 ** -20)
    else:
        _within(y, ref, (U[dtype] + 2.0 ** -20) * ref.abs())
    _no_device_error()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_of_small_values_under_large_weights(dtype):
    """Groups far below their row's size, brought back by weights of 2^15."""
    gen = _gen(62)
    x = _randn(gen, 20, 640)
    x[:, 128:] *= torch.exp2(torch.linspace(-90.0, -132.0, 20, device="cuda"))[:, None]
    weight = torch.where(_randn(gen, 640) > 0, 2.0 ** 15, -(2.0 ** 15))
    _check(x.to(dtype), weight, None, True)
    _check(x.to(dtype), weight, torch.zeros_like(x, dtype=dtype), True)


def test_outputs_over_themselves_are_refused():
    """Expanded tensors as outputs: x or residual itself, or one of the caller's."""
    from ctmr_b200 import ops

    gen = _gen(71)
    x, one = _randn(gen, 6, 256), _randn(gen, 1, 256).expand(6, -1)
    heads = _randn(gen, 6, 1, 256).expand(-1, 4, -1)
    for call in (lambda: ops.rms_norm(x, residual=one, sum_out=one),
                 lambda: ops.rms_norm(one, residual=x, sum_out=one),
                 lambda: ops.rms_norm(one, out=one),
                 lambda: ops.rms_norm(x, out=torch.empty(128 * 5 + 256, device="cuda").as_strided((6, 256), (128, 1))),
                 lambda: ops.rms_norm(heads, out=heads)):
        with pytest.raises(ValueError, match="overlap"):
            call()
    # as inputs they are fine, and one row or head may have any stride
    _check(one, None, one, True)
    _check(heads, None, heads, False)
    y = torch.empty((1, 256), device="cuda").expand(1, -1)
    assert ops.rms_norm(one[:1], out=y) is y


# ---------------------------------------------------------------------------------------------- product
@pytest.mark.parametrize(("rows", "inner", "outer"), [(1, 11264, 512), (16, 4096, 300), (32, 1024, 1536), (100, 2000, 512),
                                                      (128, 4096, 384), (617, 512, 1536), (1500, 4096, 777), (2300, 11264, 512)])
@pytest.mark.parametrize("bias", [False, True])
def test_products_are_summed_in_32_bits(rows, inner, outer, bias):
    from ctmr_b200 import ops

    gen = _gen(rows + inner + outer)
    x, w = _rows8(gen, rows, inner), _weight8(gen, outer, inner)
    bias = _randn(gen, outer, std=0.5) if bias else None
    ref, _ = _linear_ref(x, w, bias)
    err = ops.scaled_linear(x, w, bias, out_dtype=torch.float32).double() - ref
    bound = 2.0 ** -24 * (((inner + 127) // 128 / 2 + 10) ** 0.5 + (bias is not None))
    assert err.norm() <= bound * ref.norm()
    for dim in (0, 1):
        # (a line's products are as large as x's and w's; its sums may have come out small)
        size = torch.linalg.vector_norm(ref, dim=dim)
        usual = ref.norm() / ref.numel() ** 0.5 * ref.shape[dim] ** 0.5
        assert (torch.linalg.vector_norm(err, dim=dim) <= 2 * bound * torch.maximum(size, usual)).all()
    _no_device_error()
