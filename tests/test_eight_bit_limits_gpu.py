"""The 8-bit row operators at the edges of what they accept and in every form that their launchers choose, against plain
implementations in 64 bits.

Tolerances. 8-bit rows as in test_eight_bit_gpu, the bytes those of the 64-bit formula everywhere:
``step / 2 + 2^-40 |v|``.
"""

from __future__ import annotations

import pytest
import torch
from test_eight_bit_gpu import TYPES, _check_rows, _gate_ref, _gen, _no_device_error, _randn

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
