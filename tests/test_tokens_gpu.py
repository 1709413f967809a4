"""The packed-token operators (``rotary_axes``, ``adapter_linear``, ``attention``) against plain
implementations in 64 bits.

Tolerances follow from the operators' roundings. With u the half-ulp of the output's type (2^-p for a significand of p bits:
bf16 2^-8, fp16 2^-11, fp32 2^-24):

* rotary: one rounding of the result, and two fp32 products and a sum of them with a sine and cosine
  correct to a few 2^-24: ``u |y| + 8 * 2^-24 (|a| + |b|)``;
* adapter_linear: one rounding of y, the adapter's inner product rounded once to the operands' type, and
  fp32 sums of n products: ``u |y| + u scale sum |t||up| + 2^-23 sqrt(n) sum |x||w|``;
* attention: one rounding of the output and one of each softmax weight (the weights' sum is taken before
  it), exponentials good to 1e-4 (below a quarter of fp16's half-ulp), fp32 scores of size S: with
  a = sum softmax |v|, ``u |out| + (1.25 u + 2e-5 + 2^-21 S) a``; the log-sum-exp is off by the
  exponentials' error and the score's rounding: ``1e-4 + 2^-21 S``.
fp16 results below the smallest normal number round in steps of 2^-24, so 2^-25 is always allowed.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
HALF = [torch.bfloat16, torch.float16]


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float16, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def _offsets(lengths):
    return torch.tensor([0, *lengths]).cumsum(0).to(device="cuda", dtype=torch.int32)


def _within(got, ref, tol):
    got = got.double()
    assert torch.isfinite(got).all()
    over = ((got - ref).abs() - tol).max().item() if got.numel() else 0.0
    assert over <= 0.0, f"{over:.3e} over the tolerance; error {(got - ref).abs().max().item():.3e}"


def _no_device_error():
    from ctmr_b200 import _lib

    assert _lib.device_error(clear=True) == 0


# ---------------------------------------------------------------------------------------------- rotary
def _rotary_ref(x, positions, inv_freq, sections, interleaved, inverse):
    x, pairs = x.double(), sum(sections)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(x.device)
    angle = (positions.double()[:, axis] * inv_freq.double())[:, None, :]
    cos, sin = torch.cos(angle), torch.sin(angle) * (-1.0 if inverse else 1.0)
    y = x.clone()
    first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    mag = torch.zeros_like(x)
    mag[..., first] = mag[..., second] = a.abs() + b.abs()
    return y, mag


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize(("tokens", "heads", "dim", "sections", "interleaved"), [
    (1, 1, 2, (1,), False),            # one token, one pair
    (1, 8, 128, (16, 24, 24), True),
    (105, 16, 32, (4, 6, 6), False),
    (77, 3, 72, (10, 11, 11), False),  # pairs that no vector divides, 8 channels copied
    (77, 3, 72, (10, 11, 11), True),
    (33, 5, 40, (4, 0, 8), False),     # an axis without pairs, half of the head copied
    (33, 5, 40, (4, 0, 8), True),
    (257, 2, 7, (2, 1), False),        # odd head size
    (257, 2, 7, (2, 1), True),
    (4099, 7, 160, (30, 30, 20), False),
    (50, 300, 64, (32,), True),        # many heads: fewer tokens a block
    (9, 2, 4096, (2000, 48), False),   # the widest head
])
def test_rotary_axes(cuda, dtype, tokens, heads, dim, sections, interleaved):
    from ctmr_b200 import ops

    gen = _gen(tokens + dim)
    x = _randn(gen, tokens, heads, dim, dtype=dtype)
    positions = torch.randint(-40, 500, (tokens, len(sections)), generator=gen, device="cuda", dtype=torch.int32)
    inv_freq = ops.axis_frequencies(sections)
    for inverse in (False, True):
        y = ops.rotary_axes(x, positions, inv_freq, sections, interleaved=interleaved, inverse=inverse)
        ref, mag = _rotary_ref(x, positions, inv_freq, sections, interleaved, inverse)
        _within(y, ref, U[dtype] * ref.abs() + 8 * 2.0 ** -24 * mag + 2.0 ** -25 * (dtype == torch.float16))
        assert torch.equal(y[..., 2 * sum(sections):], x[..., 2 * sum(sections):])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotary_views_in_place_and_large_positions(cuda, dtype, interleaved):
    """Query and key heads of a fused projection in place, at odd element offsets too, with fractional
    positions as large as 2e6 (an fp32 product would lose the angle)."""
    from ctmr_b200 import ops

    gen, sections = _gen(5), (10, 12)
    inv_freq = ops.axis_frequencies(sections)
    positions = torch.rand((60, 3), generator=gen, device="cuda")[:, :2] * 2e6  # rows 3 elements apart
    for start, width in ((0, 144), (1, 145), (2, 146), (4, 152)):
        base = _randn(gen, 60, width * 6 + 8, dtype=dtype)
        keep = base.clone()
        view = base[:, start:start + width * 4].unflatten(1, (4, width))[..., :48]
        ref, mag = _rotary_ref(view, positions, inv_freq, sections, interleaved, False)
        assert ops.rotary_axes(view, positions, inv_freq, sections, interleaved=interleaved, out=view) is view
        _within(view, ref, U[dtype] * ref.abs() + 8 * 2.0 ** -24 * mag)
        view.copy_(keep[:, start:start + width * 4].unflatten(1, (4, width))[..., :48])
        assert torch.equal(base, keep)  # nothing beside the view was written


def test_rotary_inverse_is_the_gradient(cuda):
    """The inverse applied to an output's gradient is the gradient of the plain rotation, by autograd and by
    differences in 64 bits."""
    from ctmr_b200 import ops

    gen, sections = _gen(11), (5, 7)
    x, g = _randn(gen, 40, 3, 32, dtype=torch.float32), _randn(gen, 40, 3, 32, dtype=torch.float32)
    positions = torch.randint(0, 300, (40, 2), generator=gen, device="cuda", dtype=torch.int32)
    inv_freq = ops.axis_frequencies(sections)
    got = ops.rotary_axes(g, positions, inv_freq, sections, inverse=True)
    ref, mag = _rotary_ref(g, positions, inv_freq, sections, False, True)
    _within(got, ref, U[torch.float32] * ref.abs() + 8 * 2.0 ** -24 * mag)
    direction = _randn(gen, 40, 3, 32, dtype=torch.float32).double()
    loss = lambda t: (_rotary_ref(t, positions, inv_freq, sections, False, False)[0] * g.double()).sum()  # noqa: E731
    diff = (loss(x.double() + 1e-3 * direction) - loss(x.double() - 1e-3 * direction)) / 2e-3
    # the operator is linear: the difference is exact up to fp64, the kernel's sum of 3840 terms to fp32
    assert abs(diff.item() - (got.double() * direction).sum().item()) <= 1e-5 * (got.double() * direction).abs().sum().item()


def test_rotary_copies_infinities_past_the_pairs(cuda):
    from ctmr_b200 import ops

    x = torch.full((3, 2, 16), math.inf, device="cuda", dtype=torch.float16)
    x[..., :6] = 1.0
    positions = torch.arange(3, device="cuda", dtype=torch.int32)[:, None]
    for interleaved in (False, True):
        y = ops.rotary_axes(x, positions, ops.axis_frequencies((3,)), (3,), interleaved=interleaved)
        assert torch.isinf(y[..., 6:]).all() and torch.isfinite(y[..., :6]).all()
    assert ops.rotary_axes(x[:0], positions[:0], ops.axis_frequencies((3,)), (3,)).shape == (0, 2, 16)


def test_rotary_refusals(cuda):
    from ctmr_b200 import ops

    x = torch.zeros((4, 2, 16), device="cuda", dtype=torch.float16)
    pos = torch.zeros((4, 2), device="cuda", dtype=torch.int32)
    f = ops.axis_frequencies((3, 4))
    bad = [
        dict(x=x.cpu()), dict(x=x.double()), dict(x=x[0]), dict(positions=pos.long()), dict(positions=pos[:3]),
        dict(sections=(3, 5)), dict(sections=(8, 8), inv_freq=ops.axis_frequencies((8, 8))), dict(sections=()),
        dict(sections=(-1, 8)), dict(inv_freq=f.double()), dict(out=torch.empty_like(x, dtype=torch.bfloat16)),
        dict(x=x.transpose(1, 2), sections=(1, 0), inv_freq=f[:1]),
    ]
    for change in bad:
        a = {**dict(x=x, positions=pos, inv_freq=f, sections=(3, 4), out=None), **change}
        with pytest.raises(ValueError):
            ops.rotary_axes(a["x"], a["positions"], a["inv_freq"], a["sections"], out=a["out"])


# ---------------------------------------------------------------------------------------------- linear
def _linear_case(seed, lengths, index, inner, outer, rank, adapters, dtype):
    gen, rows = _gen(seed), sum(lengths)
    return dict(
        x=_randn(gen, rows, inner, dtype=dtype), weight=_randn(gen, outer, inner, dtype=dtype, std=inner ** -0.5),
        bias=_randn(gen, outer, dtype=dtype), down=_randn(gen, adapters, rank, inner, dtype=dtype, std=inner ** -0.5),
        up=_randn(gen, adapters, outer, rank, dtype=dtype, std=rank ** -0.5),
        scale=0.25 + torch.rand(adapters, generator=gen, device="cuda"), offsets=_offsets(lengths),
        index=torch.tensor(index, device="cuda", dtype=torch.int32))


def _linear_ref(c):
    x, w = c["x"].double(), c["weight"].double()
    u = U[c["x"].dtype]
    y, slack = x @ w.T, 2.0 ** -23 * x.shape[1] ** 0.5 * (x.abs() @ w.abs().T)
    if c["bias"] is not None:
        y += c["bias"].double()
    o = c["offsets"].tolist()
    for s, a in enumerate(c["index"].tolist()):
        if a < 0:
            continue
        rows = slice(o[s], o[s + 1])
        d, up, scale = c["down"][a].double(), c["up"][a].double(), c["scale"][a].double()
        t = scale * (x[rows] @ d.T)
        y[rows] += t @ up.T
        slack[rows] += (u * t.abs() + 2.0 ** -23 * x.shape[1] ** 0.5 * scale * (x[rows].abs() @ d.abs().T)) @ up.abs().T
    return y, u * y.abs() + slack + 2.0 ** -25


LINEAR = [  # lengths, index, inner, outer, rank, adapters
    ([1], [0], 8, 1, 8, 1),                       # one row, one output
    ([1], [-1], 64, 130, 8, 2),                   # no adapter
    ([3], [1], 4096, 512, 128, 2),                # the largest rank, a long sum
    ([1] * 17, [i % 4 - 1 for i in range(17)], 256, 384, 16, 3),
    ([1] * 64, [63 - i for i in range(64)], 136, 257, 24, 64),   # every row its own adapter, odd output
    ([5, 0, 11, 0, 0, 40], [0, 1, -1, 2, 0, 1], 72, 200, 8, 3),  # empty segments
    ([127, 1, 128, 129, 2], [2, 0, 1, -1, 2], 512, 1536, 40, 3),
    ([300, 213], [1, 0], 520, 1000, 64, 2),
    ([700, 1, 324], [0, 2, 1], 200, 333, 16, 3),
    ([1500, 548, 3], [-1, 0, 1], 1024, 768, 32, 2),
    ([0, 2000, 0], [0, 1, 0], 1032, 515, 72, 2),
    (list(range(40)), [(5 * i) % 7 - 1 for i in range(40)], 320, 640, 16, 6),
    # enough 256 x 256 tiles for the CTA pairs: an adapter border inside a tile, a last tile of two rows,
    # many short segments, the largest rank over a short sum
    ([1000, 1, 0, 1305], [2, 0, 1, 1], 136, 2310, 24, 3),
    ([61] * 39, [(3 * i) % 8 - 1 for i in range(39)], 520, 2500, 8, 7),
    ([2500, 2500], [1, 0], 64, 1100, 128, 2),
]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("case", range(len(LINEAR)))
def test_adapter_linear(cuda, case, dtype):
    from ctmr_b200 import ops

    lengths, index, inner, outer, rank, adapters = LINEAR[case]
    c = _linear_case(case, lengths, index, inner, outer, rank, adapters, dtype)
    for bias in (c["bias"], c["bias"].float(), None):
        c["bias"] = bias
        _within(ops.adapter_linear(**c), *_linear_ref(c))
    _no_device_error()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows", [1, 2, 31, 100, 513, 2300, 10007])
def test_linear_without_adapters(cuda, rows, dtype):
    from ctmr_b200 import ops

    c = _linear_case(rows, [rows], [-1], 264, 300 if rows < 10000 else 601, 8, 1, dtype)
    _within(ops.adapter_linear(c["x"], c["weight"], c["bias"]), *_linear_ref(c))


@pytest.mark.parametrize("rows", [3, 40, 600])
def test_adapter_linear_views(cuda, rows):
    """Rows of wider tensors as input, weight and output; nothing beside the output is written; the same
    answer on another stream."""
    from ctmr_b200 import ops

    c = _linear_case(rows, [rows // 2, rows - rows // 2], [1, 0], 96, 203, 16, 2, torch.float16)
    c["x"] = torch.cat((torch.full_like(c["x"], math.nan), c["x"], torch.full_like(c["x"], math.inf)), 1)[:, 96:192]
    c["weight"] = torch.cat((c["weight"], torch.full_like(c["weight"], math.nan)), 1)[:, :96]
    wide = torch.full((rows, 407), 7.0, device="cuda", dtype=torch.float16)
    out = ops.adapter_linear(**c, out=wide[:, 101:304])
    _within(out, *_linear_ref(c))
    assert (wide[:, :101] == 7).all() and (wide[:, 304:] == 7).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.adapter_linear(**c)
    side.synchronize()
    assert torch.equal(other, out)


def test_adapter_linear_rows_outside_and_bad_numbers(cuda):
    """Rows that no segment holds get the projection alone, and so do rows whose adapter does not exist; the
    latter, and offsets past the rows, are reported in the device error word."""
    from ctmr_b200 import _lib, ops

    c = _linear_case(3, [10, 30], [0, 1], 64, 96, 8, 2, torch.float16)
    c["offsets"] = torch.tensor([4, 10, 33], device="cuda", dtype=torch.int32)
    _within(ops.adapter_linear(**c), *_linear_ref(c))
    _no_device_error()
    c["index"] = torch.tensor([0, 2], device="cuda", dtype=torch.int32)
    y = ops.adapter_linear(**c)
    assert _lib.device_error(clear=True) == 32
    c["index"] = torch.tensor([0, -1], device="cuda", dtype=torch.int32)
    _within(y, *_linear_ref(c))
    c["offsets"] = torch.tensor([4, 10, 2000], device="cuda", dtype=torch.int32)
    c["index"] = torch.tensor([0, 1], device="cuda", dtype=torch.int32)
    y = ops.adapter_linear(**c)
    assert _lib.device_error(clear=True) == 32
    c["offsets"] = torch.tensor([4, 10, 40], device="cuda", dtype=torch.int32)
    _within(y, *_linear_ref(c))


def test_stack_adapters_pads_ranks(cuda):
    from ctmr_b200 import ops

    gen = _gen(9)
    loose = [(_randn(gen, r, 64), _randn(gen, 72, r), 0.5 + r) for r in (3, 12, 1)]
    stacked = ops.stack_adapters(loose, dtype=torch.float16)
    assert stacked["down"].shape == (3, 16, 64) and stacked["up"].shape == (3, 72, 16)
    x, w = _randn(gen, 9, 64), _randn(gen, 72, 64)
    index = torch.tensor([2, 0, 1], device="cuda", dtype=torch.int32)
    c = dict(x=x, weight=w, bias=None, **stacked, offsets=_offsets([2, 3, 4]), index=index)
    _within(ops.adapter_linear(**c), *_linear_ref(c))
    with pytest.raises(ValueError):
        ops.stack_adapters([loose[0], (loose[1][0][:, :32], loose[1][1], 1.0)], dtype=torch.float16)


def test_adapter_linear_refusals(cuda):
    from ctmr_b200 import ops

    c = _linear_case(1, [4, 4], [0, 1], 64, 48, 8, 2, torch.float16)
    bad = [
        dict(x=c["x"].cpu()), dict(x=c["x"].float()), dict(weight=c["weight"].bfloat16()), dict(weight=c["weight"][:, :56]),
        dict(bias=c["bias"][:5]), dict(bias=c["bias"].double()), dict(down=None), dict(down=c["down"][:, :4]),
        dict(down=c["down"][:, :4], up=c["up"][:, :, :4]), dict(scale=c["scale"].double()),
        dict(offsets=c["offsets"].long()), dict(offsets=c["offsets"][:2]), dict(index=c["index"].cpu()),
        dict(x=c["x"][:, ::2], weight=c["weight"][:, :32], down=c["down"][..., :32]),
        dict(out=torch.empty((8, 47), device="cuda", dtype=torch.float16)),
    ]
    for change in bad:
        with pytest.raises(ValueError):
            ops.adapter_linear(**{**c, **change})
    odd = _linear_case(1, [8], [0], 64, 48, 8, 1, torch.float16)
    for inner in (60, 63):
        with pytest.raises(ValueError):  # not a multiple of 8
            ops.adapter_linear(odd["x"][:, :inner].contiguous(), odd["weight"][:, :inner].contiguous())
    assert ops.adapter_linear(c["x"][:0], c["weight"]).shape == (0, 48)


# ---------------------------------------------------------------------------------------------- attention
def _document_ref(q, k, v, scale, cap, slopes, causal, prefix):
    """q (Lq, H, D), k and v (Lk, H, D) in 64 bits -> out, lse, sum of softmax |v|, largest |score|."""
    lq, lk = q.shape[0], k.shape[0]
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    if not lq or not lk:
        return out, lse, mag, 0.0
    s = torch.einsum("ihd,jhd->hij", q, k) * scale
    size = s.abs().max().item()
    if cap:
        s = cap * torch.tanh(s / cap)
    place = torch.arange(lq, device=q.device)[:, None] + lk - lq
    key = torch.arange(lk, device=q.device)[None, :]
    if slopes is not None:
        s = s - slopes.double()[:, None, None] * (place - key).abs()
    seen = ((key <= place) | (key < prefix)) if causal else torch.ones((lq, lk), dtype=torch.bool, device=q.device)
    some = seen.any(1)
    s = s.masked_fill(~seen, -math.inf)[:, some]
    size = max(size, torch.where(torch.isinf(s), torch.zeros_like(s), s).abs().max().item() if some.any() else 0.0)
    p = torch.softmax(s, dim=-1)
    out[some] = torch.einsum("hij,jhd->ihd", p, v)
    mag[some] = torch.einsum("hij,jhd->ihd", p, v.abs())
    lse[some] = torch.logsumexp(s, dim=-1).T
    return out, lse, mag, size


def _check_attention(out, lse, parts, dtype):
    """parts: per document (rows of out, rows of lse, reference)."""
    for o, m, (ref, ref_lse, mag, size) in parts:
        _within(o, ref, U[dtype] * ref.abs() + (1.25 * U[dtype] + 2e-5 + 2.0 ** -21 * size) * mag + 2.0 ** -25)
        if m is not None:
            empty = torch.isinf(ref_lse)
            assert torch.equal(torch.isinf(m) & (m < 0), empty)
            assert (o[empty] == 0).all()
            _within(m[~empty], ref_lse[~empty], torch.full_like(ref_lse[~empty], 1e-4 + 2.0 ** -21 * size))


def _packed(seed, q_len, k_len, heads, kv_heads, dim, dtype, **kw):
    gen = _gen(seed)
    fused = k_len is None
    k_len = q_len if fused else k_len
    if fused:
        rows = _randn(gen, sum(q_len), heads + 2 * kv_heads, dim, dtype=dtype)
        q, k, v = rows.split((heads, kv_heads, kv_heads), dim=1)
    else:
        q = _randn(gen, sum(q_len), heads, dim, dtype=dtype)
        k, v = (_randn(gen, sum(k_len), kv_heads, dim, dtype=dtype) for _ in range(2))
    return q, k, v, _offsets(q_len), _offsets(k_len)


def _run_packed(q, k, v, qo, ko, dtype, *, scale=None, cap=0.0, slopes=None, causal=False, prefix=None, **kw):
    from ctmr_b200 import ops

    out, lse = ops.attention(q, k, v, q_offsets=qo, k_offsets=ko, scale=scale, cap=cap, slopes=slopes, causal=causal,
                             prefix=prefix, return_lse=True, **kw)
    plain = ops.attention(q, k, v, q_offsets=qo, k_offsets=ko, scale=scale, cap=cap, slopes=slopes, causal=causal,
                          prefix=prefix, **kw)
    assert torch.equal(plain, out)
    heads = torch.arange(q.shape[1], device="cuda") // (q.shape[1] // k.shape[1])
    qo, ko = qo.tolist(), ko.tolist()
    pre = prefix.tolist() if prefix is not None else [0] * (len(qo) - 1)
    parts = []
    for d in range(len(qo) - 1):
        a, b = slice(qo[d], qo[d + 1]), slice(ko[d], ko[d + 1])
        ref = _document_ref(q[a].double(), k[b].double()[:, heads], v[b].double()[:, heads],
                            q.shape[-1] ** -0.5 if scale is None else scale, cap, slopes, causal, pre[d])
        parts.append((out[a], lse[a], ref))
    _check_attention(out, lse, parts, dtype)
    _no_device_error()
    return out


PACKED = [  # query lengths, key lengths or None, heads, kv_heads, dim
    ([1], None, 1, 1, 8),
    ([1, 1, 1], [5, 0, 300], 4, 2, 64),
    ([127, 128, 129], None, 2, 2, 32),
    ([255, 1, 257, 0, 300], None, 3, 3, 64),
    ([130, 400], [700, 129], 4, 1, 128),
    ([64, 0, 200], [0, 50, 128], 2, 1, 40),
    ([513], None, 6, 2, 72),
    ([100, 90], [3, 1000], 8, 1, 104),
    ([17] * 40, None, 2, 2, 24),
    ([1000, 24], None, 2, 1, 120),
    ([385, 640, 3], [640, 385, 1], 2, 2, 80),
    ([600, 700], None, 2, 1, 48),
    ([7, 1, 30, 2], [900, 64, 31, 513], 8, 2, 96),
]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("mode", ["plain", "causal", "prefix", "cap", "bias", "all"])
@pytest.mark.parametrize("case", range(len(PACKED)))
def test_attention_packed(cuda, case, mode, dtype):
    q_len, k_len, heads, kv_heads, dim = PACKED[case]
    q, k, v, qo, ko = _packed(case, q_len, k_len, heads, kv_heads, dim, dtype)
    kw: dict = {}
    if mode in ("causal", "prefix", "all"):
        kw["causal"] = True
    if mode in ("prefix", "all"):
        lens = k_len or q_len
        kw["prefix"] = torch.tensor([(0, n // 2, n, n + 3, 1)[i % 5] for i, n in enumerate(lens)], device="cuda",
                                    dtype=torch.int32)
    if mode in ("cap", "all"):
        kw["cap"], kw["scale"] = 5.0, 2.0 * dim ** -0.5
    if mode in ("bias", "all"):
        kw["slopes"] = torch.exp2(-torch.arange(heads, device="cuda", dtype=torch.float32)) * 0.3
    _run_packed(q, k, v, qo, ko, dtype, **kw)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dim", range(8, 129, 8))
def test_attention_every_head_size(cuda, dim, dtype):
    q, k, v, qo, ko = _packed(dim, [200, 90], None, 2, 1, dim, dtype)
    _run_packed(q, k, v, qo, ko, dtype, causal=dim % 16 == 0)


@pytest.mark.parametrize("dtype", HALF)
def test_attention_growing_and_shrinking_scores(cuda, dtype):
    """Row maxima that keep growing along the keys (every tile rescales), that are largest first, and that are
    far below zero everywhere; scores of several hundred."""
    for seed, ramp in enumerate((torch.linspace(0.1, 24, 1200), torch.linspace(24, 0.1, 1200))):
        q, k, v, qo, ko = _packed(seed, [1200], [1200], 2, 2, 64, dtype)
        q.abs_().clamp_(0.5, 2.0)
        k.copy_((k.abs().clamp(0.5, 1.0) * ramp.to("cuda")[:, None, None]).to(dtype))
        _run_packed(q, k, v, qo, ko, dtype)
        _run_packed(q, -k, v, qo, ko, dtype, causal=True)


@pytest.mark.parametrize("dtype", HALF)
def test_attention_neighbours_are_never_read(cuda, dtype):
    """NaN and infinities in other documents' rows, beside the views and past the used keys change nothing."""
    gen = _gen(77)
    q_len, k_len = [70, 50, 200], [70, 300, 129]
    q, k, v, qo, ko = _packed(3, q_len, k_len, 4, 2, 64, dtype)
    wide = [torch.full((t.shape[0], t.shape[1] * 2 + 1, 72), math.nan, device="cuda", dtype=dtype) for t in (q, k, v)]
    views = []
    for w, t in zip(wide, (q, k, v)):
        view = w[:, 1::2, :64]
        view.copy_(t)
        views.append(view)
    base = _run_packed(q, k, v, qo, ko, dtype, causal=True)
    same = _run_packed(*views, qo, ko, dtype, causal=True)
    assert torch.equal(base, same)
    from ctmr_b200 import ops

    k[70:370], v[70:370] = math.nan, math.inf  # the middle document is poisoned: the others must not notice
    for kw in (dict(causal=True), dict(), dict(cap=3.0, slopes=torch.rand(4, generator=gen, device="cuda"))):
        out = ops.attention(q, k, v, q_offsets=qo, k_offsets=ko, **kw)
        k2, v2 = k.clone(), v.clone()
        k2[70:370], v2[70:370] = 0.0, 0.0
        clean = ops.attention(q, k2, v2, q_offsets=qo, k_offsets=ko, **kw)
        assert torch.isfinite(out[:70]).all() and torch.isfinite(out[120:]).all()
        assert torch.equal(out[:70], clean[:70]) and torch.equal(out[120:], clean[120:])


def _run_batched(seed, batch, lq, lk, heads, kv_heads, dim, dtype, lengths=None, poison=True, **kw):
    from ctmr_b200 import ops

    gen = _gen(seed)
    q = _randn(gen, batch, lq, heads, dim, dtype=dtype)
    k, v = (_randn(gen, batch, lk, kv_heads, dim, dtype=dtype) for _ in range(2))
    kl = None
    if lengths is not None:
        kl = torch.tensor(lengths, device="cuda", dtype=torch.int32)
        for b, n in enumerate(lengths):
            if poison:
                k[b, n:], v[b, n:] = math.nan, math.inf
    out, lse = ops.attention(q, k, v, k_lengths=kl, return_lse=True, **kw)
    group = torch.arange(heads, device="cuda") // (heads // kv_heads)
    parts = []
    for b in range(batch):
        n = lk if lengths is None else lengths[b]
        pre = kw["prefix"][b].item() if kw.get("prefix") is not None else 0
        ref = _document_ref(q[b].double(), k[b, :n].double()[:, group], v[b, :n].double()[:, group],
                            kw.get("scale") or dim ** -0.5, kw.get("cap", 0.0), kw.get("slopes"),
                            kw.get("causal", False), pre)
        parts.append((out[b], lse[b], ref))
    _check_attention(out, lse, parts, dtype)
    _no_device_error()
    return out


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(("batch", "lq", "lk", "heads", "kv_heads", "dim", "lengths"), [
    (1, 1, 1, 1, 1, 8, None),
    (1, 1, 300, 8, 8, 64, [300]),
    (3, 1, 1000, 8, 2, 128, [1000, 1, 513]),
    (2, 1, 64, 5, 1, 80, [0, 63]),              # an empty cache
    (4, 2, 700, 16, 2, 64, [700, 2, 1, 333]),   # fewer keys than queries: rows that see nothing
    (2, 5, 4100, 8, 4, 32, [4100, 4097]),
    (1, 3, 9000, 24, 3, 120, [8999]),
    (2, 1, 40, 64, 2, 72, [40, 17]),            # 32 query heads to a key head
    (1, 7, 500, 16, 1, 104, [450]),             # 112 rows to a key head
    (2, 130, 300, 4, 2, 64, [300, 129]),
    (2, 300, 200, 2, 2, 40, [200, 77]),
    (300, 1, 33, 2, 1, 16, [i % 34 for i in range(300)]),  # many requests
])
def test_attention_cache(cuda, batch, lq, lk, heads, kv_heads, dim, lengths, dtype):
    slopes = torch.exp2(-torch.arange(heads, device="cuda", dtype=torch.float32) / 4) * 0.1
    for kw in (dict(causal=True), dict(), dict(causal=True, cap=4.0, slopes=slopes),
               dict(causal=True, prefix=torch.full((batch,), 9, device="cuda", dtype=torch.int32))):
        _run_batched(lk + lq, batch, lq, lk, heads, kv_heads, dim, dtype, lengths, **kw)


def test_attention_batched_strides_streams_and_max_q(cuda):
    """Batched views with their own document strides; the packed form with a bound on the queries equals the
    one without; a side stream gives the same bits."""
    from ctmr_b200 import ops

    gen = _gen(21)
    store = _randn(gen, 3, 2, 260, 4, 64)  # K and V of one allocation, token rows of 4 heads
    k, v = store[:, 0, :250], store[:, 1, :250]
    q = _randn(gen, 3, 8, 64)[:, None]      # (3, 1, 8, 64)
    lengths = torch.tensor([250, 3, 111], device="cuda", dtype=torch.int32)
    out = ops.attention(q, k, v, k_lengths=lengths, causal=True)
    dense = ops.attention(q.contiguous(), k.contiguous(), v.contiguous(), k_lengths=lengths, causal=True)
    assert torch.equal(out, dense)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.attention(q, k, v, k_lengths=lengths, causal=True)
    side.synchronize()
    assert torch.equal(other, out)
    packed_k, packed_v = (torch.cat([t[b, :n] for b, n in enumerate(lengths.tolist())]) for t in (k, v))
    q_one, ko = q[:, 0], _offsets(lengths.tolist())
    qo = _offsets([1, 1, 1])
    few = _run_packed(q_one, packed_k, packed_v, qo, ko, torch.float16, causal=True, max_q=1)
    more = _run_packed(q_one, packed_k, packed_v, qo, ko, torch.float16, causal=True)
    assert (few.float() - more.float()).abs().max() <= 4e-3 and few.shape == out[:, 0].shape


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_attention_log_sum_exp_is_fp32(cuda, cap, dtype):
    """The log-sum-exp is a sum of fp32 terms, not of the 16-bit softmax weights: exponentials good to 3e-6, a
    quarter of them with an error of either sign (0.7e-6 of the sum at worst), scores of size S < 8 (with the
    cap's 2e-7 S) rounded by 2^-22 S, and the logarithm's own 2^-23."""
    from ctmr_b200 import ops

    q, k, v, qo, ko = _packed(8, [700, 333], None, 4, 2, 96, dtype)
    _, lse = ops.attention(q, k, v, q_offsets=qo, cap=cap, return_lse=True)
    heads = torch.arange(4, device="cuda") // 2
    for a, b in ((0, 700), (700, 1033)):
        _, ref, _, size = _document_ref(q[a:b].double(), k[a:b].double()[:, heads], v[a:b].double()[:, heads],
                                        96 ** -0.5, cap, None, False, 0)
        _within(lse[a:b], ref, 1e-6 + (2.0 ** -22 + 2e-7) * size + 2.0 ** -22 * ref.abs())


@pytest.mark.parametrize("lq", [1, 150])
def test_attention_offsets_past_32_bits(cuda, lq):
    """Keys and values more than 2^31 elements into their tensor (the last tokens of the second request of a
    cache whose token rows are 16 KB apart)."""
    from ctmr_b200 import ops

    gen, tokens, used = _gen(31), 140_000, 300
    store = torch.empty((2, tokens, 64, 128), device="cuda", dtype=torch.bfloat16)  # 4.6 GB, two heads of 64 used
    assert store[1, tokens - used].data_ptr() - store.data_ptr() > 2 * 2 ** 31
    k, v = store[:, :, :1], store[:, :, 63:]
    part = store[:, tokens - used:]
    part[:, :, :1] = _randn(gen, 2, used, 1, 128, dtype=torch.bfloat16)
    part[:, :, 63:] = _randn(gen, 2, used, 1, 128, dtype=torch.bfloat16)
    q = _randn(gen, 2, lq, 1, 128, dtype=torch.bfloat16)
    out = ops.attention(q, k[:, tokens - used:], v[:, tokens - used:])
    rows = ops.attention(q[1], store.view(-1, 64, 128)[:, :1], store.view(-1, 64, 128)[:, 63:],
                         q_offsets=_offsets([0, lq]), k_offsets=torch.tensor([0, 2 * tokens - used, 2 * tokens],
                                                                             device="cuda", dtype=torch.int32))
    for b in range(2):
        ref = _document_ref(q[b].double(), part[b, :, :1].double(), part[b, :, 63:].double(), 128 ** -0.5, 0.0, None,
                            False, 0)
        _check_attention(out[b], None, [(out[b], None, ref)], torch.bfloat16)
    _check_attention(rows, None, [(rows, None, ref)], torch.bfloat16)
    _no_device_error()


def test_adapter_linear_offsets_past_32_bits(cuda):
    """Rows more than 2^31 elements into x and y."""
    from ctmr_b200 import ops

    c = _linear_case(6, [64, 36], [1, 0], 64, 72, 8, 2, torch.float16)
    wide = torch.empty((100, 24_000_000), device="cuda", dtype=torch.float16)  # 4.8 GB
    wide[:, :64] = c["x"]
    out = ops.adapter_linear(**{**c, "x": wide[:, :64]}, out=wide[:, 100:172])
    _within(out, *_linear_ref(c))


def test_attention_bad_offsets_are_reported(cuda):
    """Offsets and lengths out of range are clamped into the tensors and reported, never followed."""
    from ctmr_b200 import _lib, ops

    q, k, v, qo, ko = _packed(1, [40, 60], None, 2, 2, 64, torch.float16)
    far = torch.tensor([0, 40, 1 << 28], device="cuda", dtype=torch.int32)
    out = ops.attention(q, k, v, q_offsets=far, k_offsets=far)
    assert _lib.device_error(clear=True) == 32
    assert torch.equal(out, ops.attention(q, k, v, q_offsets=qo, k_offsets=ko))
    back = torch.tensor([0, -5, 100], device="cuda", dtype=torch.int32)
    ops.attention(q, k, v, q_offsets=qo, k_offsets=back)
    assert _lib.device_error(clear=True) == 32
    ops.attention(q[None], k[None], v[None], k_lengths=torch.tensor([101], device="cuda", dtype=torch.int32))
    assert _lib.device_error(clear=True) == 32
    # a document with more queries than max_q allows
    ops.attention(q, k, v, q_offsets=qo, k_offsets=ko, max_q=2)
    assert _lib.device_error(clear=True) == 32


def test_attention_empty_and_captured(cuda):
    from ctmr_b200 import ops

    q, k, v, qo, ko = _packed(1, [33, 0, 100], None, 4, 2, 64, torch.float16)
    assert ops.attention(q[:0], k[:0], v[:0]).shape == (0, 4, 64)
    out, lse = ops.attention(q, k[:0], v[:0], q_offsets=qo, k_offsets=torch.zeros_like(qo), return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    eager = ops.attention(q, k, v, q_offsets=qo, causal=True)
    one = ops.attention(q[:, :1], k[:, :1], v[:, :1], causal=True)  # no offsets: one document
    ref = _document_ref(*(t[:, :1].double() for t in (q, k, v)), 64 ** -0.5, 0.0, None, True, 0)
    _check_attention(one, None, [(one, None, ref)], torch.float16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.attention(q, k, v, q_offsets=qo, causal=True)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, eager)


def test_attention_refusals(cuda):
    from ctmr_b200 import ops

    q, k, v, qo, ko = _packed(1, [40, 60], [40, 60], 4, 2, 64, torch.float16)
    kw = dict(q=q, k=k, v=v, q_offsets=qo, k_offsets=ko)
    bad = [
        dict(q=q.cpu()), dict(q=q.float()), dict(k=k.bfloat16()), dict(v=v[:50]), dict(k=k[:, :, :56], v=v[:, :, :56]),
        dict(q=q[:, :3]), dict(q_offsets=qo.long()), dict(k_offsets=ko[:2]), dict(q_offsets=None), dict(scale=0.0),
        dict(scale=-1.0), dict(scale=math.nan), dict(cap=-1.0), dict(cap=math.inf), dict(max_q=-1),
        dict(prefix=torch.zeros(2, device="cuda", dtype=torch.int32)), dict(causal=True, prefix=ko[:1]),
        dict(slopes=torch.zeros(3, device="cuda")), dict(slopes=torch.zeros(4, device="cuda", dtype=torch.float64)),
        dict(k_lengths=ko[1:]), dict(out=torch.empty_like(q, dtype=torch.bfloat16)), dict(q=q[None]),
        dict(q=torch.empty((4, 64, 100), device="cuda", dtype=torch.float16).permute(2, 0, 1)),  # channels apart
        dict(q=torch.empty(100 * 4 * 64 + 4, device="cuda", dtype=torch.float16)[4:].view(100, 4, 64)),  # misaligned
        dict(q=torch.empty((100, 4, 68), device="cuda", dtype=torch.float16)[:, :, :64]),  # strides of 68
    ]
    for change in bad:
        with pytest.raises(ValueError):
            ops.attention(**{**kw, **change})
    for dim in (60, 136):
        t = torch.zeros((10, 1, dim), device="cuda", dtype=torch.float16)
        with pytest.raises(ValueError):
            ops.attention(t, t, t)
