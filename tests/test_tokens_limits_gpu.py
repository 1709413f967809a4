"""The packed-token operators at the edges of what they accept, against plain implementations in 64 bits: extreme caps,
queries that are not numbers, the lowest values in masked places, poisoned adapters, rows outside every document,
bad offsets, the forms for 17 to 128 rows of a key head, head-major and expanded layouts.

Tolerances. Outputs as in test_tokens_gpu. The log-sum-exp is a sum of fp32 terms: with scores of size S (per query),
exponentials good to 2^-22 (one pair in four of the tile form 2.6e-6 of either sign, 0.7e-6 of the sum at worst), a
chain of at most 32 additions (2^-24 each, 1.9e-6), scores rounded by 2^-22 S and the cap good to 2e-7 S, and the
logarithm's own 2^-22: ``3e-6 + (2^-22 + 2e-7) S + 2^-22 |lse|``.
"""

from __future__ import annotations

import ctypes
import math
import tempfile
from pathlib import Path

import pytest
import torch
from test_tokens_gpu import HALF, U, _gen, _linear_case, _linear_ref, _no_device_error, _offsets, _randn, _within

pytestmark = pytest.mark.gpu


def _rows_ref(q, k, v, *, scale=None, cap=0.0, slopes=None, causal=False, prefix=0):
    """One document: q (Lq, H, D), k and v (Lk, Hk, D) -> out, lse, sum of softmax |v|, size of the scores, each in
    64 bits and per query and head; queries that see nothing get zeros and -inf."""
    heads = torch.arange(q.shape[1], device=q.device) // (q.shape[1] // k.shape[1])
    q, k, v = q.double(), k.double()[:, heads], v.double()[:, heads]
    lq, lk = q.shape[0], k.shape[0]
    s = torch.einsum("ihd,jhd->hij", q, k) * (q.shape[-1] ** -0.5 if scale is None else scale)
    if cap:
        s = cap * torch.tanh(s / cap)
    place, key = torch.arange(lq, device=q.device)[:, None] + lk - lq, torch.arange(lk, device=q.device)[None]
    if slopes is not None:
        s = s - slopes.double()[:, None, None] * (place - key).abs()
    seen = (key <= place) | (key < prefix) if causal else torch.ones((lq, lk), dtype=torch.bool, device=q.device)
    size = s.masked_fill(~seen, 0.0).abs().amax(-1).T if lk else torch.zeros(q.shape[:2], device=q.device)
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1).T if lk else torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    p = torch.where(torch.isneginf(lse).T[..., None], 0.0, torch.exp(s - lse.T[..., None]))
    v = torch.where(seen.any(0)[:, None, None], v, 0.0)
    return torch.einsum("hij,jhd->ihd", p, v), lse, torch.einsum("hij,jhd->ihd", p, v.abs()), size


def _check(out, lse, ref, dtype):
    o, m, mag, size = ref
    _within(out, o, U[dtype] * o.abs() + (1.25 * U[dtype] + 2e-5 + 2.0 ** -21 * size[..., None]) * mag + 2.0 ** -25)
    if lse is not None:
        empty = torch.isneginf(m)
        assert torch.equal(torch.isneginf(lse), empty) and (out[empty] == 0).all()
        _within(lse[~empty], m[~empty], (3e-6 + (2.0 ** -22 + 2e-7) * size + 2.0 ** -22 * m.abs())[~empty])


def _kernels(call):
    """What a call launches, by the driver's text of a graph that it is captured in."""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    with tempfile.TemporaryDirectory() as where:
        path = Path(where) / "graph.dot"
        driver = ctypes.CDLL("libcuda.so.1")
        assert driver.cuGraphDebugDotPrint(ctypes.c_void_p(graph.raw_cuda_graph()), str(path).encode(), 1) == 0
        return path.read_text()


# Each form's cases: query tokens, key tokens, heads, key heads, head size.
TILES = [(150, 200, 2, 2, 40), (140, 300, 4, 2, 96)]
FEW = [(1, 1500, 4, 1, 64), (2, 2000, 16, 2, 128), (1, 300, 2, 2, 72)]
FORMS = [("attention_tile_kernel", c) for c in TILES] + [("attention_few_kernel", c) for c in FEW]


def _operands(seed, lq, lk, heads, kv_heads, dim, dtype):
    gen = _gen(seed)
    return _randn(gen, lq, heads, dim, dtype=dtype), *(_randn(gen, lk, kv_heads, dim, dtype=dtype) for _ in range(2))


# ---------------------------------------------------------------------------------------------- caps
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("cap", [1e-3, 2.0, 50.0, 1e3, 1e4, 1e6, 1e30, 3e38])
@pytest.mark.parametrize(("form", "case"), FORMS)
def test_attention_caps_of_any_size(cuda, form, case, cap, dtype):
    """A cap far above the scores leaves them as they are, one far below makes them its sign."""
    from ctmr_b200 import ops

    q, k, v = _operands(3, *case, dtype)
    call = lambda: ops.attention(q, k, v, cap=cap, causal=True, return_lse=True)  # noqa: E731
    _check(*call(), _rows_ref(q, k, v, cap=cap, causal=True), dtype)
    if cap == 50.0:
        assert form in _kernels(call)
    _no_device_error()


@pytest.mark.parametrize("cap", [1e2, 1e4, 1e6])
@pytest.mark.parametrize(("form", "case"), FORMS)
def test_attention_caps_beside_large_scores(cuda, form, case, cap):
    """Scores near the cap in some rows do not coarsen those of the others."""
    from ctmr_b200 import ops

    q, k, v = _operands(4, *case, torch.bfloat16)
    q[::2, ::2] *= cap
    out, lse = ops.attention(q, k, v, cap=cap, return_lse=True)
    _check(out, lse, _rows_ref(q, k, v, cap=cap), torch.bfloat16)


@pytest.mark.parametrize("cap", [1e-5, 1e-7, 1e-30, 1e-40])
@pytest.mark.parametrize(("form", "case"), FORMS)
def test_attention_tiny_caps_of_zero_scores(cuda, form, case, cap):
    """Queries of zeros see every key alike, however small the cap; others see its sign."""
    from ctmr_b200 import ops

    q, k, v = _operands(5, *case, torch.float16)
    for rows in (slice(None), slice(None, None, 2)):  # then every other head only
        some = q.clone()
        some[:, rows] = 0
        out, lse = ops.attention(some, k, v, cap=cap, return_lse=True)
        _check(out, lse, _rows_ref(some, k, v, cap=cap), torch.float16)


# ---------------------------------------------------------------------------------------------- not numbers
@pytest.mark.parametrize("kw", [dict(), dict(causal=True), dict(cap=5.0), dict(causal=True, slopes=True)])
@pytest.mark.parametrize(("form", "case"), FORMS)
def test_attention_of_nan_queries_is_nan(cuda, form, case, kw):
    """A query that is not a number gives an output that is not one (and no zeros), and no other row notices."""
    from ctmr_b200 import ops

    q, k, v = _operands(6, *case, torch.float16)
    kw = {**kw, **({"slopes": torch.full((q.shape[1],), 0.1, device="cuda")} if "slopes" in kw else {})}
    out, lse = ops.attention(q, k, v, return_lse=True, **kw)
    bad = q.clone()
    bad[-1, 1, 0] = math.nan
    got, got_lse = ops.attention(bad, k, v, return_lse=True, **kw)
    assert torch.isnan(got[-1, 1]).all() and torch.isnan(got_lse[-1, 1])
    got[-1, 1], got_lse[-1, 1] = out[-1, 1], lse[-1, 1]
    assert torch.equal(got, out) and torch.equal(got_lse, lse)


@pytest.mark.parametrize("lowest", [True, False])
@pytest.mark.parametrize(("form", "case"), FORMS)
def test_attention_lowest_values_in_masked_places(cuda, form, case, lowest):
    """Values that no query sees (causal), or that a score far below the others' leaves without weight, are the
    type's lowest: they count for nothing."""
    from ctmr_b200 import ops

    q, k, v = _operands(8, *case, torch.bfloat16)
    v[-8:] = torch.finfo(torch.bfloat16).min if lowest else torch.finfo(torch.bfloat16).max
    if q.shape[0] > 8:  # the last eight keys belong to the last eight queries
        out, lse = ops.attention(q, k, v, causal=True, return_lse=True)
        _check(out[:-8], lse[:-8], _rows_ref(q[:-8], k[:-8], v[:-8], causal=True), torch.bfloat16)
    k[:, :, 0], q[:, :, 0] = 0.0, 8.0
    k[-8:, :, 0] = -1e4  # scores of about -4e4
    out, lse = ops.attention(q, k, v, scale=0.5, return_lse=True)
    _check(out, lse, _rows_ref(q, k[:-8], v[:-8], scale=0.5), torch.bfloat16)


@pytest.mark.parametrize("key", range(24, 32))
@pytest.mark.parametrize(("form", "case"), FORMS)
def test_attention_of_a_nan_key_is_not_finite(cuda, form, case, key):
    """Used keys have to be finite; one that is not leaves no plausible result behind."""
    from ctmr_b200 import ops

    q, k, v = _operands(7, *case, torch.float16)
    k[key] = math.nan
    out = ops.attention(q, k, v)
    assert not torch.isfinite(out).any()


# ---------------------------------------------------------------------------------------------- adapters
POISONED = [  # lengths, adapters by segment, inner, outer, rank: tiles of 16 to 128 rows, splits, CTA pairs
    ([1] * 20, [i % 4 - 1 for i in range(20)], 512, 384, 16),
    ([5, 3, 40, 2, 17], [0, 1, -1, 2, 1], 136, 257, 8),
    ([100, 9, 150, 41], [2, 1, 0, -1], 4096, 512, 128),
    ([300, 77, 1, 222], [0, 1, 2, -1], 520, 1000, 24),
    ([1000, 1, 0, 1305], [2, 0, 1, 1], 136, 2310, 24),
    ([2500, 31, 2500], [1, -1, 0], 64, 1100, 72),
]


@pytest.mark.parametrize("where", ["up", "down", "scale"])
@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("case", range(len(POISONED)))
def test_poisoned_adapters_stay_in_their_rows(cuda, case, value, where):
    """An adapter that is not finite spoils the rows of its own segments, where the formula says so, and no others:
    not those beside them in a tile, with other adapters or with none."""
    from ctmr_b200 import ops

    lengths, index, inner, outer, rank = POISONED[case]
    c = _linear_case(case, lengths, index, inner, outer, rank, 3, torch.float16)
    if where == "up":
        c["up"][1, ::3, rank - 1] = value
    elif where == "down":
        c["down"][1, 0, 5] = value
    else:
        c["scale"][1] = value
    y = ops.adapter_linear(**c)
    ref, tol = _linear_ref(c)
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(y), fine) and fine.any() and not fine.all()
    _within(y[fine], ref[fine], tol[fine])
    _no_device_error()


# ---------------------------------------------------------------------------------------------- offsets
@pytest.mark.parametrize("max_q", [0, 2])
@pytest.mark.parametrize("documents", [1, 3, 40])
def test_attention_rows_outside_every_document(cuda, documents, max_q):
    """Rows before the first document and past the last (a call padded to a fixed number of rows) get zeros, and a
    log-sum-exp of -inf."""
    from ctmr_b200 import ops

    gen, lead, trail, each = _gen(documents), 33, 150, 2 if max_q else 45
    used = documents * each
    rows, heads, dim = lead + used + trail, 4, 72
    q, k, v = (_randn(gen, rows, heads, dim) for _ in range(3))
    offsets = torch.arange(documents + 1, device="cuda", dtype=torch.int32) * each + lead
    wide = torch.full((rows, heads, 96), 7.0, device="cuda", dtype=torch.float16)
    out, lse = ops.attention(q, k, v, q_offsets=offsets, max_q=max_q, out=wide[..., 8:80], return_lse=True)
    for part in (slice(0, lead), slice(lead + used, rows)):
        assert (out[part] == 0).all() and torch.isneginf(lse[part]).all()
    assert (wide[..., :8] == 7).all() and (wide[..., 80:] == 7).all()
    for d in range(documents):
        at = slice(lead + d * each, lead + (d + 1) * each)
        _check(out[at], lse[at], _rows_ref(q[at], k[at], v[at]), torch.float16)
    empty = torch.full_like(offsets, 5)  # no document has a row
    out, lse = ops.attention(q, k, v, q_offsets=empty, max_q=max_q, out=torch.full_like(q, 7.0), return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    _no_device_error()


@pytest.mark.parametrize(("q_off", "k_off"), [
    ([0, 100, 200], [0, 100, 100]), ([0, 100, 100], [0, 100, 200]), ([0, 100, 100], [0, 100, 99]),
    ([0, 100, 100], [0, -3, 100]), ([0, 60, 40], [0, 50, 100]), ([-1, 60, 100], [0, 50, 100]),
    ([101, 101, 101], [0, 50, 100]), ([0, 60, 40, 100], [0, 30, 60, 100]),
])
@pytest.mark.parametrize("documents", [0, 40])
def test_attention_reports_every_bad_offset(cuda, documents, q_off, k_off):
    """Offsets that fall or leave the tensor are reported whether or not their document has queries (with up to 32
    documents and with more)."""
    from ctmr_b200 import _lib, ops

    q, k, v = _operands(9, 100, 100, 2, 2, 64, torch.float16)
    more = [0] * (documents if q_off[0] == 0 else 0)
    tensors = [torch.tensor([*more, *o], device="cuda", dtype=torch.int32) for o in (q_off, k_off)]
    ops.attention(q, k, v, q_offsets=tensors[0], k_offsets=tensors[1])
    assert _lib.device_error(clear=True) == 32


@pytest.mark.parametrize("more", [0, 40])
@pytest.mark.parametrize("rows", [96, 128, 2304])
def test_adapter_linear_reports_every_bad_number(cuda, rows, more):
    from ctmr_b200 import _lib, ops

    c = _linear_case(2, [rows], [0], 64, 2310, 8, 2, torch.float16)
    good = [0] * more

    def call(offsets, index):
        c["offsets"] = torch.tensor([*good, *offsets], device="cuda", dtype=torch.int32)
        c["index"] = torch.tensor([*[-1] * len(good), *index], device="cuda", dtype=torch.int32)
        ops.adapter_linear(**c)
        return _lib.device_error(clear=True)

    assert call([0, rows, rows], [0, -1]) == 0
    assert call([0, rows, rows + 200], [0, -1]) == 32   # the last segment begins where the rows end
    assert call([0, rows, rows - 1], [0, -1]) == 32
    assert call([0, rows, rows], [0, 2]) == 32          # a segment without rows, an adapter that is not there
    assert call([0, rows, rows], [2, -1]) == 32


@pytest.mark.parametrize(("inner", "outer", "rank", "lengths"), [
    (512, 1536, 16, [1] * 4096), (4096, 520, 128, [1] * 1000), (256, 384, 72, [3] * 700), (72, 264, 8, [0, 1, 0] * 1500),
])
def test_adapter_linear_many_short_segments(cuda, inner, outer, rank, lengths):
    """Hundreds to thousands of requests of a row or a few."""
    from ctmr_b200 import ops

    c = _linear_case(inner, lengths, [(5 * i) % 24 - 1 for i in range(len(lengths))], inner, outer, rank, 23, torch.bfloat16)
    _within(ops.adapter_linear(**c), *_linear_ref(c))
    _no_device_error()


# ---------------------------------------------------------------------------------------------- the packed block
def test_packed_block_refuses_what_it_would_ignore(cuda):
    """Adapters under names that the block does not have, and tokens that are not the grid's."""
    from ctmr_b200 import ops, packed

    gen, c = _gen(1), 32
    weights = {f"attn.{n}.{part}": _randn(gen, *((c, c) if part == "weight" else (c,)))
               for n in ("to_q", "to_k", "to_v", "out_proj") for part in ("weight", "bias")}
    grid = packed.PackedGrid.of([(2, 2, 2), (1, 2, 3)])
    tokens, index = _randn(gen, 14, c), torch.tensor([0, -1], device="cuda", dtype=torch.int32)

    def stack(outputs):
        return ops.stack_adapters([(_randn(gen, 8, c), _randn(gen, outputs, 8), 1.0)], dtype=torch.float16)

    def run(tokens, include_fc=True, **adapters):
        return packed.packed_self_attention_tokens(tokens, grid, weights, heads=2, scale=0.25, include_fc=include_fc,
                                                   adapters=adapters, index=index)

    assert run(tokens, qkv=stack(3 * c), out_proj=stack(c)).shape == (14, c)
    assert run(tokens, include_fc=False, qkv=stack(3 * c)).shape == (14, c)
    for bad in (dict(to_q=stack(c)), dict(qkv=stack(3 * c), proj=stack(c)), dict(include_fc=False, out_proj=stack(c))):
        with pytest.raises(ValueError, match="adapters for"):
            run(tokens, **bad)
    for bad in (tokens[:13], torch.cat((tokens, tokens)), tokens[None]):
        with pytest.raises(ValueError, match="rows"):
            run(bad)


# ---------------------------------------------------------------------------------------------- 17 to 128 rows
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("mode", ["plain", "causal", "all"])
@pytest.mark.parametrize(("lq", "lk", "heads", "kv_heads", "dim"), [
    (1, 4000, 17, 1, 64), (2, 4001, 16, 1, 32), (1, 3000, 20, 1, 80), (4, 4100, 16, 2, 128),  # one group of 17 to 32 rows
    (1, 5000, 33, 1, 40), (11, 4000, 6, 2, 64), (8, 6000, 16, 2, 64),                         # two and more, heads to 64
    (3, 4000, 11, 1, 128), (16, 5003, 4, 1, 72), (16, 9000, 8, 1, 128), (128, 6000, 1, 1, 96), (42, 8000, 3, 1, 104),
])
def test_attention_few_rows_of_a_key_head(cuda, lq, lk, heads, kv_heads, dim, mode, dtype):
    """17 to 128 rows of a key head over long keys, in groups of 32: queries and heads that start inside a group."""
    from ctmr_b200 import ops

    q, k, v = _operands(lq + dim, lq, lk, heads, kv_heads, dim, dtype)
    kw: dict = dict(causal=mode != "plain")
    if mode == "all":
        kw |= dict(cap=5.0, scale=2 * dim ** -0.5, slopes=torch.exp2(-torch.arange(heads, device="cuda") / 4.0) * 0.01)
    pre = lk - lq + 3 if mode == "all" else 0
    prefix = torch.tensor([pre], device="cuda", dtype=torch.int32) if pre else None
    call = lambda: ops.attention(q, k, v, return_lse=True, **kw, prefix=prefix)  # noqa: E731
    out, lse = call()
    _check(out, lse, _rows_ref(q, k, v, **kw, prefix=pre), dtype)
    assert "attention_few_kernel" in _kernels(call)
    _no_device_error()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize(("batch", "lk", "heads", "kv_heads", "dim"), [
    (200, 100, 4, 2, 64), (1, 2000, 8, 8, 128), (1, 2000, 16, 1, 72), (3, 1300, 24, 1, 40),
])
def test_attention_few_log_sum_exp_is_fp32(cuda, batch, lk, heads, kv_heads, dim, cap, dtype):
    """One CTA to a request (200 of them), and keys split over a cluster."""
    from ctmr_b200 import ops

    gen = _gen(lk)
    q = _randn(gen, batch, 1, heads, dim, dtype=dtype)
    k, v = (_randn(gen, batch, lk, kv_heads, dim, dtype=dtype) for _ in range(2))
    call = lambda: ops.attention(q, k, v, cap=cap, return_lse=True)  # noqa: E731
    out, lse = call()
    for b in range(0, batch, 37):
        _check(out[b], lse[b], _rows_ref(q[b], k[b], v[b], cap=cap), dtype)
    assert "attention_few_kernel" in _kernels(call)


# ---------------------------------------------------------------------------------------------- layouts
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(("lq", "lk", "heads", "kv_heads", "dim"), [
    (150, 200, 4, 2, 64), (130, 131, 2, 2, 72), (1, 700, 8, 2, 128), (2, 4000, 16, 1, 40),
])
def test_attention_head_major_and_expanded(cuda, lq, lk, heads, kv_heads, dim, dtype):
    """(batch, head, token, channel) tensors transposed, one context expanded over the batch, and one key head's
    values expanded over the heads: the bits of the dense copies."""
    from ctmr_b200 import ops

    gen, batch = _gen(dim), 3
    q = _randn(gen, batch, heads, lq, dim, dtype=dtype).transpose(1, 2)
    k, v = (_randn(gen, batch, kv_heads, lk, dim, dtype=dtype).transpose(1, 2) for _ in range(2))
    kw = dict(k_lengths=torch.tensor([lk, lk // 2, 1], device="cuda", dtype=torch.int32), return_lse=True)

    def same(q, k, v):
        out, lse = ops.attention(q, k, v, **kw)
        dense, dense_lse = ops.attention(*(t.contiguous() for t in (q, k, v)), **kw)
        assert torch.equal(out, dense) and torch.equal(lse, dense_lse)
        for b, n in enumerate((lk, lk // 2, 1)):
            _check(out[b], lse[b], _rows_ref(q[b], k[b, :n], v[b, :n]), dtype)

    same(q, k, v)
    same(q, k[:1].expand(batch, -1, -1, -1), v[1:2].expand(batch, -1, -1, -1))
    same(q[:1].expand(batch, -1, -1, -1), k, v)
    same(q, k, v[:, :, :1].expand(-1, -1, kv_heads, -1))
    same(q[:, :, :1].expand(-1, -1, heads, -1), k[:, :, :1].expand(-1, -1, kv_heads, -1), v)
    out = torch.full((batch, heads, lq, dim), 7.0, device="cuda", dtype=dtype).transpose(1, 2)
    assert ops.attention(q, k, v, out=out, **kw)[0] is out
    assert torch.equal(out, ops.attention(q, k, v, **kw)[0])
    packed = [t.flatten(0, 1) for t in (q, k, v)]  # copies: token-major; then head-major packed rows
    major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in packed]
    offsets = dict(q_offsets=_offsets([lq] * batch), k_offsets=_offsets([lk] * batch))
    assert torch.equal(ops.attention(*packed, **offsets), ops.attention(*major, **offsets))
    _no_device_error()


def test_adapter_linear_captured(cuda):
    """Both launches in a graph, for the small and the pair kernel; replays on changed inputs follow them."""
    from ctmr_b200 import ops

    for rows, outer in ((40, 200), (2304, 2310)):
        c = _linear_case(rows, [rows // 3, rows - rows // 3], [1, 0], 136, outer, 24, 2, torch.float16)
        eager = ops.adapter_linear(**c)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = ops.adapter_linear(**c)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(captured, eager)
            c["x"].copy_(c["x"].flip(0))
            eager = ops.adapter_linear(**c)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize(("form", "case"), FORMS)
def test_attention_small_weights_keep_their_bits(cuda, form, case, dtype):
    """One key far above the others, whose values are zero: the output is what weights of 2^-18 to 2^-20 of it add up
    to, and each of them is rounded to the type's relative precision (below 2^-14 fp16 by itself has fewer bits)."""
    from ctmr_b200 import ops

    q, k, v = _operands(9, *case, dtype)
    q[..., 0], k[:, :, 0], k[:, :, 1:] = 1.0, 0.0, k[:, :, 1:] * 0.02
    k[5, :, 0], v[5] = 19 * math.log(2), 0.0
    out, lse = ops.attention(q, k, v, scale=1.0, return_lse=True)
    _check(out, lse, _rows_ref(q, k, v, scale=1.0), dtype)
