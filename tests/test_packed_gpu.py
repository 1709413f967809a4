"""The packed spatial-attention block (``ctmr_b200.packed``): several volumes in one call, with adapters and
rotary positions, against a 64-bit restatement per volume, and without either against the block that the
networks call volume by volume.

Bound: the block rounds its tokens, weights, Q/K/V, adapter inner products, softmax weights, merged heads and
output projection to 16 bits, seven roundings of relative size u (2^-11 fp16, 2^-8 bf16) that add up like
independent errors at worst doubled by the softmax: relative 2-norm of the added part <= 2 sqrt(7) u < 6 u."""

from __future__ import annotations

import pytest
import torch

from oracle.ops_ref import group_norm_ref

pytestmark = pytest.mark.gpu

U = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
C, HEAD, GROUPS = 128, 32, 32
EXTENTS = [(4, 8, 8), (1, 1, 1), (3, 5, 7), (8, 8, 9)]


def _weights(gen):
    w = {"norm.weight": 1 + 0.1 * torch.randn(C, generator=gen), "norm.bias": 0.1 * torch.randn(C, generator=gen)}
    for n in ("to_q", "to_k", "to_v", "out_proj"):
        w[f"attn.{n}.weight"] = torch.randn((C, C), generator=gen) * C ** -0.5
        w[f"attn.{n}.bias"] = 0.1 * torch.randn(C, generator=gen)
    return w


def _linear(x, w, b, loose):
    y = x @ w.T + b
    return y if loose is None else y + loose[2] * (x @ loose[0].T) @ loose[1].T


def _rotate(x, positions, inv_freq, sections):  # (L, heads, HEAD)
    axis = torch.repeat_interleave(torch.arange(3), torch.tensor(sections))
    angle = (positions.double()[:, axis] * inv_freq.double())[:, None]
    n = sum(sections)
    a, b, rest = x[..., :n], x[..., n:2 * n], x[..., 2 * n:]
    return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), rest), -1)


def _block_ref(x, w, qkv_adapter, out_adapter, positions, inv_freq, sections):
    h = group_norm_ref(x, w["norm.weight"], w["norm.bias"], GROUPS, 1e-6)
    tokens = h.reshape(C, -1).T
    stacked = torch.cat([w[f"attn.to_{n}.weight"] for n in "qkv"]), torch.cat([w[f"attn.to_{n}.bias"] for n in "qkv"])
    q, k, v = (t.reshape(-1, C // HEAD, HEAD) for t in _linear(tokens, *stacked, qkv_adapter).split(C, 1))
    if positions is not None:
        q, k = (_rotate(t, positions, inv_freq, sections) for t in (q, k))
    p = torch.softmax(torch.einsum("ihd,jhd->hij", q, k) * HEAD ** -0.5, -1)
    merged = torch.einsum("hij,jhd->ihd", p, v).reshape(-1, C)
    return _linear(merged, w["attn.out_proj.weight"], w["attn.out_proj.bias"], out_adapter).T.reshape(x.shape)


@pytest.mark.parametrize("precision", ["fp16", "bf16"])
@pytest.mark.parametrize("with_rotary", [False, True])
@pytest.mark.parametrize("with_adapters", [False, True])
def test_packed_block_matches_64_bits(cuda, precision, with_rotary, with_adapters):
    from ctmr_b200 import fast_b200, ops, packed

    gen = torch.Generator().manual_seed(3)
    w = _weights(gen)
    volumes = [torch.randn((1, C, *e), generator=gen) for e in EXTENTS]
    sections = (4, 6, 5)
    grid = packed.PackedGrid.of(EXTENTS)
    inv_freq = ops.axis_frequencies(sections)
    index = [1, -1, 0, 2]

    def loose(outputs, rank):
        return (torch.randn((rank, C), generator=gen) * C ** -0.5, torch.randn((outputs, rank), generator=gen) * 0.3, 1.5)

    qkv, out = [loose(3 * C, r) for r in (8, 3, 16)], [loose(C, r) for r in (4, 12, 8)]
    dtype = torch.float16 if precision == "fp16" else torch.bfloat16
    gw = {k: v.cuda() for k, v in w.items()}
    with fast_b200.arithmetic_precision(precision):
        got = packed.packed_spatial_attention_ncdhw(
            [x.cuda() for x in volumes], grid, gw, num_groups=GROUPS, eps=1e-6, num_head_channels=HEAD, include_fc=True,
            adapters={"qkv": ops.stack_adapters(qkv, dtype=dtype), "out_proj": ops.stack_adapters(out, dtype=dtype)}
            if with_adapters else None,
            index=torch.tensor(index, dtype=torch.int32, device="cuda"),
            rotary=(inv_freq, sections) if with_rotary else None)
    assert len(got) == len(volumes)
    wd = {k: v.double() for k, v in w.items()}

    def adapter(stack, i):
        return tuple(t.double() if torch.is_tensor(t) else t for t in stack[index[i]]) if with_adapters and index[i] >= 0 else None

    for i, (x, y) in enumerate(zip(volumes, got)):
        at = slice(grid.starts[i], grid.starts[i + 1])
        ref = _block_ref(x.double(), wd, adapter(qkv, i), adapter(out, i),
                         grid.positions[at].cpu() if with_rotary else None, inv_freq.cpu(), sections)
        added = y.cpu().double() - x.double()
        assert ((added - ref).norm() / ref.norm()).item() <= 6 * U[precision]


@pytest.mark.parametrize("precision", ["fp16", "bf16"])
def test_packed_block_is_the_networks_block(cuda, precision):
    from ctmr_b200 import fast_b200, packed

    gen = torch.Generator().manual_seed(4)
    w = {k: v.cuda() for k, v in _weights(gen).items()}
    volumes = [torch.randn((1, C, *e), generator=gen).cuda() for e in EXTENTS]
    kw = dict(num_groups=GROUPS, eps=1e-6, num_head_channels=HEAD, include_fc=True)
    with fast_b200.arithmetic_precision(precision):
        got = packed.packed_spatial_attention_ncdhw(volumes, packed.PackedGrid.of(EXTENTS), w, **kw)
        for x, y in zip(volumes, got):
            ref = fast_b200.spatial_attention_ncdhw(x, w, **kw) - x
            assert ((y - x - ref).norm() / ref.norm()).item() <= 2 * 6 * U[precision]


def test_packed_block_refusals(cuda):
    from ctmr_b200 import fast_b200, packed

    with pytest.raises(ValueError):
        packed.PackedGrid.of([])
    with pytest.raises(ValueError):
        packed.PackedGrid.of([(4, 0, 2)])
    grid = packed.PackedGrid.of([(2, 2, 2), (1, 2, 3)], spacing_mm=[(1.0, 0.5, 2.0), (2.0, 2.0, 2.0)])
    assert grid.positions[7].tolist() == [1.0, 0.5, 2.0] and grid.positions[-1].tolist() == [0.0, 2.0, 4.0]
    assert grid.offsets.tolist() == [0, 8, 14]
    w = {k: v.cuda() for k, v in _weights(torch.Generator().manual_seed(1)).items()}
    a, b = torch.zeros((1, C, 2, 2, 2), device="cuda"), torch.zeros((1, C, 1, 2, 3), device="cuda")
    kw = dict(num_groups=GROUPS, eps=1e-6, num_head_channels=HEAD, include_fc=True)
    with pytest.raises(ValueError, match="16-bit"):
        packed.packed_spatial_attention_ncdhw([a, b], grid, w, **kw)
    with fast_b200.arithmetic_precision("fp16"):
        with pytest.raises(ValueError):
            packed.packed_spatial_attention_ncdhw([a], grid, w, **kw)
        with pytest.raises(ValueError):
            packed.packed_spatial_attention_ncdhw([b, a], grid, w, **kw)
        with pytest.raises(ValueError):
            packed.packed_spatial_attention_ncdhw([a, b], grid, w, **{**kw, "num_head_channels": 12})
