"""The packed blocks with 8-bit projections (``ctmr_b200.packed``): the operators run together, as they are used.

Bounds. A value rounded to e4m3 is off by at most 2^-4 of itself and by 2.6e-2 of itself in the mean square (a step of
2^-3 of the value's power of two, evenly spread, over significands between 1 and 2); a product of two such operands by
sqrt(2) times that, 3.7e-2, of its 2-norm, whatever its length, as the errors are independent. The attention block's
added part passes two products (values and output projection) and scores whose errors, 3.7e-2 of scores of about 1, move
the softmax weights by as much: relative 2-norm near sqrt(3) 3.7e-2 = 6.4e-2, and 0.13 allowed. A transformer block's
two branches add up; the second one's two products and its gate see the first one's error too: 0.2 of what was
added. The 64-bit restatement of the same 8-bit steps is nearer: it differs where a 16-bit rounding (u = 2^-9 of the value
in the mean) tips an 8-bit one, one value in some 2^5.5, by a step of 2^-3.5: 2^-6 relative to each operand, twice a
product, five products in a row: below 0.08.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

C, HEAD, GROUPS, HIDDEN = 256, 32, 32, 640
EXTENTS = [(4, 8, 8), (1, 1, 1), (3, 5, 7), (8, 8, 9)]
SECTIONS = (4, 6, 6)


def _weights(gen):
    w = {"norm.weight": 1 + 0.1 * torch.randn(C, generator=gen), "norm.bias": 0.1 * torch.randn(C, generator=gen)}
    for n in ("to_q", "to_k", "to_v", "out_proj"):
        w[f"attn.{n}.weight"] = torch.randn((C, C), generator=gen) * C ** -0.5
        w[f"attn.{n}.bias"] = 0.1 * torch.randn(C, generator=gen)
    return {k: v.cuda() for k, v in w.items()}


@pytest.mark.parametrize("precision", ["fp16", "bf16"])
@pytest.mark.parametrize("include_fc", [False, True])
def test_attention_block(cuda, precision, include_fc):
    from ctmr_b200 import _lib, fast_b200, ops, packed

    gen = torch.Generator().manual_seed(6)
    w = _weights(gen)
    volumes = [torch.randn((1, C, *e), generator=gen).cuda() for e in EXTENTS]
    grid = packed.PackedGrid.of(EXTENTS)
    kw = dict(num_groups=GROUPS, eps=1e-6, num_head_channels=HEAD, include_fc=include_fc,
              rotary=(ops.axis_frequencies(SECTIONS), SECTIONS))
    with fast_b200.arithmetic_precision(precision):
        scaled = packed.scaled_projections(w, include_fc=include_fc)
        got = packed.packed_spatial_attention_ncdhw(volumes, grid, w, scaled=scaled, **kw)
        ref = packed.packed_spatial_attention_ncdhw(volumes, grid, w, **kw)
    for x, a, b in zip(volumes, got, ref):
        far = ((a - b).norm() / (b - x).norm()).item()
        assert 1e-4 < far <= 0.13  # (it did run in 8 bits)
    assert _lib.device_error(clear=True) == 0


def _eight(v):
    """64-bit rows as the operators round them."""
    groups = torch.nn.functional.pad(v, (0, -v.shape[1] % 128)).unflatten(1, (-1, 128))
    fraction, exponent = torch.frexp(groups.abs().amax(dim=2, keepdim=True))
    scale = torch.exp2(torch.where(fraction == 0, -100, (exponent - 9 + (fraction > 0.875)).clamp(min=-100)).double())
    u = groups / scale
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3.0)
    return ((u / step).round() * step * scale).flatten(1)[:, :v.shape[1]]


def _transformer_ref(x, grid, blocks, heads, rotary, rounded):
    """In 64 bits; with the 8-bit roundings of rows, or without."""
    eight = _eight if rounded else (lambda v: v)
    inv_freq, sections = rotary
    axis = torch.repeat_interleave(torch.arange(3), torch.tensor(sections)).cuda()
    angle = (grid.positions.double()[:, axis] * inv_freq.double())[:, None]
    n = sum(sections)

    def norm(h, w):
        return h / torch.sqrt(h.square().mean(dim=1, keepdim=True) + 1e-6) * w.double()

    def turn(t):
        a, b, rest = t[..., :n], t[..., n:2 * n], t[..., 2 * n:]
        return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), rest), -1)

    x = x.double()
    for blk in blocks:
        w = {k: v.float().double() for k, v in blk.items() if k not in ("norm1", "norm2")}
        qkv = (eight(norm(x, blk["norm1"])) @ w["qkv"].T).view(x.shape[0], 3 * heads, -1)
        q, k, v = turn(qkv[:, :heads]), turn(qkv[:, heads:2 * heads]), qkv[:, 2 * heads:]
        merged = torch.empty_like(v)
        for a, b in zip(grid.starts, grid.starts[1:]):
            p = torch.softmax(torch.einsum("ihd,jhd->hij", q[a:b], k[a:b]) * q.shape[-1] ** -0.5, -1)
            merged[a:b] = torch.einsum("hij,jhd->ihd", p, v[a:b])
        x = x + eight(merged.flatten(1)) @ w["out_proj"].T
        up, by = (eight(norm(x, blk["norm2"])) @ w["gate_up"].T).chunk(2, dim=1)
        x = x + eight(up * torch.sigmoid(up) * by) @ w["down"].T
    return x


def _blocks(gen, count):
    from ctmr_b200 import ops

    def weight(out, inner):
        return ops.scale_weight(torch.randn((out, inner), generator=gen).cuda() * inner ** -0.5)

    return [{"norm1": 1 + 0.1 * torch.randn(C, generator=gen).cuda(), "norm2": 1 + 0.1 * torch.randn(C, generator=gen).cuda(),
             "qkv": weight(3 * C, C), "out_proj": weight(C, C), "gate_up": weight(2 * HIDDEN, C), "down": weight(C, HIDDEN)}
            for _ in range(count)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("count", [1, 2])
def test_transformer_blocks(cuda, dtype, count):
    from ctmr_b200 import _lib, ops, packed

    gen = torch.Generator().manual_seed(7)
    blocks = _blocks(gen, count)
    grid = packed.PackedGrid.of(EXTENTS)
    tokens = torch.randn((grid.starts[-1], C), generator=gen).to(dtype).cuda()
    rotary = (ops.axis_frequencies(SECTIONS), SECTIONS)
    got = packed.packed_transformer_tokens(tokens, grid, blocks, heads=C // HEAD, rotary=rotary)
    assert got.dtype == dtype
    for rounded, bound in ((True, 0.08), (False, 0.2)):
        ref = _transformer_ref(tokens, grid, blocks, C // HEAD, rotary, rounded) - tokens.double()
        added = got.double() - tokens.double()
        assert ((added - ref).norm() / ref.norm()).item() <= bound
    assert _lib.device_error(clear=True) == 0


def test_transformer_blocks_captured(cuda):
    """A captured run replayed on other tokens, with the eager run's bits."""
    from ctmr_b200 import ops, packed

    gen = torch.Generator().manual_seed(8)
    blocks = _blocks(gen, 1)
    grid = packed.PackedGrid.of(EXTENTS)
    tokens = torch.randn((grid.starts[-1], C), generator=gen).half().cuda()
    rotary = (ops.axis_frequencies(SECTIONS), SECTIONS)

    def run():
        return packed.packed_transformer_tokens(tokens, grid, blocks, heads=C // HEAD, rotary=rotary)

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = run()
    tokens.copy_(torch.randn(tokens.shape, generator=gen))
    graph.replay()
    assert torch.equal(kept, run())


def test_refusals(cuda):
    from ctmr_b200 import ops, packed

    gen = torch.Generator().manual_seed(9)
    w = _weights(gen)
    grid = packed.PackedGrid.of([(2, 2, 2)])
    tokens = torch.zeros((8, C), dtype=torch.float16, device="cuda")
    scaled = packed.scaled_projections(w, include_fc=True)
    kw = dict(heads=C // HEAD, scale=1.0)
    adapters = {"qkv": ops.stack_adapters([(torch.zeros(8, C), torch.zeros(3 * C, 8), 1.0)], dtype=torch.float16)}
    with pytest.raises(ValueError):
        packed.packed_self_attention_tokens(tokens, grid, w, include_fc=False, scaled=scaled, **kw)
    with pytest.raises(ValueError):
        packed.packed_self_attention_tokens(tokens, grid, w, include_fc=True, scaled={"qkv": scaled["qkv"]}, **kw)
    with pytest.raises(ValueError):
        packed.packed_self_attention_tokens(tokens, grid, w, include_fc=True, scaled=scaled, adapters=adapters,
                                            index=torch.zeros(1, dtype=torch.int32, device="cuda"), **kw)
    with pytest.raises(ValueError):
        packed.packed_transformer_tokens(tokens[:7], grid, _blocks(gen, 1), heads=8)
    with pytest.raises(ValueError):
        packed.packed_transformer_tokens(tokens, grid, _blocks(gen, 1), heads=7)
    assert packed.packed_transformer_tokens(tokens, grid, [], heads=8) is tokens
