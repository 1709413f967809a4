"""The spatial self-attention block for several volumes of different extents in one call.

``fast_b200.spatial_attention_ncdhw`` takes one tensor, so volumes of different extents, or of different
fine-tuned variants (one per site, scanner or contrast), have to run one by one. Here the voxels of all of
them are packed as the rows of one token tensor: the group norm of each volume writes its rows, one shared
Q/K/V projection carries each volume's low-rank adapter beside it (``ops.adapter_linear``), the query and key
heads optionally get rotary positions along depth, height and width (``ops.rotary_axes``), attention stays
inside each volume (``ops.attention``), and the output projection again carries the adapters. Without adapters
and positions the result is that of ``spatial_attention_ncdhw`` volume by volume (``attention.py:92-160``).

The projections may run in 8 bits instead (``scaled_projections``): rows are quantised as they are made
(``ops.quantize_rows``, ``ops.rms_norm``) and multiplied by 8-bit weights (``ops.scaled_linear``).
``packed_transformer_tokens`` runs pre-norm blocks (norm, attention, norm, gated hidden channels) that way.
"""

from __future__ import annotations

from collections.abc import Mapping, Sequence
from dataclasses import dataclass

import torch

from . import fast_b200, ops


@dataclass(frozen=True)
class PackedGrid:
    """Where each volume's voxels lie among the packed rows, made once for a set of extents."""

    extents: tuple[tuple[int, int, int], ...]
    starts: tuple[int, ...]        # first row of each volume, and the number of rows
    offsets: torch.Tensor          # the same, int32 on the device
    positions: torch.Tensor        # (rows, 3): depth, height, width of each row's voxel

    @classmethod
    def of(cls, extents: Sequence[tuple[int, int, int]], *, spacing_mm: Sequence[tuple[float, float, float]] | None = None,
           device="cuda") -> PackedGrid:
        """Rows for volumes of ``extents`` (D, H, W), in order. Positions are voxel indices (int32), or
        millimetres (fp32) where ``spacing_mm`` gives each volume's voxel size."""
        if not extents:
            raise ValueError("no volumes to pack")
        extents = tuple((int(d), int(h), int(w)) for d, h, w in extents)
        starts, parts = [0], []
        for i, e in enumerate(extents):
            if min(e) < 1:
                raise ValueError(f"volume extents must be positive; got {e}")
            starts.append(starts[-1] + e[0] * e[1] * e[2])
            at = torch.cartesian_prod(*(torch.arange(n, dtype=torch.int32) for n in e)).reshape(-1, 3)
            parts.append(at * torch.tensor(spacing_mm[i], dtype=torch.float32) if spacing_mm is not None else at)
        return cls(extents, tuple(starts), torch.tensor(starts, dtype=torch.int32).to(device),
                   torch.cat(parts).contiguous().to(device))


def _project(tokens, weight, bias, grid, adapters, index):
    if adapters is None:
        return ops.adapter_linear(tokens, weight, bias)
    return ops.adapter_linear(tokens, weight, bias, **adapters, offsets=grid.offsets, index=index)


def _attend(qkv: torch.Tensor, grid: PackedGrid, heads: int, scale: float, rotary: tuple | None) -> torch.Tensor:
    """Attention inside each volume, of the stacked projection's rows ``(rows, 3 C)``; gives ``(rows, C)``."""
    rows, c = qkv.shape[0], qkv.shape[1] // 3
    qkv = qkv.view(rows, 3 * heads, c // heads)
    if rotary is not None:  # query and key heads lie side by side: one call, in place
        inv_freq, sections = rotary
        turned = qkv[:, :2 * heads]
        ops.rotary_axes(turned, grid.positions, inv_freq, sections, out=turned)
    q, k, v = qkv.split(heads, dim=1)
    return ops.attention(q, k, v, q_offsets=grid.offsets, scale=scale).view(rows, c)


def scaled_projections(weights: Mapping[str, torch.Tensor], *, include_fc: bool,
                       prefix: str = "attn") -> dict[str, ops.ScaledWeight]:
    """The 8-bit weights of an attention block's projections, made once, where the block is loaded."""
    scaled = {"qkv": ops.scale_weight(torch.cat([weights[f"{prefix}.to_{n}.weight"] for n in ("q", "k", "v")]))}
    if include_fc:
        scaled["out_proj"] = ops.scale_weight(weights[f"{prefix}.out_proj.weight"])
    return scaled


def packed_self_attention_tokens(tokens: torch.Tensor, grid: PackedGrid, weights: Mapping[str, torch.Tensor], *,
                                 heads: int, scale: float, include_fc: bool,
                                 adapters: Mapping[str, Mapping[str, torch.Tensor]] | None = None,
                                 index: torch.Tensor | None = None, rotary: tuple | None = None, prefix: str = "attn",
                                 qkv_bias: bool = True,
                                 scaled: Mapping[str, ops.ScaledWeight] | None = None) -> torch.Tensor:
    """``fast_b200.self_attention_tokens`` on the packed rows ``(rows, C)`` of a grid's volumes, 16-bit.

    ``adapters`` may hold stacks (``ops.stack_adapters``) under ``"qkv"`` (C -> 3C) and ``"out_proj"``
    (C -> C); ``index`` (int32 on the device) names each volume's, negative for none. ``rotary`` is
    ``(inv_freq, sections)`` for three axes (``ops.axis_frequencies``). ``scaled`` (``scaled_projections``) runs the
    projections in 8 bits, without adapters.
    """
    dt = tokens.dtype
    if tokens.dim() != 2 or tokens.shape[0] != grid.starts[-1]:
        raise ValueError(f"tokens {tuple(tokens.shape)} where the grid has {grid.starts[-1]} rows")
    used = ("qkv", "out_proj") if include_fc else ("qkv",)
    if unknown := sorted(set(adapters or ()) - set(used)):
        raise ValueError(f"adapters for {unknown}; this block has {', '.join(used)}")
    if scaled is not None and (adapters or set(scaled) != set(used)):
        raise ValueError(f"8-bit projections take no adapters and are {', '.join(used)}; got {', '.join(sorted(scaled))}")
    names = ("q", "k", "v")
    b_qkv = fast_b200._stacked_dense(tuple(weights[f"{prefix}.to_{n}.bias"] for n in names), dt) if qkv_bias else None
    adapters = adapters or {}
    if scaled is not None:
        qkv = ops.scaled_linear(ops.quantize_rows(tokens), scaled["qkv"], b_qkv, out_dtype=dt)
    else:
        w_qkv = fast_b200._stacked_dense(tuple(weights[f"{prefix}.to_{n}.weight"] for n in names), dt)
        qkv = _project(tokens, w_qkv, b_qkv, grid, adapters.get("qkv"), index)
    merged = _attend(qkv, grid, heads, scale, rotary)
    if include_fc and scaled is not None:
        merged = ops.scaled_linear(ops.quantize_rows(merged), scaled["out_proj"],
                                   fast_b200._dense_weight(weights[f"{prefix}.out_proj.bias"], dt), out_dtype=dt)
    elif include_fc:
        merged = _project(merged, fast_b200._dense_weight(weights[f"{prefix}.out_proj.weight"], dt),
                          fast_b200._dense_weight(weights[f"{prefix}.out_proj.bias"], dt), grid,
                          adapters.get("out_proj"), index)
    return merged


def packed_spatial_attention_ncdhw(volumes: Sequence[torch.Tensor], grid: PackedGrid, weights: Mapping[str, torch.Tensor],
                                   *, num_groups: int, eps: float, num_head_channels: int, include_fc: bool,
                                   adapters: Mapping[str, Mapping[str, torch.Tensor]] | None = None,
                                   index: torch.Tensor | None = None, rotary: tuple | None = None,
                                   scaled: Mapping[str, ops.ScaledWeight] | None = None) -> list[torch.Tensor]:
    """``fast_b200.spatial_attention_ncdhw`` of several ``(1, C, D, H, W)`` volumes at once; see the module's
    head. Needs a 16-bit arithmetic precision (``fast_b200.arithmetic_precision("fp16" | "bf16")``)."""
    dt = fast_b200.dense_dtype()
    if dt == torch.float32:
        raise ValueError("packed attention runs in a 16-bit arithmetic precision (fp16 or bf16)")
    if len(volumes) != len(grid.extents):
        raise ValueError(f"{len(volumes)} volumes for a grid of {len(grid.extents)}")
    c = int(volumes[0].shape[1])
    if c % num_head_channels or num_head_channels % 8:
        raise ValueError("channels must be a multiple of the head's, and the head's a multiple of 8")
    tokens = torch.empty((grid.starts[-1], c), dtype=dt, device=volumes[0].device)
    kept = []
    for x, (d, h, w), start in zip(volumes, grid.extents, grid.starts):
        if tuple(x.shape) != (1, c, d, h, w):
            raise ValueError(f"volume of shape {tuple(x.shape)} where the grid has (1, {c}, {d}, {h}, {w})")
        x = ops.to_ndhwc(x, fast_b200.activation_dtype())
        affine = ops.group_norm_affine(x, weights["norm.weight"], weights["norm.bias"], groups=num_groups, eps=eps)
        place = tokens[start:start + d * h * w].view(1, d, h, w, c).permute(0, 4, 1, 2, 3)
        ops.transform(x, affine=affine, out=place)  # straight into the volume's rows
        kept.append(x)
    heads, scale = c // num_head_channels, float(num_head_channels) ** -0.5
    merged = packed_self_attention_tokens(tokens, grid, weights, heads=heads, scale=scale, include_fc=include_fc,
                                          adapters=adapters, index=index, rotary=rotary, scaled=scaled)
    return [torch.add(x, merged[start:start + d * h * w].view(1, d, h, w, c).permute(0, 4, 1, 2, 3))
            for x, (d, h, w), start in zip(kept, grid.extents, grid.starts)]


def packed_transformer_tokens(tokens: torch.Tensor, grid: PackedGrid, blocks: Sequence[Mapping[str, object]], *, heads: int,
                              eps: float = 1e-6, rotary: tuple | None = None) -> torch.Tensor:
    """Pre-norm transformer blocks on a grid's packed rows ``(rows, C)`` in 16 bits, projections in 8.

    A block holds ``norm1`` and ``norm2`` (``(C,)``), and ``ops.ScaledWeight``s ``qkv`` (C -> 3C), ``out_proj``
    (C -> C), ``gate_up`` (C -> 2F: what is gated by silu, then what it multiplies) and ``down`` (F -> C). Each norm
    adds the branch before it to the residual stream and gives 8-bit rows in the same pass."""
    if tokens.dim() != 2 or tokens.shape[0] != grid.starts[-1] or heads < 1 or tokens.shape[1] % heads:
        raise ValueError(f"tokens {tuple(tokens.shape)} where the grid has {grid.starts[-1]} rows, in {heads} heads")
    dt, scale = tokens.dtype, (tokens.shape[1] // heads) ** -0.5
    stream, branch = tokens, None
    for block in blocks:
        if branch is None:
            rows = ops.rms_norm(stream, block["norm1"], eps=eps, quantize=True)
        else:
            rows, stream = ops.rms_norm(branch, block["norm1"], residual=stream, eps=eps, quantize=True)
        merged = _attend(ops.scaled_linear(rows, block["qkv"], out_dtype=dt), grid, heads, scale, rotary)
        branch = ops.scaled_linear(ops.quantize_rows(merged), block["out_proj"], out_dtype=dt)
        rows, stream = ops.rms_norm(branch, block["norm2"], residual=stream, eps=eps, quantize=True)
        hidden = ops.quantize_rows(ops.scaled_linear(rows, block["gate_up"], out_dtype=dt), gate=True)
        branch = ops.scaled_linear(hidden, block["down"], out_dtype=dt)
    return stream if branch is None else torch.add(stream, branch)
