"""Attention over several volumes of different extents in one call, each with its own adapter.

Runs the level-3 attention block of the diffusion network (512 channels, 16 heads of 32) on the latent grids of
five requests: once packed (``ctmr_b200.packed``), once volume by volume (``fast_b200``, which has no
adapters), and prints both times and, with the adapters off, how far the two are apart.

    python examples/packed_volumes.py
"""

from __future__ import annotations

import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "mlx-generate-ctmr_b200"))

import torch  # noqa: E402

from ctmr_b200 import fast_b200, ops, packed  # noqa: E402

CHANNELS, HEAD, GROUPS, RANK, ADAPTERS = 512, 32, 32, 16, 3
EXTENTS = [(16, 16, 8), (8, 8, 4), (12, 16, 8), (5, 7, 3), (16, 8, 8)]


def block_weights(gen: torch.Generator) -> dict[str, torch.Tensor]:
    def randn(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * std

    w = {"norm.weight": 1 + randn(CHANNELS, std=0.1), "norm.bias": randn(CHANNELS, std=0.1)}
    for name in ("to_q", "to_k", "to_v", "out_proj"):
        w[f"attn.{name}.weight"] = randn(CHANNELS, CHANNELS, std=CHANNELS ** -0.5)
        w[f"attn.{name}.bias"] = randn(CHANNELS, std=0.1)
    return w


def adapter_stack(gen: torch.Generator, outputs: int, dtype: torch.dtype) -> dict[str, torch.Tensor]:
    """Low-rank adapters as they come from fine-tuning: (down, up, alpha / rank)."""
    loose = [(torch.randn(RANK, CHANNELS, generator=gen, device="cuda") * CHANNELS ** -0.5,
              torch.randn(outputs, RANK, generator=gen, device="cuda") * 0.1, 2.0) for _ in range(ADAPTERS)]
    return ops.stack_adapters(loose, dtype=dtype)


def milliseconds(run, times: int = 20) -> float:
    run()
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    torch.cuda.synchronize()
    start.record()
    for _ in range(times):
        run()
    end.record()
    torch.cuda.synchronize()
    return start.elapsed_time(end) / times


def main() -> None:
    gen = torch.Generator(device="cuda").manual_seed(0)
    weights = block_weights(gen)
    volumes = [ops.to_ndhwc(torch.randn((1, CHANNELS, *e), generator=gen, device="cuda")) for e in EXTENTS]
    grid = packed.PackedGrid.of(EXTENTS)
    sections = (4, 6, 6)
    rotary = (ops.axis_frequencies(sections), sections)
    index = torch.tensor([0, 2, -1, 1, 0], dtype=torch.int32, device="cuda")
    kw = dict(num_groups=GROUPS, eps=1e-6, num_head_channels=HEAD, include_fc=True)
    with fast_b200.arithmetic_precision("fp16"):
        adapters = {"qkv": adapter_stack(gen, 3 * CHANNELS, torch.float16),
                    "out_proj": adapter_stack(gen, CHANNELS, torch.float16)}

        def together():
            return packed.packed_spatial_attention_ncdhw(volumes, grid, weights, adapters=adapters, index=index,
                                                         rotary=rotary, **kw)

        def apart():
            return [fast_b200.spatial_attention_ncdhw(x, weights, **kw) for x in volumes]

        plain = packed.packed_spatial_attention_ncdhw(volumes, grid, weights, **kw)
        far = max(((a - b).norm() / b.norm()).item() for a, b in zip(plain, apart()))
        print(f"{len(volumes)} volumes, {grid.starts[-1]} tokens: packed with adapters and rotary positions "
              f"{milliseconds(together):.3f} ms, one by one without either {milliseconds(apart):.3f} ms; "
              f"without either the two differ by {far:.1e} (relative)")


if __name__ == "__main__":
    main()
