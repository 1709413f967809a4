"""Cases of the 8-bit token operators, with their plain forms.

Three operators carry packed tokens through projections in 8 bits (e4m3): ``rms_norm`` (root-mean-square
norm of the rows, with the residual's addition, and an output in 16 or 32 bits or in 8 with a scale for
every 128 channels), ``quantize_rows`` (the same output for rows as they are, or for a gated pair
``silu(a) * b``) and ``scaled_linear`` (the product of such rows with a weight that has a scale for every
block of 128 x 128). ``run`` computes one of them with elementary torch operations in 32 bits, or, with
``own``, by the package's own call.

Rows in 8 bits are e4m3 values times powers of two: the scale of 128 channels is the least power of two,
and at least 2^-100, with which the largest of them is at most 448. A weight's scales may be any numbers.
"""

import functools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128


@functools.cache  # imported once, as a program does
def _ops():
    import sys
    from pathlib import Path

    package = str(Path(__file__).resolve().parents[1] / "mlx-generate-ctmr_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from ctmr_b200 import ops

    return ops


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # Prompts: the residual stream of 8192 packed tokens is updated and normed for an 8-bit projection.
        dict(name="norm-prompts", op="norm", dtype="bf16", rows=8192, channels=4096, residual=True, quantize=True),
        # Serving, one new token for each of 32 requests: latency.
        dict(name="norm-token-32", op="norm", dtype="bf16", rows=32, channels=4096, residual=True, quantize=True),
        # The packed latent voxels of seven volumes at level 3's 512 channels, kept in 16 bits.
        dict(name="norm-volumes", op="norm", dtype="fp16", rows=8968, channels=512, residual=True, quantize=False),
        # fp32 activations of an odd width, the last group of channels not full.
        dict(name="norm-odd", op="norm", dtype="fp32", rows=1777, channels=1001, residual=False, quantize=True),
        # The gated hidden channels of the same prompts, ahead of the projection back: the largest in bytes.
        dict(name="gate-prompts", op="quantize", dtype="bf16", rows=8192, channels=11264, gate=True),
        # Attention outputs of three volumes of the level-2 blocks, ahead of their output projection: small.
        dict(name="rows-volumes", op="quantize", dtype="fp16", rows=617, channels=256, gate=False),
        # Serving: the gated channels of 16 requests.
        dict(name="gate-token-16", op="quantize", dtype="bf16", rows=16, channels=11264, gate=True),
        # Prompts through the stacked Q/K/V projection, an odd number of rows: the largest product.
        dict(name="linear-prompts", op="linear", dtype="bf16", rows=8191, inner=4096, outer=12288, bias=False),
        # Fewer rows through the projection back from the hidden channels, into a 32-bit stream.
        dict(name="linear-down", op="linear", dtype="fp32", rows=2300, inner=11264, outer=4096, bias=True),
        # The level-3 attention's Q/K/V projection (512 channels) for three volumes of 256 tokens or fewer.
        dict(name="linear-volumes", op="linear", dtype="fp16", rows=617, inner=512, outer=1536, bias=True),
        # Serving, one row for each of 32 requests: the weight's bytes.
        dict(name="linear-token-32", op="linear", dtype="bf16", rows=32, inner=4096, outer=4096, bias=False),
        # Serving, a single row through the projection back.
        dict(name="linear-token-1", op="linear", dtype="bf16", rows=1, inner=11264, outer=4096, bias=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "quantize", "linear", "linear"])
    dtype = rng.choice(["bf16", "fp16", "bf16", "fp16", "fp32"])
    if kind == "linear":
        # From one row to a prompt's, widths down to 64 and of any remainder: rows fall until the product is
        # no larger than the largest listed one.
        inner, outer = rng.choice([1, 8, 16]) * _log_int(rng, 64, 768), _log_int(rng, 64, 12288)
        rows = min(_log_int(rng, 1, 16000), 8191 * 4096 * 12288 // (inner * outer))
        return dict(op="linear", dtype=dtype, rows=rows, inner=inner, outer=outer, bias=rng.random() < 0.5)
    channels = rng.choice([_log_int(rng, 5, 16384), 8 * _log_int(rng, 4, 2048)])
    rows = min(_log_int(rng, 1, 40000), 8192 * 4096 // channels)
    if kind == "norm":
        return dict(op="norm", dtype=dtype, rows=rows, channels=channels, residual=rng.random() < 0.6,
                    quantize=rng.random() < 0.6)
    return dict(op="quantize", dtype=dtype, rows=rows, channels=channels, gate=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------- inputs
def _power(top):
    """The scale of a group whose largest magnitude is `top`: 448 is 0.875 * 2^9."""
    fraction, exponent = torch.frexp(top)
    exponent = torch.where(top == 0, -100, (exponent - 9 + (fraction > 0.875)).clamp(min=-100))
    return torch.ldexp(torch.ones_like(top), exponent)


def _grouped(x, size=BLOCK):
    """The last axis in groups of `size`, zeros behind the last one's end."""
    n = x.shape[-1]
    return torch.nn.functional.pad(x, (0, -n % size)).unflatten(-1, (-1, size))


def _quantized(x):
    """8-bit values and scales of fp32 rows."""
    groups = _grouped(x)
    scale = _power(groups.abs().amax(dim=-1))
    values = (groups / scale.unsqueeze(-1)).flatten(-2)[:, :x.shape[1]]
    return values.to(torch.float8_e4m3fn), scale


def _rows_apart(values):
    """8-bit rows laid out as the operators take them: a multiple of 16 bytes apart."""
    room = torch.zeros((values.shape[0], (values.shape[1] + 15) // 16 * 16), dtype=torch.uint8, device=values.device)
    room[:, :values.shape[1]] = values.view(torch.uint8)
    return room.view(torch.float8_e4m3fn)[:, :values.shape[1]]


def _quantized_blocks(w):
    """8-bit values and scales of an fp32 weight, by blocks of 128 x 128; scales of any value, as checkpoints hold them."""
    out, inner = w.shape
    blocks = _grouped(_grouped(w).permute(1, 2, 0)).permute(2, 3, 0, 1)  # (out blocks, 128, in blocks, 128)
    scale = (blocks.abs().amax(dim=(1, 3)) / 448.0).clamp(min=2.0 ** -100)
    values = (blocks / scale[:, None, :, None]).flatten(2).flatten(0, 1)[:out, :inner]
    return values.to(torch.float8_e4m3fn), scale


def _inputs(case, seed, device):
    gen = torch.Generator(device=device).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device=device) * std

    rows = case["rows"]
    if case["op"] == "norm":
        # A residual stream has rows of different size and a few channels far above the others.
        channels = case["channels"]
        x = randn(rows, channels) * torch.exp(randn(rows, 1))
        x[:, torch.randint(channels, (channels // 200,), generator=gen, device=device)] *= 20.0
        return dict(x=x.to(dtype), residual=randn(rows, channels, std=0.5).to(dtype) if case["residual"] else None,
                    weight=(1.0 + randn(channels, std=0.2)), eps=1e-6)
    if case["op"] == "quantize":
        width = case["channels"] * (2 if case["gate"] else 1)
        return dict(x=(randn(rows, width) * torch.exp(randn(rows, 1, std=0.5))).to(dtype))
    inner, outer = case["inner"], case["outer"]
    values, scale = _quantized(randn(rows, inner) * torch.exp(randn(rows, 1)))
    w_values, w_scale = _quantized_blocks(randn(outer, inner, std=inner ** -0.5))
    return dict(values=_rows_apart(values), scale=scale, w_values=_rows_apart(w_values), w_scale=w_scale,
                bias=randn(outer, std=0.5) if case["bias"] else None)


def prepare(case, seed):
    return dict(_inputs(case, seed, "cuda"), op=case["op"], dtype=DTYPES[case["dtype"]],
                quantize=case.get("quantize", True), gate=case.get("gate", False))


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    y = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + s["eps"]) * s["weight"]
    y = _quantized(y) if s["quantize"] else y.to(s["dtype"])
    return (y, x.to(s["dtype"])) if s["residual"] is not None else y


def _plain_quantize(s):
    x = s["x"].float()
    if s["gate"]:
        a, b = x.chunk(2, dim=-1)
        x = a / (1.0 + torch.exp(-a)) * b
    return _quantized(x)


def _spread(scale, size, dim):
    return scale.repeat_interleave(BLOCK, dim=dim).narrow(dim, 0, size)


def _plain_linear(s):
    inner, outer = s["values"].shape[1], s["w_values"].shape[0]
    x = s["values"].float() * _spread(s["scale"], inner, 1)
    w = s["w_values"].float() * _spread(_spread(s["w_scale"], inner, 1), outer, 0)
    y = x @ w.T
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["dtype"])


def run(state):
    if state["op"] == "norm":
        if not own:
            return _plain_norm(state)
        return _ops().rms_norm(state["x"], state["weight"], residual=state["residual"], eps=state["eps"],
                               quantize=state["quantize"])
    if state["op"] == "quantize":
        return _ops().quantize_rows(state["x"], gate=state["gate"]) if own else _plain_quantize(state)
    if not own:
        return _plain_linear(state)
    ops = _ops()
    return ops.scaled_linear(ops.ScaledRows(state["values"], state["scale"]),
                             ops.ScaledWeight(state["w_values"], state["w_scale"]), state["bias"],
                             out_dtype=state["dtype"])


# ---------------------------------------------------------------------------------------------- work
def work(case):
    size, rows = 4 if case["dtype"] == "fp32" else 2, case["rows"]
    if case["op"] == "linear":
        inner, outer = case["inner"], case["outer"]
        blocks, wide = -(-inner // BLOCK), -(-outer // BLOCK)
        return {"bytes": rows * inner + inner * outer + 4 * blocks * (rows + wide) + size * rows * outer
                + (4 * outer if case["bias"] else 0), "flops": 2 * rows * inner * outer}
    channels = case["channels"]
    eight = rows * channels + 4 * rows * -(-channels // BLOCK)
    if case["op"] == "norm":
        out = eight if case["quantize"] else size * rows * channels
        return {"bytes": size * rows * channels * (3 if case["residual"] else 1) + 4 * channels + out,
                "flops": rows * channels * (6 if case["residual"] else 5)}
    return {"bytes": size * rows * channels * (2 if case["gate"] else 1) + eight,
            "flops": rows * channels * (8 if case["gate"] else 2)}


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_quantized(v):
    """The nearest e4m3 values, ties to even, of 64-bit rows over their groups' scales; and the scales."""
    rows, channels = v.shape
    values = torch.empty_like(v)
    scales = []
    for c in range(0, channels, BLOCK):
        part = v[:, c:c + BLOCK]
        top = part.abs().amax(dim=1)
        power = torch.full_like(top, -100.0)
        # The least power that reaches, found from below the logarithm's.
        near = torch.floor(torch.log2(top.clamp(min=2.0 ** -120) / 448.0))
        for step in (1.0, 0.0, -1.0):
            power = torch.where(top <= 448.0 * torch.exp2(near + step), near + step, power)
        scale = torch.exp2(power.clamp(min=-100.0))
        u = part / scale[:, None]
        # Steps of 1/8 of the value's power of two, of 2^-9 below 2^-6.
        grid = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3.0)
        values[:, c:c + BLOCK] = torch.round(u / grid) * grid
        scales.append(scale)
    return values, torch.stack(scales, dim=1)


def exact(case, seed):
    s = _inputs(case, seed, "cuda")
    if case["op"] == "linear":
        values, w = s["values"].double(), s["w_values"].double()
        y = torch.zeros((values.shape[0], w.shape[0]), dtype=torch.float64, device=w.device)
        per_out = torch.arange(w.shape[0], device=w.device) // BLOCK
        for b in range(s["scale"].shape[1]):
            k = slice(b * BLOCK, (b + 1) * BLOCK)
            weight = w[:, k] * s["w_scale"].double()[per_out, b].unsqueeze(1)
            y.addmm_(values[:, k] * s["scale"].double()[:, b:b + 1], weight.T)
        return y if s["bias"] is None else y + s["bias"].double()
    x = s["x"].double()
    if case["op"] == "quantize":
        if case["gate"]:
            n = case["channels"]
            x = x[:, :n] * torch.sigmoid(x[:, :n]) * x[:, n:]
        return _exact_quantized(x)
    if s["residual"] is not None:
        x = x + s["residual"].double()
    y = x / torch.sqrt(torch.mean(x * x, dim=1, keepdim=True) + s["eps"]) * s["weight"].double()
    y = _exact_quantized(y) if case["quantize"] else y
    return (y, x) if s["residual"] is not None else y
