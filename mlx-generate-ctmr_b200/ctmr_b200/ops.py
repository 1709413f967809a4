"""Torch-tensor entry points over the C ABI.

Activations are torch tensors with the reference's logical NCDHW shape stored
channels-last (``torch.channels_last_3d``), i.e. physically NDHWC rows; a
channel slice of such a tensor is also accepted (its rows keep the parent's
stride). Every function launches on the current torch CUDA stream and
allocates its outputs and workspaces through torch's caching allocator, so the
calls can be captured in CUDA graphs.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import NamedTuple

import torch

from . import _lib
from ._lib import LIB, check

F32 = torch.float32
BF16 = torch.bfloat16
PRECISIONS = ("fp32", "bf16", "fp16", "tf32")

# Instrumentation: LAUNCHES counts the library's kernel launches issued from
# Python; when PROFILE is a list, conv3d and group_norm_affine append one record
# per stage ({"kind": "prepare" | "gemm" | "gn", "start", "end", "flops", "what"},
# CUDA events on the current stream) around their launches.
LAUNCHES = [0]
PROFILE: list | None = None


def _count(n: int) -> None:
    LAUNCHES[0] += n


class _profiled:
    """Append a PROFILE record bracketing the enclosed launches with CUDA events."""

    def __init__(self, kind: str, flops: float, what: str) -> None:
        self.rec = {"kind": kind, "flops": flops, "what": what,
                    "start": torch.cuda.Event(enable_timing=True), "end": torch.cuda.Event(enable_timing=True)}

    def __enter__(self):
        self.rec["start"].record()
        return self

    def __exit__(self, *exc) -> None:
        self.rec["end"].record()
        PROFILE.append(self.rec)


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _dtype_code(dtype: torch.dtype, *, allow_f16: bool = False) -> int:
    if dtype == F32:
        return _lib.DTYPE_F32
    if dtype == BF16:
        return _lib.DTYPE_BF16
    if allow_f16 and dtype == torch.float16:
        return _lib.DTYPE_F16
    raise ValueError(f"ctmr_b200 activations must be float32 or bfloat16, got {dtype}")


def _precision_code(precision: str) -> int:
    if precision == "fp32":
        return _lib.PRECISION_FP32
    if precision == "bf16":
        return _lib.PRECISION_BF16
    if precision == "fp16":
        return _lib.PRECISION_FP16
    if precision == "tf32":
        return _lib.PRECISION_TF32
    raise ValueError(f"precision must be one of {PRECISIONS}; got {precision!r}")


def rows_stride(x: torch.Tensor) -> int:
    """Elements between voxel rows of an NDHWC-stored NCDHW tensor; raises if not so stored."""
    if x.dim() != 5:
        raise ValueError(f"expected an NCDHW tensor, got shape {tuple(x.shape)}")
    b, c, d, h, w = (int(n) for n in x.shape)
    if w > 1:
        cs = x.stride(4)
    elif h > 1:
        cs = x.stride(3)
    elif d > 1:
        cs = x.stride(2)
    elif b > 1:
        cs = x.stride(0)
    else:
        cs = c
    ok = cs >= c and (c == 1 or x.stride(1) == 1)
    ok = ok and (w == 1 or x.stride(4) == cs) and (h == 1 or x.stride(3) == w * cs)
    ok = ok and (d == 1 or x.stride(2) == h * w * cs) and (b == 1 or x.stride(0) == d * h * w * cs)
    if not ok:
        raise ValueError(
            f"tensor of shape {tuple(x.shape)} and strides {x.stride()} is not channels-last (NDHWC rows)"
        )
    return int(cs)


class LabelBits:
    """An int16 label volume ``(N, 1, D, H, W)`` that ``conv3d`` reads as its 8 bit-plane
    channels (channel k = bit k of the id, 0.0 or 1.0), formed in the conv's operand pass
    (``CTMR_DTYPE_LABEL8``) instead of as a materialised fp32 condition: the ControlNet
    condition of ``condition.binarize_labels_ncdhw`` (``condition.py:20-43``)."""

    def __init__(self, label: torch.Tensor) -> None:
        if label.dim() != 5 or int(label.shape[1]) != 1 or not label.is_cuda:
            raise ValueError(f"label must be a CUDA (N, 1, D, H, W) tensor; got {tuple(label.shape)}")
        if label.dtype not in (torch.int16, torch.int32, torch.int64, torch.uint8):
            raise ValueError(f"label must be integer; got {label.dtype}")
        self.label = label.to(torch.int16).contiguous()
        self.shape = torch.Size((int(label.shape[0]), 8, *(int(s) for s in label.shape[2:])))
        self.device = label.device
        self.dtype = torch.int16

    def dim(self) -> int:
        return 5


def view(x) -> _lib.Tensor:
    """``ctmr_tensor`` for an NDHWC-stored tensor, a ``LabelBits`` volume, or an absent one."""
    if x is None:
        return _lib.Tensor(None, 0, 0, 0)
    if isinstance(x, LabelBits):
        return _lib.Tensor(x.label.data_ptr(), _lib.DTYPE_LABEL8, 8, 1)
    if not x.is_cuda:
        raise ValueError("ctmr_b200 tensors must live on a CUDA device")
    return _lib.Tensor(x.data_ptr(), _dtype_code(x.dtype), int(x.shape[1]), rows_stride(x))


def empty_ndhwc(b: int, c: int, d: int, h: int, w: int, dtype: torch.dtype, device) -> torch.Tensor:
    """Uninitialised NCDHW tensor with channels-last storage."""
    return torch.empty((b, c, d, h, w), dtype=dtype, device=device, memory_format=torch.channels_last_3d)


def to_ndhwc(x: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    """Channels-last copy of an NCDHW tensor (via the library's transpose kernel when contiguous NCDHW)."""
    dtype = dtype or x.dtype
    try:
        rows_stride(x)
        return x if x.dtype == dtype else transform(x, out_dtype=dtype)
    except ValueError:
        pass
    x = x.contiguous()
    b, c, d, h, w = x.shape
    out = empty_ndhwc(b, c, d, h, w, dtype, x.device)
    _count(1)
    check(
        LIB.ctmr_ncdhw_to_ndhwc(
            x.data_ptr(), _dtype_code(x.dtype), out.data_ptr(), _dtype_code(dtype), b, c, d * h * w, _stream()
        ),
        "ncdhw_to_ndhwc",
    )
    return out


def to_ncdhw(x: torch.Tensor, dtype: torch.dtype = F32) -> torch.Tensor:
    """Contiguous NCDHW copy of a channels-last tensor (library transpose kernel)."""
    cs = rows_stride(x)
    b, c, d, h, w = x.shape
    if cs != c:
        x = transform(x, out_dtype=x.dtype)
    out = torch.empty((b, c, d, h, w), dtype=dtype, device=x.device)
    _count(1)
    check(
        LIB.ctmr_ndhwc_to_ncdhw(
            x.data_ptr(), _dtype_code(x.dtype), out.data_ptr(), _dtype_code(dtype), b, c, d * h * w, _stream()
        ),
        "ndhwc_to_ncdhw",
    )
    return out


@dataclass(frozen=True)
class PackedWeight:
    """Convolution weight packed for the tensor cores (``ctmr_pack_weight``)."""

    hi: torch.Tensor
    lo: torch.Tensor | None
    out_channels: int
    in_channels: int
    kernel_size: int
    upsample: bool
    precision: str


def pack_weight(weight: torch.Tensor, precision: str, *, upsample: bool = False) -> PackedWeight:
    """Pack a Torch ``(O, C, k, k, k)`` weight; the nearest-2x fold with ``upsample``.

    Counterpart of ``pack_weight`` / ``pack_upsample_weight`` (``_nax_conv.py:391-445``).
    A weight whose storage is channels-last ``(O, k, k, k, C)`` — the Torch-layout view
    ``weights.load_network_file`` returns for a released checkpoint — is packed from
    that storage directly (``ctmr_pack_weight_channels_last``), without a transposed copy.
    """
    if weight.dim() != 5 or weight.shape[2] != weight.shape[3] or weight.shape[3] != weight.shape[4]:
        raise ValueError(f"conv weight must be (O, C, k, k, k); got {tuple(weight.shape)}")
    o, c, k = int(weight.shape[0]), int(weight.shape[1]), int(weight.shape[2])
    code = _precision_code(precision)
    w = weight.detach()
    channels_last = (w.dtype == F32 and c > 1 and k > 1 and
                     w.is_contiguous(memory_format=torch.channels_last_3d))
    if not channels_last:
        w = w.to(dtype=F32).contiguous()
    entry = LIB.ctmr_pack_weight_channels_last if channels_last else LIB.ctmr_pack_weight
    n = int(LIB.ctmr_packed_weight_elems(o, c, k, int(upsample)))
    if n == 0:
        raise ValueError(f"unsupported conv weight shape {tuple(weight.shape)}")
    if precision == "fp32":
        hi = torch.empty(n, dtype=torch.float16, device=w.device)
        lo = torch.empty(n, dtype=torch.float16, device=w.device)
    elif precision == "tf32":  # TF32-rounded fp32 rows of round8(C) values
        hi = torch.empty(int(LIB.ctmr_packed_weight_bytes(o, c, k, int(upsample), code)) // 4, dtype=F32,
                         device=w.device)
        lo = None
    else:
        hi = torch.empty(n, dtype=BF16 if precision == "bf16" else torch.float16, device=w.device)
        lo = None
    _count(1)
    check(
        entry(
            w.data_ptr(), o, c, k, int(upsample), code, hi.data_ptr(), lo.data_ptr() if lo is not None else None,
            _stream(),
        ),
        "pack_weight",
    )
    return PackedWeight(hi, lo, o, c, k, upsample, precision)


def conv3d(
    x: torch.Tensor,
    packed: PackedWeight,
    bias: torch.Tensor | None = None,
    *,
    x2: torch.Tensor | None = None,
    affine: torch.Tensor | None = None,
    silu: bool = False,
    stride: int = 1,
    trilinear: bool = False,
    avgpool: bool = False,
    residual: torch.Tensor | None = None,
    residual_upsampled: bool = False,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    stats: bool = False,
    workspace: torch.Tensor | None = None,
    stages: int | None = None,
    norm: tuple | None = None,
) -> torch.Tensor:
    """``conv(prepare(x ++ x2)) + bias (+ residual)`` in one call (``ctmr_conv3d``).

    Mirrors ``nax_conv3d`` (``_nax_conv.py:475-487``): ``bias`` is ``(O,)`` or per
    batch item ``(B, O)``; ``affine`` is the ``(B, C, 2)`` group-norm scale/offset;
    ``silu`` follows it; ``packed.upsample`` convolves the nearest-2x upsampling,
    ``trilinear`` the half-pixel trilinear-2x upsampling and ``avgpool`` the 2x2x2
    mean of the prepared input; the residual (on the output grid, or the half grid
    when ``residual_upsampled``) is added before the single rounding.
    """
    b, cx, d, h, w = (int(n) for n in x.shape)
    cin = cx + (int(x2.shape[1]) if x2 is not None else 0)
    if x2 is not None and tuple(x2.shape[2:]) != (d, h, w):
        raise ValueError(f"concat inputs differ in grid: {tuple(x.shape)} vs {tuple(x2.shape)}")
    if cin != packed.in_channels:
        raise ValueError(f"packed weight has {packed.in_channels} input channels, input has {cin}")
    k = packed.kernel_size
    if packed.upsample:
        od, oh, ow = 2 * d, 2 * h, 2 * w
    elif trilinear:
        od, oh, ow = 2 * d, 2 * h, 2 * w
    elif avgpool:
        od, oh, ow = d // 2, h // 2, w // 2
    elif stride == 2:
        od, oh, ow = (d - 1) // 2 + 1, (h - 1) // 2 + 1, (w - 1) // 2 + 1
    else:
        od, oh, ow = d, h, w
    o = packed.out_channels
    bias_rows = 0
    if bias is not None:
        if not (bias.shape == (o,) or bias.shape == (b, o)):
            raise ValueError(f"bias shape {tuple(bias.shape)} must be ({o},) or ({b}, {o})")
        if bias.dim() == 2 and bias.dtype == F32 and bias.stride(1) == 1 and bias.stride(0) >= o:
            bias_rows = int(bias.stride(0))  # a column slice of a wider table: read in place
        else:
            bias = bias.to(dtype=F32).contiguous()
    if affine is not None:
        affine = affine.to(dtype=F32).contiguous()
        if affine.numel() != b * cin * 2:
            raise ValueError(f"affine must hold (B, C, 2) = ({b}, {cin}, 2) values")
    if residual is not None:
        expect = (b, o, od // 2, oh // 2, ow // 2) if residual_upsampled else (b, o, od, oh, ow)
        if tuple(residual.shape) != expect:
            raise ValueError(f"residual shape {tuple(residual.shape)} != output {expect}")
    if out is None:
        dtype = out_dtype or F32
        out = empty_ndhwc(b, o, od, oh, ow, dtype, x.device)
    elif tuple(out.shape) != (b, o, od, oh, ow):
        raise ValueError(f"out shape {tuple(out.shape)} != {(b, o, od, oh, ow)}")
    ycs = rows_stride(out)
    desc = _lib.Conv3dDesc()
    desc.batch, desc.depth, desc.height, desc.width = b, d, h, w
    desc.x = view(x)
    desc.x2 = view(x2)
    desc.out_channels = o
    desc.kernel_size = k
    desc.stride = stride
    desc.upsample = int(packed.upsample)
    desc.trilinear = int(trilinear)
    desc.avgpool = int(avgpool)
    desc.precision = _precision_code(packed.precision)
    desc.weight = packed.hi.data_ptr()
    desc.weight_lo = packed.lo.data_ptr() if packed.lo is not None else None
    desc.affine = affine.data_ptr() if affine is not None else None
    desc.silu = int(silu)
    desc.bias = bias.data_ptr() if bias is not None else None
    desc.bias_per_batch = int(bias is not None and bias.dim() == 2)
    desc.bias_row_stride = bias_rows
    desc.residual = view(residual)
    desc.residual_upsampled = int(residual_upsampled)
    desc.y = out.data_ptr()  # a channel slice's pointer already includes its first channel
    desc.y_dtype = _dtype_code(out.dtype)
    desc.y_cstride = ycs
    desc.y_coffset = 0
    keep = []
    if norm is not None:  # (gamma, beta, groups, eps): the input's GroupNorm computed inside the call
        gamma, beta, groups, eps = norm
        gamma = gamma.to(dtype=F32).contiguous() if gamma is not None else None
        beta = beta.to(dtype=F32).contiguous() if beta is not None else None
        keep = [gamma, beta]
        desc.gn_gamma = gamma.data_ptr() if gamma is not None else None
        desc.gn_beta = beta.data_ptr() if beta is not None else None
        desc.gn_groups = int(groups)
        desc.gn_eps = float(eps)
    stats_buf = None
    if stats:  # GroupNorm moments of the output from the conv epilogue, when its kernel can produce them
        slots = int(LIB.ctmr_conv3d_stats_slots(ctypes.byref(desc)))
        if slots > 0:
            stats_buf = torch.empty((b, slots, o, 3), dtype=F32, device=x.device)
            desc.stats = stats_buf.data_ptr()
            desc.stats_slots = slots
    ws_bytes = int(LIB.ctmr_conv3d_workspace_size(ctypes.byref(desc)))
    if workspace is not None:  # caller-held workspace (e.g. to time the GEMM stage alone)
        if workspace.numel() < ws_bytes:
            raise WorkspaceTooSmall(ws_bytes, workspace.numel())
        ws = workspace
    else:
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    ws_ptr = ws.data_ptr() if ws is not None else None
    if stages is not None:  # one or both stages (_lib.CONV_PREPARE | _lib.CONV_GEMM)
        _count(int(LIB.ctmr_conv3d_launch_count(ctypes.byref(desc))))
        check(LIB.ctmr_conv3d_stages(ctypes.byref(desc), ws_ptr, ws_bytes, int(stages), _stream()), "conv3d stages")
        return out
    _count(int(LIB.ctmr_conv3d_launch_count(ctypes.byref(desc))))
    if PROFILE is None:
        check(LIB.ctmr_conv3d(ctypes.byref(desc), ws_ptr, ws_bytes, _stream()), "conv3d")
    else:
        taps = 8 if packed.upsample else k ** 3
        what = (f"{b}x{cin}->{o} out {od}x{oh}x{ow} k{k} s{stride} up{int(packed.upsample)} tri{int(trilinear)} "
                f"pool{int(avgpool)} norm{int(affine is not None or norm is not None)} res{int(residual is not None)} "
                f"{packed.precision}")
        if ws_bytes:
            with _profiled("prepare", 0.0, what):
                check(LIB.ctmr_conv3d_stages(ctypes.byref(desc), ws_ptr, ws_bytes, _lib.CONV_PREPARE, _stream()),
                      "conv3d prepare")
        with _profiled("gemm", 2.0 * b * od * oh * ow * o * cin * taps, what):
            check(LIB.ctmr_conv3d_stages(ctypes.byref(desc), ws_ptr, ws_bytes, _lib.CONV_GEMM, _stream()),
                  "conv3d gemm")
    if stats_buf is not None:
        out._ctmr_stats = OutputStats(stats_buf, int(desc.stats_slots), o)
    del keep
    return out


class WorkspaceTooSmall(ValueError):
    """A caller-held conv3d workspace is smaller than the call needs (``needed`` bytes)."""

    def __init__(self, needed: int, given: int) -> None:
        super().__init__(f"conv3d workspace holds {given} bytes, needs {needed}")
        self.needed = needed


class OutputStats:
    """Per-(batch item, slot, channel) moments a convolution wrote for its output tensor."""

    __slots__ = ("buffer", "slots", "channels")

    def __init__(self, buffer: torch.Tensor, slots: int, channels: int) -> None:
        self.buffer, self.slots, self.channels = buffer, slots, channels


def output_stats(t: torch.Tensor | None) -> OutputStats | None:
    """The statistics attached to ``t`` by the convolution that produced it, if any."""
    return getattr(t, "_ctmr_stats", None) if t is not None else None


def group_norm_affine(
    x: torch.Tensor,
    weight: torch.Tensor | None,
    bias: torch.Tensor | None,
    *,
    groups: int,
    eps: float,
    x2: torch.Tensor | None = None,
) -> torch.Tensor:
    """GroupNorm statistics of ``x ++ x2`` as ``(B, C, 2)`` (scale, offset) pairs (``ctmr_group_norm_affine``)."""
    b, c, d, h, w = (int(n) for n in x.shape)
    ctot = c + (int(x2.shape[1]) if x2 is not None else 0)
    voxels = d * h * w
    if ctot % groups:
        raise ValueError("group_norm channels must be divisible by num_groups")
    gamma = weight.to(dtype=F32).contiguous() if weight is not None else None
    beta = bias.to(dtype=F32).contiguous() if bias is not None else None
    affine = torch.empty((b, ctot, 2), dtype=F32, device=x.device)
    sa, sb = output_stats(x), output_stats(x2)
    if (sa is not None and sa.channels == c and (x2 is None or (sb is not None and sb.slots == sa.slots and
                                                                sb.channels == ctot - c))):
        # The producing convolutions already reduced the moments: merge them only.
        _count(1)

        def from_stats() -> None:
            check(LIB.ctmr_group_norm_affine_from_stats(
                sa.buffer.data_ptr(), c, sb.buffer.data_ptr() if sb is not None else None, ctot - c if sb else 0,
                sa.slots, b, gamma.data_ptr() if gamma is not None else None,
                beta.data_ptr() if beta is not None else None, groups, float(eps), affine.data_ptr(), _stream()),
                "group_norm_affine_from_stats")

        if PROFILE is None:
            from_stats()
        else:
            with _profiled("gn", 0.0, f"{b}x{ctot} {d}x{h}x{w} g{groups} from-stats"):
                from_stats()
        return affine
    _count(int(LIB.ctmr_group_norm_launch_count(voxels, ctot, groups)))
    ws_bytes = int(LIB.ctmr_group_norm_workspace_size(b, voxels, groups))
    ws = torch.empty(max(ws_bytes, 4), dtype=torch.uint8, device=x.device)
    def launch() -> None:
        check(
            LIB.ctmr_group_norm_affine(
                view(x), view(x2), b, voxels,
                gamma.data_ptr() if gamma is not None else None,
                beta.data_ptr() if beta is not None else None,
                groups, float(eps), affine.data_ptr(), ws.data_ptr(), ws_bytes, _stream(),
            ),
            "group_norm_affine",
        )

    if PROFILE is None:
        launch()
    else:
        with _profiled("gn", 0.0, f"{b}x{ctot} {d}x{h}x{w} g{groups}"):
            launch()
    return affine


def group_norm_moments(x: torch.Tensor, *, groups: int, x2: torch.Tensor | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """Merged ``(count, mean, M2)`` per (batch item, group) of ``x ++ x2`` as ``(B, groups, 3)`` fp32
    (``ctmr_group_norm_moments``): the statistics of ``group_norm_affine`` before the affine, for
    tensors split across devices. ``out`` may be a view into a larger (exchange) buffer."""
    b, c, d, h, w = (int(n) for n in x.shape)
    ctot = c + (int(x2.shape[1]) if x2 is not None else 0)
    if ctot % groups:
        raise ValueError("group_norm channels must be divisible by num_groups")
    if out is None:
        out = torch.empty((b, groups, 3), dtype=F32, device=x.device)
    elif out.dtype != F32 or out.numel() != b * groups * 3 or not out.is_contiguous():
        raise ValueError(f"moments output must be {b * groups * 3} contiguous float32 values")
    voxels = d * h * w
    ws_bytes = int(LIB.ctmr_group_norm_workspace_size(b, voxels, groups))
    ws = torch.empty(max(ws_bytes, 4), dtype=torch.uint8, device=x.device)
    _count(2)
    check(LIB.ctmr_group_norm_moments(view(x), view(x2), b, voxels, groups, out.data_ptr(), ws.data_ptr(), ws_bytes,
                                      _stream()), "group_norm_moments")
    return out


def group_norm_affine_from_moments(moments: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, *,
                                   channels: int, groups: int, eps: float) -> torch.Tensor:
    """``(B, C, 2)`` affine from the moments ``(parts, B, groups, 3)`` of the parts of one tensor
    (``ctmr_group_norm_affine_from_moments``; merged in part order)."""
    if moments.dim() != 4 or int(moments.shape[2]) != groups or int(moments.shape[3]) != 3:
        raise ValueError(f"moments must be (parts, B, {groups}, 3); got {tuple(moments.shape)}")
    moments = moments.to(dtype=F32).contiguous()
    parts, b = int(moments.shape[0]), int(moments.shape[1])
    gamma = weight.to(dtype=F32).contiguous() if weight is not None else None
    beta = bias.to(dtype=F32).contiguous() if bias is not None else None
    affine = torch.empty((b, channels, 2), dtype=F32, device=moments.device)
    _count(1)
    check(LIB.ctmr_group_norm_affine_from_moments(
        moments.data_ptr(), parts, b, int(channels), gamma.data_ptr() if gamma is not None else None,
        beta.data_ptr() if beta is not None else None, int(groups), float(eps), affine.data_ptr(), _stream()),
        "group_norm_affine_from_moments")
    return affine


def attention_d32(qkv: torch.Tensor, heads: int, scale: float) -> torch.Tensor:
    """``softmax(Q K^T * scale) V`` per head for head size 32 (``ctmr_attention_d32``).

    ``qkv`` is the fused projection ``(B, L, 3 * heads * 32)`` in fp16 or bf16 with
    ``L`` a multiple of 128; returns ``(B, L, heads * 32)`` in the same type. The
    counterpart of the reference's ``flash_attention`` (``_flash_attention.py:320-360``).
    """
    if qkv.dim() != 3 or qkv.dtype not in (torch.float16, BF16) or not qkv.is_contiguous():
        raise ValueError("qkv must be a contiguous (B, L, 3C) fp16/bf16 tensor")
    b, length, c3 = (int(n) for n in qkv.shape)
    if c3 != 3 * heads * 32 or length % 128:
        raise ValueError(f"qkv {tuple(qkv.shape)} does not hold {heads} heads of 32 over a multiple of 128 tokens")
    out = torch.empty((b, length, heads * 32), dtype=qkv.dtype, device=qkv.device)
    _count(1)
    check(LIB.ctmr_attention_d32(qkv.data_ptr(), _lib.DTYPE_BF16 if qkv.dtype == BF16 else _lib.DTYPE_F16, b, length,
                                 heads, float(scale), out.data_ptr(), _stream()), "attention")
    return out


_HALF_CODES = {BF16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_FLOAT_CODES = {F32: _lib.DTYPE_F32, **_HALF_CODES}


def _device_stream(t: torch.Tensor, name: str) -> tuple[int, int]:
    """Index of the CUDA device that holds ``t``, which must be the current one, and its current stream.
    (The raw calls: a small kernel is over before ``torch.cuda.current_stream()`` returns.)"""
    dev = t.get_device()
    if dev < 0 or dev != torch._C._cuda_getDevice():
        raise ValueError(f"{name} must be on the current CUDA device; it is on {t.device}")
    return dev, torch._C._cuda_getCurrentRawStream(dev)


def _int32_vector(t: torch.Tensor, n: int | None, name: str, dev: int) -> torch.Tensor:
    if t.dtype != torch.int32 or t.dim() != 1 or (n is not None and t.shape[0] != n) or t.get_device() != dev:
        raise ValueError(f"{name} must be {'' if n is None else f'{n} '}int32 values on cuda:{dev}; got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def axis_frequencies(sections: tuple[int, ...], *, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """``inv_freq`` for ``rotary_axes``: pair l of an axis with n pairs turns by ``theta ** (-l / n)`` per unit."""
    freq = [theta ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in sections]
    return torch.cat(freq).to(F32).to(device)


def rotary_axes(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, sections: tuple[int, ...], *,
                interleaved: bool = False, inverse: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions along several axes (``ctmr_rotary_axes``).

    ``x`` is ``(tokens, heads, head_dim)`` in fp32, bf16 or fp16, any strides over tokens and heads (the query
    and key heads of a fused projection are one such view); ``positions`` is ``(tokens, axes)`` int32 or fp32;
    ``sections`` gives the number of pairs of each axis and ``inv_freq`` one fp32 frequency per pair
    (``axis_frequencies``). Pairs are ``(c, c + pairs)``, or ``(2c, 2c + 1)`` when ``interleaved``; channels past
    them are copied. ``inverse`` turns back (the transpose: a gradient's direction). ``out`` may be ``x``.
    """
    code = _FLOAT_CODES.get(x.dtype)
    if x.dim() != 3 or code is None:
        raise ValueError(f"x must be a (tokens, heads, head_dim) fp32/bf16/fp16 tensor; got {tuple(x.shape)} {x.dtype}")
    dev, stream = _device_stream(x, "x")
    shape = x.shape
    tokens, heads, dim = shape
    axes, pairs = len(sections), sum(sections)
    if not 1 <= axes <= _lib.MAX_ROTARY_AXES or min(sections) < 0:
        raise ValueError(f"sections {sections} must name 1 to {_lib.MAX_ROTARY_AXES} axes")
    fractional = positions.dtype == F32
    if (positions.shape != (tokens, axes) or not (fractional or positions.dtype == torch.int32)
            or positions.get_device() != dev):
        raise ValueError(f"positions must be ({tokens}, {axes}) int32 or float32 on cuda:{dev}; got "
                         f"{tuple(positions.shape)} {positions.dtype} on {positions.device}")
    if inv_freq.dtype != F32 or inv_freq.shape != (pairs,) or inv_freq.get_device() != dev:
        raise ValueError(f"inv_freq must be {pairs} float32 values on cuda:{dev}")
    if axes > 1 and positions.stride(1) != 1:
        positions = positions.contiguous()
    if out is None:
        out = x.new_empty(shape)
    elif out.shape != shape or out.dtype != x.dtype or out.get_device() != dev:
        raise ValueError(f"out must be like x: {tuple(shape)} {x.dtype}")
    xt, xh, xc = x.stride()
    yt, yh, yc = out.stride()
    if dim > 1 and (xc != 1 or yc != 1):
        raise ValueError("the channels of x and out must be contiguous")
    if heads == 1:  # a stride that addresses nothing must not narrow the accesses
        xh = yh = 0
    if tokens == 1:
        xt = yt = 0
    inv_freq = inv_freq.contiguous()
    desc = _lib.RotaryDesc(x.data_ptr(), out.data_ptr(), code, tokens, heads, dim, xt, xh, yt, yh,
                           positions.data_ptr(), fractional, positions.stride(0), inv_freq.data_ptr(), axes,
                           (*sections, *(0,) * (_lib.MAX_ROTARY_AXES - axes)), interleaved, inverse)
    LAUNCHES[0] += 1
    status = LIB.ctmr_rotary_axes(ctypes.byref(desc), stream)
    if status:
        check(status, "rotary_axes")
    return out


def stack_adapters(adapters, *, dtype: torch.dtype, device="cuda") -> dict[str, torch.Tensor]:
    """The ``down``, ``up`` and ``scale`` of ``adapter_linear`` for ``(down, up, scale)`` triples of any ranks up
    to 128: ``down`` ``(rank, in)`` and ``up`` ``(out, rank)``, padded with zeros to the largest rank's next
    multiple of 8. Done once, where the adapters are loaded."""
    adapters = list(adapters)
    if not adapters:
        raise ValueError("no adapters to stack")
    inner, outer = int(adapters[0][0].shape[1]), int(adapters[0][1].shape[0])
    for d, u, _ in adapters:
        if d.dim() != 2 or u.dim() != 2 or d.shape[1] != inner or u.shape[0] != outer or d.shape[0] != u.shape[1]:
            raise ValueError(f"adapter of shapes {tuple(d.shape)}, {tuple(u.shape)} beside a ({outer}, {inner}) "
                             "projection")
    rank = (max(int(d.shape[0]) for d, _, _ in adapters) + 7) // 8 * 8
    down = torch.zeros((len(adapters), rank, inner), dtype=dtype, device=device)
    up = torch.zeros((len(adapters), outer, rank), dtype=dtype, device=device)
    for i, (d, u, _) in enumerate(adapters):
        down[i, :d.shape[0]] = d.to(device=device, dtype=dtype)
        up[i, :, :u.shape[1]] = u.to(device=device, dtype=dtype)
    scale = torch.tensor([float(s) for _, _, s in adapters], dtype=F32, device=device)
    return {"down": down, "up": up, "scale": scale}


def adapter_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                   down: torch.Tensor | None = None, up: torch.Tensor | None = None,
                   scale: torch.Tensor | None = None, offsets: torch.Tensor | None = None,
                   index: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """A shared projection with each request's low-rank adapter beside it (``ctmr_adapter_linear``).

    ``x`` ``(rows, in)`` holds the requests' rows one after another, request s at
    ``offsets[s]:offsets[s + 1]`` (int32, on the device); ``index[s]`` is its adapter, negative for none:
    ``y = x weight^T + bias + scale[a] * (x down[a]^T) up[a]^T``. 16-bit operands (all of one type; ``bias`` may
    be fp32), fp32 sums. ``down`` ``(n, rank, in)``, ``up`` ``(n, out, rank)`` and ``scale`` ``(n,)`` come from
    ``stack_adapters``. Without them it is the plain projection. ``out`` must not overlap ``x``. The adapter's inner
    product ``scale * x down^T`` is rounded to the operands' type and must stay in its range; an adapter that is not
    finite spoils its own requests' rows only.
    """
    dtype = x.dtype
    code = _HALF_CODES.get(dtype)
    if x.dim() != 2 or code is None:
        raise ValueError(f"x must be a (rows, in) bf16/fp16 tensor; got {tuple(x.shape)} {dtype}")
    dev, stream = _device_stream(x, "x")
    rows, inner = x.shape
    if weight.dim() != 2 or weight.shape[1] != inner or weight.dtype != dtype or weight.get_device() != dev:
        raise ValueError(f"weight must be (out, {inner}) {dtype} on cuda:{dev}; got {tuple(weight.shape)} {weight.dtype}")
    outer = weight.shape[0]
    bias_at, bias_code = None, 0
    if bias is not None:
        if bias.shape != (outer,) or bias.dtype not in (F32, dtype) or bias.get_device() != dev:
            raise ValueError(f"bias must be {outer} float32 or {dtype} values on cuda:{dev}")
        bias = bias.contiguous()
        bias_at, bias_code = bias.data_ptr(), _FLOAT_CODES[bias.dtype]
    if out is None:
        out = x.new_empty((rows, outer))
    elif out.shape != (rows, outer) or out.dtype != dtype or out.get_device() != dev:
        raise ValueError(f"out must be ({rows}, {outer}) {dtype} on cuda:{dev}")
    (xs, xc), (ws, wc), (ys, yc) = x.stride(), weight.stride(), out.stride()
    if (inner > 1 and (xc != 1 or wc != 1)) or (outer > 1 and yc != 1):
        raise ValueError("the columns of x, weight and out must be contiguous")
    adapted = (None, None, None, 0, 0, None, None, 0)
    if down is None:
        if up is not None or scale is not None or offsets is not None or index is not None:
            raise ValueError("down, up, scale, offsets and index come together")
    else:
        if up is None or scale is None or offsets is None or index is None:
            raise ValueError("down, up, scale, offsets and index come together")
        n, rank = down.shape[0], down.shape[1] if down.dim() == 3 else 0
        if down.shape != (n, rank, inner) or up.shape != (n, outer, rank) or scale.shape != (n,):
            raise ValueError(f"adapters must be (n, rank, {inner}), (n, {outer}, rank) and (n,); got "
                             f"{tuple(down.shape)}, {tuple(up.shape)}, {tuple(scale.shape)}")
        if (down.dtype != dtype or up.dtype != dtype or scale.dtype != F32 or down.get_device() != dev
                or up.get_device() != dev or scale.get_device() != dev):
            raise ValueError(f"down and up must be {dtype}, scale float32, all on cuda:{dev}")
        down, up, scale = down.contiguous(), up.contiguous(), scale.contiguous()
        index = _int32_vector(index, None, "index", dev)
        segments = index.shape[0]
        offsets = _int32_vector(offsets, segments + 1, "offsets", dev)
        adapted = (down.data_ptr(), up.data_ptr(), scale.data_ptr(), n, rank, offsets.data_ptr(), index.data_ptr(),
                   segments)
    desc = _lib.AdapterLinearDesc(
        x.data_ptr(), xs if rows > 1 else inner, code, rows, inner, outer, weight.data_ptr(),
        ws if outer > 1 else inner, bias_at, bias_code, *adapted, out.data_ptr(), ys if rows > 1 else outer)
    ref = ctypes.byref(desc)
    ws_bytes = LIB.ctmr_adapter_linear_workspace_size(ref)
    if ws_bytes:
        workspace = x.new_empty(ws_bytes, dtype=torch.uint8)
        LAUNCHES[0] += 2
        status = LIB.ctmr_adapter_linear(ref, workspace.data_ptr(), ws_bytes, stream)
    else:
        LAUNCHES[0] += 1
        status = LIB.ctmr_adapter_linear(ref, None, 0, stream)
    if status:
        check(status, "adapter_linear")
    return out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, q_offsets: torch.Tensor | None = None,
              k_offsets: torch.Tensor | None = None, k_lengths: torch.Tensor | None = None, max_q: int = 0,
              scale: float | None = None, causal: bool = False, prefix: torch.Tensor | None = None, cap: float = 0.0,
              slopes: torch.Tensor | None = None, out: torch.Tensor | None = None, return_lse: bool = False):
    """Softmax attention inside documents (``ctmr_attention``); 16-bit, head size a multiple of 8 up to 128.

    Packed: ``q`` ``(q_tokens, heads, head_dim)``, ``k`` and ``v`` ``(k_tokens, kv_heads, head_dim)``; document d is
    rows ``q_offsets[d]:q_offsets[d + 1]`` and ``k_offsets[d]:k_offsets[d + 1]`` (int32 on the device; ``k_offsets``
    defaults to ``q_offsets``, no offsets at all to one document). ``max_q``, where known, says that no document has
    more queries (few query rows to a key head: the keys are split over the GPU instead). Batched:
    ``(batch, tokens, heads, head_dim)``, of each item's keys the first ``k_lengths[b]``.

    ``causal``: query i of Lq sees keys up to i + Lk - Lq, and those before ``prefix[d]``; otherwise all of its
    document. ``cap`` > 0 caps the scaled scores with a tanh; ``slopes`` ``(heads,)`` then subtracts
    ``slopes[h] * |i + Lk - Lq - j|``. A query that sees no key gives zeros (log-sum-exp -inf), and so does a
    row of ``q`` before the first document or past the last. ``heads`` may be a multiple of ``kv_heads``. Any
    strides that are multiples of 8. Keys outside a document or past its length may hold anything; those inside must
    be finite. Returns ``out``, or ``(out, lse)`` with the fp32 natural log-sum-exp ``(.., tokens, heads)``.
    """
    dtype, dims = q.dtype, q.dim()
    code = _HALF_CODES.get(dtype)
    if dims not in (3, 4) or code is None:
        raise ValueError(f"q must be a (tokens, heads, head_dim) or (batch, tokens, heads, head_dim) bf16/fp16 tensor; "
                         f"got {tuple(q.shape)} {dtype}")
    dev, stream = _device_stream(q, "q")
    shape, k_shape = q.shape, k.shape
    heads, dim, kv_heads = shape[-2], shape[-1], k_shape[-2]
    if (len(k_shape) != dims or v.shape != k_shape or k_shape[-1] != dim or k_shape[:-3] != shape[:-3] or kv_heads < 1
            or heads % kv_heads):
        raise ValueError(f"q {tuple(shape)}, k {tuple(k_shape)} and v {tuple(v.shape)} do not belong together")
    if k.dtype != dtype or v.dtype != dtype or k.get_device() != dev or v.get_device() != dev:
        raise ValueError(f"k and v must be {dtype} on cuda:{dev}")
    if out is None:
        out = q.new_empty(shape)
    elif out.shape != shape or out.dtype != dtype or out.get_device() != dev:
        raise ValueError(f"out must be {tuple(shape)} {dtype} on cuda:{dev}")
    qo = ko = kl = None
    documents = 1
    if dims == 4:
        if q_offsets is not None or k_offsets is not None:
            raise ValueError("offsets belong to packed (tokens, heads, head_dim) tensors")
        documents = shape[0]
        if k_lengths is not None:
            k_lengths = _int32_vector(k_lengths, documents, "k_lengths", dev)
            kl = k_lengths.data_ptr()
    elif k_lengths is not None:
        raise ValueError("k_lengths belong to batched (batch, tokens, heads, head_dim) tensors")
    elif q_offsets is not None:
        q_offsets = _int32_vector(q_offsets, None, "q_offsets", dev)
        documents = q_offsets.shape[0] - 1
        if k_offsets is None and k_shape[0] != shape[0]:
            raise ValueError("k_offsets are needed where k has other tokens than q")
        k_offsets = q_offsets if k_offsets is None else _int32_vector(k_offsets, documents + 1, "k_offsets", dev)
        qo, ko = q_offsets.data_ptr(), k_offsets.data_ptr()
    elif k_offsets is not None:
        raise ValueError("q_offsets and k_offsets come together")
    if documents < 1:
        if dims == 3:
            raise ValueError("q_offsets name no document")
        return (out, torch.empty(shape[:-1], dtype=F32, device=q.device)) if return_lse else out
    prefix_at = slopes_at = lse = lse_at = None
    if prefix is not None:
        prefix = _int32_vector(prefix, documents, "prefix", dev)
        prefix_at = prefix.data_ptr()
    if slopes is not None:
        if slopes.dtype != F32 or slopes.shape != (heads,) or slopes.get_device() != dev:
            raise ValueError(f"slopes must be {heads} float32 values on cuda:{dev}")
        slopes = slopes.contiguous()
        slopes_at = slopes.data_ptr()
    if return_lse:
        lse = q.new_empty(shape[:-1], dtype=F32)
        lse_at = lse.data_ptr()
    qs, ks, vs, ys = q.stride(), k.stride(), v.stride(), out.stride()
    if qs[-1] != 1 or ks[-1] != 1 or vs[-1] != 1 or ys[-1] != 1:
        raise ValueError("the channels of q, k, v and out must be contiguous")
    if dims == 3:
        qs, ks, vs, ys = (0, *qs), (0, *ks), (0, *vs), (0, *ys)
    if documents == 1 or heads == 1 or kv_heads == 1 or shape[-3] <= 1 or k_shape[-3] <= 1:
        # a stride over an extent of one addresses nothing, whatever torch calls it
        def cut(st, tokens, n):
            return (st[0] if documents > 1 else 0, st[1] if tokens > 1 else 0, st[2] if n > 1 else 0)

        qs, ys = cut(qs, shape[-3], heads), cut(ys, shape[-3], heads)
        ks, vs = cut(ks, k_shape[-3], kv_heads), cut(vs, k_shape[-3], kv_heads)
    desc = _lib.AttentionDesc(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse_at, code, documents, shape[-3], k_shape[-3], heads,
        kv_heads, dim, *qs[:3], *ks[:3], *vs[:3], *ys[:3], qo, ko, kl, prefix_at, slopes_at,
        dim ** -0.5 if scale is None else scale, cap, causal, max_q)
    LAUNCHES[0] += 1
    status = LIB.ctmr_attention(ctypes.byref(desc), stream)
    if status:
        check(status, "attention")
    return (out, lse) if return_lse else out


E4M3 = torch.float8_e4m3fn
SCALE_GROUP = 128  # channels that share a scale


class ScaledRows(NamedTuple):
    """Rows in 8 bits: ``values[i, c] * scale[i, c // 128]``."""

    values: torch.Tensor  # (rows, channels) e4m3, rows a multiple of 16 bytes apart
    scale: torch.Tensor   # (rows, ceil(channels / 128)) fp32

    def float(self) -> torch.Tensor:
        return self.values.float() * self.scale.repeat_interleave(SCALE_GROUP, dim=1)[:, :self.values.shape[1]]


class ScaledWeight(NamedTuple):
    """A projection's weight in 8 bits: ``values[o, i] * scale[o // 128, i // 128]``."""

    values: torch.Tensor  # (out, in) e4m3, rows a multiple of 16 bytes apart
    scale: torch.Tensor   # (ceil(out / 128), ceil(in / 128)) fp32, any values

    def float(self) -> torch.Tensor:
        out, inner = self.values.shape
        scale = self.scale.repeat_interleave(SCALE_GROUP, dim=0)[:out]
        return self.values.float() * scale.repeat_interleave(SCALE_GROUP, dim=1)[:, :inner]


def scale_weight(weight: torch.Tensor) -> ScaledWeight:
    """A ``(out, in)`` weight in 8 bits, for ``scaled_linear``: for every block of 128 x 128 the least power of two,
    at least 2^-100, with which its largest magnitude is at most 448. Done once, where the weight is loaded; one that
    is stored in 8 bits already is ``ScaledWeight(values, scale)``."""
    if weight.dim() != 2 or not weight.is_floating_point() or min(weight.shape) < 1:
        raise ValueError(f"weight must be a (out, in) tensor; got {tuple(weight.shape)} {weight.dtype}")
    out, inner = weight.shape
    w = weight.detach().to(F32)
    if not torch.isfinite(w).all():
        raise ValueError("weight holds values that are not finite in fp32")
    w = torch.nn.functional.pad(w, (0, -inner % SCALE_GROUP, 0, -out % SCALE_GROUP))
    blocks = w.unflatten(1, (-1, SCALE_GROUP)).unflatten(0, (-1, SCALE_GROUP))
    top = blocks.abs().amax(dim=(1, 3))
    fraction, exponent = torch.frexp(top)  # 448 is 0.875 * 2^9
    power = torch.where(top == 0, -100, (exponent - 9 + (fraction > 0.875)).clamp(min=-100))
    scale = ((power.to(torch.int32) + 127) << 23).view(F32)
    values = (blocks / scale[:, None, :, None]).flatten(2).flatten(0, 1)[:out]
    room = (inner + 15) // 16 * 16
    return ScaledWeight(values[:, :room].to(E4M3).contiguous()[:, :inner], scale)


def _allocator(root=torch._C):
    """Uninitialised memory of a shape, strides and type on the current device, from torch's caching allocator: by the
    entry that compiled programs use where this torch has it, at a fifth of ``new_empty``'s 3 us."""
    for name in ("_dynamo", "guards", "_empty_strided_cuda"):
        root = getattr(root, name, None)
    return root or (lambda size, stride, dtype: torch.empty_strided(size, stride, dtype=dtype, device="cuda"))


_empty = _allocator()


def _empty_rows8(rows: int, channels: int) -> ScaledRows:
    """Uninitialised 8-bit rows; scales lie group by group, as the products read them."""
    return ScaledRows(_empty((rows, channels), ((channels + 15) & ~15, 1), E4M3),
                      _empty((rows, (channels + 127) >> 7), (1, rows), F32))


def _row_place(t: torch.Tensor, like: torch.Tensor, dev: int, name: str) -> tuple[int, int, int]:
    """Address of rows like another tensor's, and their strides over tokens and heads."""
    shape = like.shape
    if t is not like and (t.shape != shape or t.dtype != like.dtype or t.get_device() != dev):
        raise ValueError(f"{name} must be like x: {tuple(shape)} {like.dtype} on cuda:{dev}")
    st = t.stride()
    if st[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"the channels of x, residual and the outputs must be contiguous; {name} has strides {st}")
    # a stride over an extent of one addresses nothing, whatever torch calls it
    return t.data_ptr(), st[0] if shape[0] > 1 else 0, st[1] if len(shape) == 3 and shape[1] > 1 else 0


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
             eps: float = 1e-6, quantize: bool = False, out: torch.Tensor | None = None,
             sum_out: torch.Tensor | None = None):
    """Root-mean-square norm over the channels, after the residual's addition (``ctmr_rms_norm``).

    ``h = x + residual``, ``y = h / sqrt(mean(h ** 2) + eps) * weight``. ``x`` is ``(rows, channels)`` or
    ``(tokens, heads, channels)`` in fp32, bf16 or fp16, up to 32,768 channels, any strides over rows; ``weight``
    ``(channels,)`` in fp32 or x's type. Returns ``y`` of x's type, or as ``ScaledRows`` with ``quantize`` (two
    dimensions; the bytes that the formula in 64 bits rounds to); with a residual ``(y, h)``, h rounded to x's type.
    The norm is taken of the unrounded sum (of 16-bit x: the sum in fp32, exact unless one term is 2^13 times the
    other); ``eps`` is an fp32 number. The bytes are exact for rows of a root mean square up to 2^126 and weights up
    to 2^15. ``sum_out`` may be ``x`` or ``residual``, and so may ``out``.
    """
    dtype, dims, shape = x.dtype, x.dim(), x.shape
    code = _FLOAT_CODES.get(dtype)
    if dims not in (2, 3) or code is None:
        raise ValueError(f"x must be a (rows, channels) or (tokens, heads, channels) fp32/bf16/fp16 tensor; got "
                         f"{tuple(shape)} {dtype}")
    dev, stream = _device_stream(x, "x")
    tokens, channels, heads = shape[0], shape[-1], shape[1] if dims == 3 else 1
    weight_at, weight_code = 0, 0
    if weight is not None:
        if weight.shape != (channels,) or weight.dtype not in (F32, dtype) or weight.get_device() != dev:
            raise ValueError(f"weight must be {channels} float32 or {dtype} values on cuda:{dev}")
        if not weight.is_contiguous():
            weight = weight.contiguous()
        weight_at, weight_code = weight.data_ptr(), _FLOAT_CODES[weight.dtype]
    dense = channels * heads, channels if heads > 1 else 0  # strides of what this call allocates
    new = ((tokens, channels), (channels, 1)) if dims == 2 else ((tokens, heads, channels), (channels * heads, channels, 1))
    x_at, r_at, s_at = _row_place(x, x, dev, "x"), (0, 0, 0), (0, 0, 0)
    if residual is not None:
        r_at = _row_place(residual, x, dev, "residual")
        if sum_out is None:
            sum_out = _empty(*new, dtype)
            s_at = (sum_out.data_ptr(), *dense)
        else:
            s_at = _row_place(sum_out, x, dev, "sum_out")
    elif sum_out is not None:
        raise ValueError("sum_out belongs to a residual")
    if quantize:
        if dims != 2 or out is not None:
            raise ValueError("8-bit rows are made of (rows, channels) tensors, and allocated by the call")
        out = _empty_rows8(tokens, channels)
        y_at = (out[0].data_ptr(), (channels + 15) & ~15, 0, *s_at, out[1].data_ptr(), 1, tokens)
    elif out is None:
        out = _empty(*new, dtype)
        y_at = (out.data_ptr(), *dense, *s_at, 0, 0, 0)
    else:
        y_at = (*_row_place(out, x, dev, "out"), *s_at, 0, 0, 0)
        if y_at[0] == s_at[0] and y_at[0]:
            raise ValueError("out and sum_out must be two tensors")
    LAUNCHES[0] += 1
    status = LIB.ctmr_rms_norm(_lib.pack_rms_norm(
        x_at[0], r_at[0], weight_at, code, weight_code, tokens, heads, channels, *x_at[1:], *r_at[1:], eps, *y_at), stream)
    if status:
        check(status, "rms_norm")
    return (out, sum_out) if residual is not None else out


def quantize_rows(x: torch.Tensor, *, gate: bool = False) -> ScaledRows:
    """Rows in 8 bits with a scale for every 128 channels (``ctmr_quantize_rows``).

    ``x`` is ``(rows, channels)`` in fp32, bf16 or fp16, any stride over rows; with ``gate`` ``(rows, 2 * channels)``,
    and what is rounded is ``silu(x[:, :channels]) * x[:, channels:]``. The bytes are those that the formula in 64
    bits rounds to. A group that holds an infinity, a NaN or a product past 448 * 2^127 becomes NaN as a whole.
    """
    code = _FLOAT_CODES.get(x.dtype)
    if x.dim() != 2 or code is None:
        raise ValueError(f"x must be a (rows, channels) fp32/bf16/fp16 tensor; got {tuple(x.shape)} {x.dtype}")
    dev, stream = _device_stream(x, "x")
    rows, channels = x.shape
    if channels > 1 and x.stride(1) != 1:
        raise ValueError("the channels of x must be contiguous")
    if gate:
        if channels % 2:
            raise ValueError(f"a gated pair has an even number of channels; got {channels}")
        channels //= 2
    out = _empty_rows8(rows, channels)
    LAUNCHES[0] += 1
    status = LIB.ctmr_quantize_rows(_lib.pack_quantize_rows(
        x.data_ptr(), code, rows, channels, gate, x.stride(0) if rows > 1 else 0, out[0].data_ptr(), (channels + 15) & ~15,
        out[1].data_ptr(), 1, rows), stream)
    if status:
        check(status, "quantize_rows")
    return out


def scaled_linear(x: ScaledRows, weight: ScaledWeight, bias: torch.Tensor | None = None, *,
                  out_dtype: torch.dtype = BF16, out: torch.Tensor | None = None) -> torch.Tensor:
    """A projection of 8-bit rows by an 8-bit weight, both with scales along blocks of 128 inputs
    (``ctmr_scaled_linear``): ``y = x weight^T + bias`` of the values that they stand for, fp32 sums, rounded once to
    ``out_dtype`` (bf16, fp16 or fp32).

    ``x`` comes from ``quantize_rows`` or ``rms_norm``, ``weight`` from ``scale_weight`` or a checkpoint; both scales
    may be any numbers whose products fp32 holds as normal ones, in any strides. Any number of rows, inputs and outputs. ``bias`` is fp32 or of the output's type.
    What is not finite in a row, or in an output's weights, stays in that row, or output.
    """
    values, x_scale = x
    w, w_scale = weight
    if values.dtype != E4M3 or w.dtype != E4M3 or values.dim() != 2 or w.dim() != 2 or w.shape[1] != values.shape[1]:
        raise ValueError(f"x and weight must be (rows, in) and (out, in) e4m3 tensors; got {tuple(values.shape)} "
                         f"{values.dtype} and {tuple(w.shape)} {w.dtype}")
    dev, stream = _device_stream(values, "x")
    rows, inner = values.shape
    outer = w.shape[0]
    blocks = (inner + 127) // 128
    if (x_scale.dtype != F32 or w_scale.dtype != F32 or x_scale.shape != (rows, blocks)
            or w_scale.shape != ((outer + 127) // 128, blocks)):
        raise ValueError(f"scales must be ({rows}, {blocks}) and ({(outer + 127) // 128}, {blocks}) float32; got "
                         f"{tuple(x_scale.shape)} {x_scale.dtype} and {tuple(w_scale.shape)} {w_scale.dtype}")
    if w.get_device() != dev or x_scale.get_device() != dev or w_scale.get_device() != dev:
        raise ValueError(f"weight and scales must be on cuda:{dev}")
    bias_at, bias_code = 0, 0
    if out is not None:
        out_dtype = out.dtype
    code = _FLOAT_CODES.get(out_dtype)
    if code is None:
        raise ValueError(f"the output is bf16, fp16 or fp32; got {out_dtype}")
    if bias is not None:
        if bias.shape != (outer,) or bias.dtype not in (F32, out_dtype) or bias.get_device() != dev:
            raise ValueError(f"bias must be {outer} float32 or {out_dtype} values on cuda:{dev}")
        if not bias.is_contiguous():
            bias = bias.contiguous()
        bias_at, bias_code = bias.data_ptr(), _FLOAT_CODES[bias.dtype]
    (xs, xc), (ws, wc) = values.stride(), w.stride()
    if out is None:
        out = _empty((rows, outer), (outer, 1), out_dtype)
        ys = outer
    else:
        if out.shape != (rows, outer) or out.get_device() != dev:
            raise ValueError(f"out must be ({rows}, {outer}) on cuda:{dev}")
        ys, yc = out.stride()
        if outer > 1 and yc != 1:
            raise ValueError("the columns of out must be contiguous")
    if inner > 1 and (xc != 1 or wc != 1):
        raise ValueError("the columns of x and weight must be contiguous")
    room = (inner + 15) & ~15  # a stride over an extent of one addresses nothing
    LAUNCHES[0] += 1
    status = LIB.ctmr_scaled_linear(_lib.pack_scaled_linear(
        values.data_ptr(), xs if rows > 1 else room, x_scale.data_ptr(), *x_scale.stride(), rows, inner, outer,
        w.data_ptr(), ws if outer > 1 else room, w_scale.data_ptr(), *w_scale.stride(), bias_at, bias_code,
        out.data_ptr(), code, ys if rows > 1 else outer), stream)
    if status:
        check(status, "scaled_linear")
    return out


def transform(
    x: torch.Tensor,
    *,
    x2: torch.Tensor | None = None,
    mode: int = _lib.TRANSFORM_COPY,
    affine: torch.Tensor | None = None,
    silu: bool = False,
    out_dtype: torch.dtype | None = None,
    out_channels: int | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Materialise ``mode(silu?(affine?(x ++ x2)))`` channels-last (``ctmr_transform``)."""
    b, c, d, h, w = (int(n) for n in x.shape)
    ctot = c + (int(x2.shape[1]) if x2 is not None else 0)
    if mode == _lib.TRANSFORM_TRILINEAR:
        od, oh, ow = 2 * d, 2 * h, 2 * w
    elif mode == _lib.TRANSFORM_AVGPOOL:
        od, oh, ow = d // 2, h // 2, w // 2
    else:
        od, oh, ow = d, h, w
    cout = out_channels or ctot
    if out is None:
        out = empty_ndhwc(b, cout, od, oh, ow, out_dtype or x.dtype, x.device)
    if affine is not None:
        affine = affine.to(dtype=F32).contiguous()
    desc = _lib.TransformDesc()
    desc.batch, desc.depth, desc.height, desc.width = b, d, h, w
    desc.x = view(x)
    desc.x2 = view(x2)
    desc.mode = mode
    desc.affine = affine.data_ptr() if affine is not None else None
    desc.silu = int(silu)
    desc.y = out.data_ptr()
    desc.y_dtype = _dtype_code(out.dtype, allow_f16=True)  # fp16 is a transform-only output (dense operands)
    desc.y_channels = int(out.shape[1])
    desc.y_cstride = rows_stride(out)
    _count(1)
    check(LIB.ctmr_transform(ctypes.byref(desc), _stream()), "transform")
    return out


def rflow_step(z: torch.Tensor, velocity: torch.Tensor, *, guidance: float | None, dt: float | torch.Tensor,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Guided Euler update ``z + dt * (u + s (c - u))`` (``ctmr_rflow_step``).

    ``z`` and ``velocity`` are fp32 and share one memory layout (``velocity`` holds
    the [cond, uncond] batch when guided); ``dt`` may be a device scalar tensor,
    read at execution time; ``out`` may be ``z``.
    """
    if z.dtype != F32 or velocity.dtype != F32:
        raise ValueError("rflow_step takes float32 tensors")
    # (a batch-1 tensor's batch stride is immaterial: e.g. the inner planes of a depth shard)
    first = 1 if int(z.shape[0]) == 1 else 0
    if z.stride()[first:] != velocity[: z.shape[0]].stride()[first:] or not (z.is_contiguous() or z.is_contiguous(
            memory_format=torch.channels_last_3d)):
        raise ValueError("z and velocity must be dense with the same memory layout")
    n = z.numel()
    guided = guidance is not None
    if velocity.numel() != (2 * n if guided else n):
        raise ValueError("velocity must hold the [cond, uncond] batch when guided")
    out = out if out is not None else torch.empty_like(z)
    dt_dev = dt.data_ptr() if isinstance(dt, torch.Tensor) else None
    _count(1)
    check(
        LIB.ctmr_rflow_step(z.data_ptr(), velocity.data_ptr(), n, float(guidance or 0.0), int(guided),
                            0.0 if dt_dev is not None else float(dt), dt_dev, out.data_ptr(), _stream()),
        "rflow_step",
    )
    return out


def window_accumulate(pred: torch.Tensor, acc: torch.Tensor, wsum: torch.Tensor, *, origin: tuple[int, int, int],
                      tables: list[torch.Tensor], scale: int, floor: float) -> None:
    """Add one decoded window, Gaussian-weighted, into the blend (``ctmr_window_accumulate``).

    ``pred`` is the channels-last window ``(B, C, wd, wh, ww)``; ``acc`` is the
    fp32 NDHWC accumulator ``(B, OD, OH, OW, C)`` and ``wsum`` the fp32 weight
    sum ``(OD, OH, OW)``; ``tables`` are the per-axis 1-D Gaussians over the
    latent ROI, resized by ``scale`` with nearest indexing.
    """
    b, c, wd, wh, ww = (int(n) for n in pred.shape)
    od, oh, ow = (int(n) for n in acc.shape[1:4])
    if acc.dtype != F32 or wsum.dtype != F32 or not acc.is_contiguous() or not wsum.is_contiguous():
        raise ValueError("window accumulators must be contiguous float32")
    gz, gy, gx = (t.to(F32).contiguous() for t in tables)
    _count(1)
    check(
        LIB.ctmr_window_accumulate(view(pred), b, wd, wh, ww, int(origin[0]), int(origin[1]), int(origin[2]), od, oh,
                                   ow, gz.data_ptr(), gy.data_ptr(), gx.data_ptr(), int(scale), float(floor),
                                   acc.data_ptr(), wsum.data_ptr(), _stream()),
        "window_accumulate",
    )


def window_finalize(acc: torch.Tensor, wsum: torch.Tensor, *, origin: tuple[int, int, int],
                    extent: tuple[int, int, int]) -> torch.Tensor:
    """``acc / wsum`` over the crop at ``origin`` as a contiguous NCDHW fp32 tensor (``ctmr_window_finalize``)."""
    b, od, oh, ow, c = (int(n) for n in acc.shape)
    out = torch.empty((b, c, *(int(e) for e in extent)), dtype=F32, device=acc.device)
    _count(1)
    check(
        LIB.ctmr_window_finalize(acc.data_ptr(), wsum.data_ptr(), out.data_ptr(), b, c, od, oh, ow, int(origin[0]),
                                 int(origin[1]), int(origin[2]), int(extent[0]), int(extent[1]), int(extent[2]),
                                 _stream()),
        "window_finalize",
    )
    return out
