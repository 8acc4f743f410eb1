"""LayerNorm on the sm_100a kernels: ``layer_norm``, ``check_supported``, ``prebuild``, ``release``.

Per row of ``x [..., C]`` (BF16, FP16 or FP32) with a weight and a bias ``[C]``, each optional::

    unit = (x - mean(x)) / sqrt(var(x) + eps)            # FP32, var about the mean
    y    = unit * weight + bias                          # FP32, one rounding to x's type

    dn = dy * weight;   dx = (dn - mean(dn) - unit * mean(dn * unit)) / sqrt(var(x) + eps)
    dweight = sum over rows of dy * unit;   dbias = sum over rows of dy

The autograd node keeps ``x`` and two FP32 statistics a row, or, with ``checkpoint="e4m3"``, the rows of ``unit`` as
e4m3 codes and one statistic: half the bytes of a BF16 ``x``, for gradients that take ``unit`` rounded to 3 mantissa
bits (off by at most 2^-4 of the value; ``|unit| <= sqrt(C)``, so the codes need no scale).  ``y`` does not change.  The
parameter gradients are summed in FP32 per block and in FP64 across the blocks, in an order fixed by the extents and by
whether the rows start on 16-byte boundaries.
"""

from __future__ import annotations

from ctypes import c_int64
from pathlib import Path
from typing import Any

import torch

from ..._runtime import loader, registry, workspace
from ..gdn import native
from ..gdn.native import pointer
from ..rows import TYPES, check_device, checkpoint_format, on_device, once_differentiable, recorded

__all__ = ["check_supported", "layer_norm", "prebuild", "release"]

OP = "layer_norm"
_fwd = native.Entry("layer_norm_fwd", "pippipppplllf")
_bwd = native.Entry("layer_norm_bwd", "ppippppipppplll")
_CHECKPOINT_WIDTH = 200704  # 448^2: a wider row's largest value could exceed e4m3


def check_supported(width: int, dtype: torch.dtype, param_dtype: torch.dtype | None = None, *, checkpoint: str | None = None,
                    device=None) -> None:
    """Raise ``ValueError`` unless the kernels run this LayerNorm on ``device`` (default: the current CUDA device): rows
    of 1 to 2^24 elements (200,704 with a checkpoint) in BF16, FP16 or FP32, parameters in one of these types, a B200."""
    _check_types(dtype, param_dtype or dtype)
    _check_width(width, checkpoint_format(OP, checkpoint))
    check_device(OP, "the LayerNorm kernels", device)


def _check_types(dtype: torch.dtype, param_dtype: torch.dtype) -> None:
    if dtype not in TYPES:
        raise ValueError(f"layer_norm takes BF16, FP16 or FP32 rows, got {dtype}")
    if param_dtype not in TYPES:
        raise ValueError(f"layer_norm takes a BF16, FP16 or FP32 weight and bias, got {param_dtype}")


def _check_width(width: int, keep: bool) -> None:
    if not 1 <= width <= (_CHECKPOINT_WIDTH if keep else 1 << 24):
        raise ValueError(f"layer_norm normalizes rows of 1 to 2^24 elements ({_CHECKPOINT_WIDTH} with an 8-bit "
                         f"checkpoint), got {width}")


def _rows_of(x: torch.Tensor) -> torch.Tensor:
    """``x`` as ``[rows, C]`` with unit stride inside a row: read in place where the leading dimensions merge to one
    row stride, else copied once."""
    if x.is_contiguous() and x.dim() == 2:
        return x
    width = x.shape[-1]
    if x.dim() != 2:
        try:
            x = x.view(-1, width)
        except RuntimeError:
            x = x.reshape(-1, width)
    if (x.stride(1) != 1 and width > 1) or (x.stride(0) < width and x.shape[0] > 1):
        x = x.contiguous()
    return x


def _forward(x, weight, bias, eps, keep, train):
    """``(y, kept)``: ``kept`` is what the backward reads -- ``(x, None, statistics)`` or ``(None, codes, statistics)``
    with the statistics ``[mean, rstd]`` or ``[rstd]`` of the rows, ``None`` when there will be none."""
    width = x.shape[-1]
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    rows = x.numel() // width
    mean = rstd = codes = statistics = None
    if train:
        statistics = x.new_empty((1 if keep else 2, rows), dtype=torch.float32)
        rstd = statistics.data_ptr() + (0 if keep else 4 * rows)
        if keep:
            codes = x.new_empty((rows, width), dtype=torch.uint8)
        else:
            mean = statistics.data_ptr()
    if rows:
        xv = _rows_of(x)
        param = weight if weight is not None else bias
        with on_device(x.device):
            _fwd(x.device, xv.data_ptr(), TYPES[x.dtype], pointer(weight), pointer(bias),
                 TYPES[param.dtype] if param is not None else 0, y.data_ptr(), mean, rstd, pointer(codes), rows, width,
                 xv.stride(0), eps)
    return y, ((None if keep else x), codes, statistics) if train else None


def _gradients(ctx, dy):
    x, codes, statistics, weight, bias = ctx.saved_tensors
    device = dy.device
    width = ctx.shape[-1]
    rows = statistics.shape[1]
    dy = dy.contiguous()
    dx = torch.empty_like(dy)
    _, want_dw, want_db, _, _ = ctx.needs_input_grad
    dw = torch.empty_like(weight) if want_dw else None
    db = torch.empty_like(bias) if want_db else None
    if not rows:
        for grad in (dw, db):
            if grad is not None:
                grad.zero_()
        return dx, dw, db, None, None
    xv = None if x is None else _rows_of(x)
    kind = TYPES[dy.dtype]
    param = weight if weight is not None else bias
    with on_device(device):
        partial = None
        if want_dw or want_db:
            blocks = native.library().mek_layer_norm_partial_rows(c_int64(rows), c_int64(width), kind)
            partial = workspace.take(OP, "partial", (blocks, 2, width), torch.float32, device)
        first = statistics.data_ptr()
        _bwd(device, dy.data_ptr(), pointer(xv), kind, pointer(codes), None if x is None else first,
             first if x is None else first + 4 * rows, pointer(weight), TYPES[param.dtype] if param is not None else 0,
             dx.data_ptr(), pointer(partial), pointer(dw), pointer(db), rows, width, 0 if xv is None else xv.stride(0))
    return dx, dw, db, None, None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep):
        y, kept = _forward(x, weight, bias, eps, keep, any(ctx.needs_input_grad))
        if kept is not None:
            ctx.save_for_backward(*kept, weight, bias)
            ctx.shape = x.shape
        return y

    backward = staticmethod(once_differentiable(_gradients))


def _explain(x, weight, bias, keep):
    """Raise the ``ValueError`` that says what is wrong with a call's arguments; returns where nothing is."""
    if x.dim() < 1:
        raise ValueError("layer_norm: x must have at least one dimension")
    width = x.shape[-1]
    _check_width(width, keep)
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if tuple(p.shape) != (width,):
            raise ValueError(f"layer_norm: {name} must be [{width}]; got {tuple(p.shape)}")
        if p.device != x.device:
            raise ValueError(f"layer_norm: {name} is on {p.device}, x on {x.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"layer_norm: weight and bias must have one type; got {weight.dtype} and {bias.dtype}")
    param = weight if weight is not None else bias
    _check_types(x.dtype, x.dtype if param is None else param.dtype)
    if not x.is_cuda:
        raise ValueError("layer_norm: x must be a CUDA tensor")


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5, *,
               checkpoint: str | None = None) -> torch.Tensor:
    """Autograd-enabled LayerNorm over the last dimension of ``x [..., C]``; returns ``y`` of ``x``'s shape and type.

    ``x``: BF16, FP16 or FP32 on a B200, read in place when its rows have unit stride inside and one stride between
    them, else copied once.  ``weight``, ``bias``: ``[C]``, each optional, both of one type out of the three, which their
    gradients have too.  ``checkpoint``: ``None`` keeps ``x`` for the backward, ``"e4m3"`` keeps the normalised rows in 8
    bits instead (``C`` up to 200,704).  Not twice differentiable, and
    without a forward-mode derivative."""
    keep = checkpoint is not None and checkpoint_format(OP, checkpoint)
    if not (  # one test for the usual call; _explain says what is wrong with any other
        weight is not None and bias is not None and x.is_cuda and x.dim() > 0 and x.dtype in TYPES and weight.dtype in TYPES
        and weight.dtype is bias.dtype and weight.shape == bias.shape == x.shape[-1:]
        and weight.device == bias.device == x.device and 0 < x.shape[-1] <= _CHECKPOINT_WIDTH
    ):
        _explain(x, weight, bias, keep)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)
            ) and torch.is_grad_enabled() or recorded():
        return _LayerNorm.apply(x, weight, bias, float(eps), keep)
    return _forward(x, weight, bias, float(eps), keep, False)[0]


def prebuild(*, device: Any = None, max_workers: int | None = None) -> list[Path]:
    """Build (or find) the native library for ``device``."""
    arch = loader.device_arch(device)
    loader.check_toolkit(arch, "the LayerNorm kernels")
    return loader.prebuild_libraries(registry.op_spec(OP).packages, arch, max_workers=max_workers)


def release() -> None:
    """Nothing is kept between calls besides the workspace pool (emptied by the runtime) and the library handle."""
