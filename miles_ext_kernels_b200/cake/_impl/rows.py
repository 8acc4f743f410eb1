"""What the row operators (LayerNorm, the gated norm's checkpoint, the linear recurrence) share on the host: element
types as the C ABI numbers them, checkpoint formats, alignment, the device check and the device guard."""

from __future__ import annotations

from contextlib import nullcontext
from typing import Any

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable as _guarded

from .._runtime import loader

__all__ = ["CHECKPOINTS", "TYPES", "aligned", "check_device", "checkpoint_format", "forward_mode", "on_device",
           "once_differentiable", "recorded"]

# element types of the C ABI
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
# how a forward may keep what its backward needs: as it came, or in 8 bits
CHECKPOINTS = (None, "e4m3")

_NOTHING = nullcontext()
_tracing_state = torch._C._get_tracing_state


def forward_mode() -> bool:
    """Whether tensors may carry forward-mode tangents."""
    return forward_ad._current_level >= 0


def recorded() -> bool:
    """Whether something besides the backward follows the call -- forward mode, a trace -- so that it has to go through its
    autograd function even where nothing requires a gradient: the kernels work on addresses, which neither sees."""
    return forward_ad._current_level >= 0 or _tracing_state() is not None


def on_device(device: torch.device) -> Any:
    """``torch.cuda.device(device)``, without its cost where ``device`` is the current one."""
    if device.index is None or device.index == torch.cuda.current_device():
        return _NOTHING
    return torch.cuda.device(device)


def aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` dense and on a 16-byte boundary, copied once where it is not (a slice of a flat buffer is contiguous and may
    start anywhere)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def once_differentiable(backward: Any) -> Any:
    """``torch.autograd.function.once_differentiable``, which costs as much as a small backward's launch, where it can
    matter: a backward that is itself being recorded (``create_graph=True``)."""
    guarded = _guarded(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


def checkpoint_format(op: str, checkpoint: Any) -> bool:
    """Whether ``checkpoint`` asks for e4m3 codes; ``ValueError`` for anything but the formats of ``CHECKPOINTS``."""
    if checkpoint not in CHECKPOINTS:
        raise ValueError(f"{op}: checkpoint must be one of {CHECKPOINTS}, got {checkpoint!r}")
    return checkpoint is not None


def check_device(op: str, what: str, device: Any = None) -> None:
    """Raise ``ValueError`` unless the kernels run on ``device`` (default: the current CUDA device)."""
    served = tuple(loader.ARCH_BY_CAPABILITY)
    if not torch.cuda.is_available():
        raise ValueError(f"{op} needs a CUDA device of compute capability {served}")
    capability = tuple(torch.cuda.get_device_capability(device))
    arch = loader.ARCH_BY_CAPABILITY.get(capability)
    if arch is None:
        raise ValueError(f"{op} runs on compute capability {served}, not {capability}")
    loader.check_toolkit(arch, what)
