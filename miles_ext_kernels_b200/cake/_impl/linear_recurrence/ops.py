"""The gated linear recurrence on the sm_100a kernels: ``gated_linear_recurrence``, ``gated_linear_recurrence_step``,
``check_supported``, ``prebuild``, ``release``.

Per channel, with ``a = exp(g)`` and the state of a sequence starting at ``h0`` (or zero)::

    h[t] = a[t] h[t-1] + x[t],   y[t] = h[t]
    dh[t] = dy[t] + a[t+1] dh[t+1],   dx = dh,   dg[t] = dh[t] a[t] h[t-1],   dh0 = a[0] dh[0]

States and sums in FP32, one rounding per output; a decay below e^-86.98 = 1.67e-38, at FP32's end, counts as zero.  The
autograd node keeps ``x``, ``g`` and the FP32 state after every tile of 128 tokens; the backward recomputes the states
inside a tile, so ``dg`` does not see a rounded ``y``.
"""

from __future__ import annotations

from pathlib import Path
from typing import Any

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.graph import increment_version

from ..._runtime import loader, registry, workspace
from ..gdn import native
from ..gdn.native import pointer
from ..rows import TYPES, check_device, forward_mode, on_device, once_differentiable, recorded

__all__ = ["check_supported", "gated_linear_recurrence", "gated_linear_recurrence_step", "prebuild", "release"]

OP = "linear_recurrence"
_fwd = native.Entry("linear_recurrence_fwd", "pipiplllllllplppp")
_bwd = native.Entry("linear_recurrence_bwd", "ppipipplllllllplppppp")
_step = native.Entry("linear_recurrence_step", "pipippipllllll")
_MAX_TOKENS, _MAX_CHANNELS = 1 << 30, 1 << 23


def check_supported(channels: int, dtype: torch.dtype, gate_dtype: torch.dtype = torch.float32, *, device=None) -> None:
    """Raise ``ValueError`` unless the kernels run this recurrence on ``device`` (default: the current CUDA device): 1 to
    2^23 channels, inputs and gates each in BF16, FP16 or FP32, a B200."""
    _check_types(dtype, gate_dtype)
    _check_channels(channels)
    check_device(OP, "the linear recurrence kernels", device)


def _check_types(dtype: torch.dtype, gate_dtype: torch.dtype) -> None:
    if dtype not in TYPES or gate_dtype not in TYPES:
        raise ValueError(f"linear_recurrence takes x and g in BF16, FP16 or FP32, got {dtype} and {gate_dtype}")


def _check_channels(channels: int) -> None:
    if not 1 <= channels <= _MAX_CHANNELS:
        raise ValueError(f"linear_recurrence takes 1 to 2^23 channels, got {channels}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t [B, T, ...]`` as ``[B, T, C]`` with unit stride over the channels: read in place where it can be, else copied
    once."""
    batch, tokens = t.shape[:2]
    if t.dim() != 3:
        try:
            t = t.view(batch, tokens, -1)
        except RuntimeError:
            t = t.reshape(batch, tokens, -1)
    if (t.stride(2) != 1 and t.shape[2] > 1) or t.stride(0) < 0 or t.stride(1) < 0:
        t = t.contiguous()
    return t


def _flat_rows(t: torch.Tensor, channels: int) -> torch.Tensor:
    """``t [R, ...]`` as ``[R, C]`` with unit stride over the channels, in place where it can be, else copied once."""
    if t.dim() != 2:
        t = t.reshape(t.shape[0], channels)  # a view where the trailing dimensions merge
    if t.stride(1) != 1 and channels > 1:
        t = t.contiguous()
    return t


def _words(batch: int, tokens: int, channels: int) -> int:
    """How many floats carry the state from tile to tile: 0 where one tile holds all tokens."""
    tile = native.library().mek_linear_recurrence_tile()
    return 2 * batch * -(-tokens // tile) * channels + 1 if tokens > tile else 0


def _forward(x, g, h0, cu, want_final, train):
    """``(y, final, states)`` for ``x``, ``g [B, T, C]``; ``states`` holds the state after every tile for the backward
    (``None`` where one tile holds all tokens)."""
    batch, tokens, channels = x.shape
    device = x.device
    sequences = batch if cu is None else cu.numel() - 1
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    final = x.new_empty((sequences, channels), dtype=torch.float32) if want_final else None
    with on_device(device):
        words = _words(batch, tokens, channels)
        states = None
        if words:
            states = (x.new_empty(words, dtype=torch.float32) if train
                      else workspace.take(OP, "states", (words,), torch.float32, device))
        _fwd(device, x.data_ptr(), TYPES[x.dtype], g.data_ptr(), TYPES[g.dtype], y.data_ptr(), batch, tokens, channels,
             *x.stride()[:2], *g.stride()[:2], pointer(cu), sequences, pointer(h0), pointer(final), pointer(states))
    return y, final, states


def _gradients(ctx, dy, d_final):
    x, g, h0, cu, states = ctx.saved_tensors
    batch, tokens, channels = x.shape
    device = x.device
    sequences = batch if cu is None else cu.numel() - 1
    dy = dy.contiguous()
    d_final = None if d_final is None else d_final.contiguous()
    dx = torch.empty_like(dy)
    dg = torch.empty_like(g, memory_format=torch.contiguous_format)
    dh0 = torch.empty_like(h0) if ctx.needs_input_grad[2] else None
    with on_device(device):
        scratch = None
        if states is not None:
            scratch = workspace.take(OP, "scratch", states.shape, torch.float32, device)
        _bwd(device, dy.data_ptr(), x.data_ptr(), TYPES[x.dtype], g.data_ptr(), TYPES[g.dtype], dx.data_ptr(),
             dg.data_ptr(), batch, tokens, channels, *x.stride()[:2], *g.stride()[:2], pointer(cu), sequences,
             pointer(h0), pointer(d_final), pointer(states), pointer(dh0), pointer(scratch))
    return dx, dg, dh0, None, None


class _GatedLinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, g, h0, cu, want_final):
        train = any(ctx.needs_input_grad)
        y, final, states = _forward(x, g, h0, cu, want_final, train)
        if train:
            ctx.save_for_backward(x, g, h0, cu, states)
        return y, final

    backward = staticmethod(once_differentiable(_gradients))


def _no_tokens(x, g, h0, sequences, channels, want_final):
    """A call without tokens: the states pass through (and the empty output hangs on both empty inputs)."""
    y = x + g.to(x.dtype)
    final = None
    if want_final:
        final = x.new_zeros((sequences, channels), dtype=torch.float32) if h0 is None else h0.clone()
    return y, final


def gated_linear_recurrence(
    x: torch.Tensor,
    g: torch.Tensor,
    initial_state: torch.Tensor | None = None,
    output_final_state: bool = False,
    cu_seqlens: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Autograd-enabled ``h[t] = exp(g[t]) h[t-1] + x[t]`` along the second dimension; returns ``(y, final_state)``.

    ``x``: BF16, FP16 or FP32 ``[B, T, ...]``; every element of the trailing dimensions is a channel of its own.  ``g``:
    the log decay in nats, ``x``'s shape, in any of the three types (expand a gate that channels share; autograd sums
    its gradient).  A gate may be positive; a state that is not zero comes out infinite where a sequence grows by more
    than e^88 within 128 tokens, FP32's range.  Both are read in place when the channels have unit stride, whatever the
    token and batch strides, else copied once.  ``initial_state``: FP32 ``[N, ...]`` or ``None`` (zero); ``N`` is ``B``, or
    the number of sequences that ``cu_seqlens`` (``[N + 1]`` prefix sums of their lengths, on ``x``'s device, ``B = 1``)
    packs into the one row.  A sequence may be empty: its state passes through.  Tokens behind the last sequence belong to
    none: their ``y`` and gradients are zero.  ``final_state``: FP32 ``[N, ...]`` when ``output_final_state``, else
    ``None``.  Not twice differentiable, and without a forward-mode derivative."""
    if x.dim() < 3:
        raise ValueError(f"linear_recurrence: x must be [B, T, ...channels]; got {tuple(x.shape)}")
    if g.shape != x.shape:
        raise ValueError(f"linear_recurrence: g must have x's shape {tuple(x.shape)}; got {tuple(g.shape)}")
    _check_types(x.dtype, g.dtype)
    batch, tokens, *trailing = x.shape
    channels = 1
    for extent in trailing:
        channels *= extent
    _check_channels(channels)
    if batch < 1 or tokens > _MAX_TOKENS:
        raise ValueError(f"linear_recurrence takes at least one batch row of at most 2^30 tokens; got {tuple(x.shape)}")
    sequences = batch
    if cu_seqlens is not None:
        if batch != 1:
            raise ValueError(f"linear_recurrence: cu_seqlens packs the sequences of one row; x has {batch}")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise ValueError("linear_recurrence: cu_seqlens must be int32 or int64 [num_sequences + 1]")
        sequences = cu_seqlens.numel() - 1
    if initial_state is not None:
        if tuple(initial_state.shape) != (sequences, *trailing) or initial_state.dtype != torch.float32:
            raise ValueError(f"linear_recurrence: initial_state must be FP32 {(sequences, *trailing)}; got "
                             f"{initial_state.dtype} {tuple(initial_state.shape)}")
    for name, t in (("g", g), ("initial_state", initial_state), ("cu_seqlens", cu_seqlens)):
        if t is not None and t.device != x.device:
            raise ValueError(f"linear_recurrence: {name} is on {t.device}, x on {x.device}")
    if not x.is_cuda:
        raise ValueError("linear_recurrence: x must be a CUDA tensor")
    h0 = None if initial_state is None else initial_state.reshape(sequences, channels).contiguous()
    if tokens == 0:
        y, final = _no_tokens(x, g, h0, sequences, channels, output_final_state)
    else:
        cu = None if cu_seqlens is None else cu_seqlens.to(torch.int32).contiguous()
        xv, gv = _rows(x), _rows(g)
        if torch.is_grad_enabled() and (x.requires_grad or g.requires_grad or (h0 is not None and h0.requires_grad)
                                        ) or recorded():
            y, final = _GatedLinearRecurrence.apply(xv, gv, h0, cu, bool(output_final_state))
        else:
            y, final, _ = _forward(xv, gv, h0, cu, output_final_state, False)
    if len(trailing) > 1:
        y = y.view(x.shape)
        final = None if final is None else final.view(sequences, *trailing)
    return y, final


def _explain_step(x, g, state, state_indices):
    """Raise the ``ValueError`` that says what is wrong with a step's arguments; returns where nothing is."""
    if x.dim() < 2:
        raise ValueError(f"linear_recurrence: x must be [rows, ...channels]; got {tuple(x.shape)}")
    if g.shape != x.shape:
        raise ValueError(f"linear_recurrence: g must have x's shape {tuple(x.shape)}; got {tuple(g.shape)}")
    _check_types(x.dtype, g.dtype)
    rows, *trailing = x.shape
    channels = 1
    for extent in trailing:
        channels *= extent
    _check_channels(channels)
    if state.dim() != x.dim() or list(state.shape[1:]) != trailing or state.dtype != torch.float32 or state.shape[0] < 1:
        raise ValueError(f"linear_recurrence: state must be FP32 [N, {', '.join(map(str, trailing))}]; got {state.dtype} "
                         f"{tuple(state.shape)}")
    pool = state.shape[0]
    if state_indices is None:
        if rows > pool:
            raise ValueError(f"linear_recurrence: {rows} rows need as many states without state_indices; got {pool}")
    elif tuple(state_indices.shape) != (rows,) or state_indices.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"linear_recurrence: state_indices must be int32 or int64 [{rows}]; got {state_indices.dtype} "
                         f"{tuple(state_indices.shape)}")
    if torch.is_grad_enabled() and (x.requires_grad or g.requires_grad or state.requires_grad):
        raise ValueError("linear_recurrence: the step updates its state in place and has no gradient; use "
                         "gated_linear_recurrence, or torch.no_grad()")
    if forward_mode():
        if any(unpack_dual(t).tangent is not None for t in (x, g, state)):
            raise ValueError("linear_recurrence: the step updates its state in place and has no forward-mode derivative")
    elif recorded():
        raise ValueError("linear_recurrence: the step updates its state in place, which a trace would not hold")
    for name, t in (("g", g), ("state", state), ("state_indices", state_indices)):
        if t is not None and t.device != x.device:
            raise ValueError(f"linear_recurrence: {name} is on {t.device}, x on {x.device}")
    if not x.is_cuda:
        raise ValueError("linear_recurrence: x must be a CUDA tensor")


def gated_linear_recurrence_step(x: torch.Tensor, g: torch.Tensor, state: torch.Tensor,
                                 state_indices: torch.Tensor | None = None) -> torch.Tensor:
    """One token of every row: ``state[i] = exp(g) state[i] + x`` in place; returns the new state as ``y`` in ``x``'s type.

    ``x``: BF16, FP16 or FP32 ``[R, ...]``; ``g``: the log decay in nats, ``x``'s shape, in any of the three types.
    ``state``: the FP32 pool ``[N, ...]``, dense inside a slot (any stride between them), updated in place, so not for
    autograd (a recorded call that saved the pool, as its ``initial_state`` for example, raises in its backward).
    ``state_indices``: int32 or int64 ``[R]``, the slot of every row (``None``: row ``r`` uses slot ``r`` and ``N >= R``).
    A row whose index is outside ``[0, N)``, -1 for example, is padding: no state changes and its ``y`` is zero.  Rows that
    name one slot are applied one after the other, in row order."""
    device, shape, trailing = x.device, x.shape, state.shape[1:]
    if not (  # one test for the usual call; _explain_step says what is wrong with any other
        x.is_cuda and x.dim() == 2 and g.shape == shape and trailing == shape[1:] and state.dtype is torch.float32
        and x.dtype in TYPES and g.dtype in TYPES and g.device == device and state.device == device
        and state_indices is not None and state_indices.dtype in (torch.int32, torch.int64)
        and state_indices.shape == shape[:1] and state_indices.device == device and 0 < shape[1] <= _MAX_CHANNELS
        and state.shape[0] > 0
        and not ((x.requires_grad or g.requires_grad or state.requires_grad) and torch.is_grad_enabled())
        and not recorded()
    ):
        _explain_step(x, g, state, state_indices)
    rows, pool = shape[0], state.shape[0]
    channels = shape[1:].numel()
    pooled = state
    if state.dim() > 2:
        try:
            pooled = state.view(pool, channels)
        except RuntimeError:
            pooled = None
    if pooled is None or (channels > 1 and pooled.stride(1) != 1) or (pool > 1 and pooled.stride(0) < channels):
        raise ValueError(f"linear_recurrence: a state must be dense inside its slot; strides {state.stride()}")
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    if rows == 0:
        return y
    xv, gv = _flat_rows(x, channels), _flat_rows(g, channels)
    slots = None if state_indices is None else state_indices.contiguous()
    with on_device(device):
        _step(device, xv.data_ptr(), TYPES[x.dtype], gv.data_ptr(), TYPES[g.dtype], pooled.data_ptr(), pointer(slots),
              slots is not None and slots.dtype == torch.int64, y.data_ptr(), rows, pool, channels, xv.stride(0),
              gv.stride(0), pooled.stride(0))
    if not state.is_inference():  # a graph that saved the pool as it was has to hear of the change
        increment_version(state)
    return y


def prebuild(*, device: Any = None, max_workers: int | None = None) -> list[Path]:
    """Build (or find) the native library for ``device``."""
    arch = loader.device_arch(device)
    loader.check_toolkit(arch, "the linear recurrence kernels")
    return loader.prebuild_libraries(registry.op_spec(OP).packages, arch, max_workers=max_workers)


def release() -> None:
    """Nothing is kept between calls besides the workspace pool (emptied by the runtime) and the library handle."""
