"""The registered ops and the two calls that reach every op's implementation: :func:`prebuild` and :func:`release`.

:data:`OPS` names every ``cake/<op>.py`` of this package.  :func:`op_spec` imports only the thin op module, never
its implementation (reference: miles_ext_kernels/cake/_runtime/registry.py:26-158; the reference lists 13 ops, this
package ships those of the gated-delta-rule path and, without a counterpart there, the other ops of a recurrent
layer's training path).
"""

from __future__ import annotations

import sys
from collections.abc import Iterator, Mapping, Set
from importlib import import_module
from pathlib import Path
from typing import Any

from . import loader, workspace
from .spec import OpSpec

__all__ = ["OPS", "op_spec", "prebuild", "release"]

OPS: tuple[str, ...] = ("gdn", "kda", "gated_rmsnorm", "conv1d", "layer_norm", "linear_recurrence")

# <pkg>.cake: op modules are its submodules, implementations those of its _impl package
_SOURCE = __name__.rsplit(".", 2)[0]
# What prebuild returned in this process, by (op, device, toolkit, cache directory, model parameters, op options).
_PREBUILT: dict[tuple[Any, ...], tuple[Path, ...]] = {}


def op_spec(op: str) -> OpSpec:
    """The ``OP`` of ``cake.<op>``; ``KeyError`` for an op that is not registered."""
    if op not in OPS:
        raise KeyError(f"no cake op {op!r}; the ops are {OPS}")
    qualified = f"{_SOURCE}.{op}"
    module = sys.modules.get(qualified)
    if module is None or not hasattr(module, "OP"):
        module = import_module(qualified)
    return module.OP


def _hashable(value: Any) -> Any:
    """``value`` compared by content and type (``12`` and ``12.0`` differ); containers become hashable."""
    if isinstance(value, Mapping):
        return frozenset((key, _hashable(item)) for key, item in value.items())
    if isinstance(value, Set):
        return frozenset(_hashable(item) for item in value)
    if isinstance(value, (list, tuple)):
        return tuple(_hashable(item) for item in value)
    return type(value), value


def _cuda_target(device: Any) -> tuple[int, str] | None:
    """``(index, architecture)`` of the CUDA ``device`` (an index, ``"cuda"``, ``"cuda:N"``, a ``torch.device`` or
    ``None`` for the current one); ``None`` when it cannot be told or is not served."""
    try:
        import torch

        if not isinstance(device, int):
            where = torch.device("cuda" if device is None else device)
            if where.type != "cuda":
                return None
            device = torch.cuda.current_device() if where.index is None else where.index
        arch = loader.ARCH_BY_CAPABILITY.get(tuple(torch.cuda.get_device_capability(device)))
    except (ImportError, AssertionError, RuntimeError, TypeError, ValueError):
        return None
    return None if arch is None else (device, arch)


def _memo_key(op: str, device: Any, model_params: Mapping[str, Any]) -> tuple[Any, ...] | None:
    """The key under which :func:`prebuild` remembers its result; ``None`` when it cannot (no CUDA device, no
    toolkit, an unhashable model parameter) -- the op's own prebuild then reports the problem."""
    from . import config  # config imports this module

    target = _cuda_target(device)
    if target is None:
        return None
    try:
        toolkit = loader._toolkit()
    except RuntimeError:
        return None
    options = {flag.dest: config.option(op, flag.dest) for flag in op_spec(op).flags}
    key = (op, target, toolkit, str(loader.cache_dir()), _hashable(model_params), _hashable(options))
    try:
        hash(key)
    except TypeError:
        return None
    return key


def prebuild(op: str, /, *, device: Any = None, max_workers: int | None = None, **model_params: Any) -> list[Path]:
    """Build every library ``op`` may launch for ``model_params`` on ``device`` (default: the current device).

    Afterwards no call of ``op`` with these model parameters compiles on that device, whatever the variant, token
    count or route.  ``model_params`` are model shapes only, never a token count or a variant.  Unsupported
    parameters raise ``ValueError``, an unsupported device ``NotImplementedError``, a toolkit too old
    ``RuntimeError``.  Idempotent: the paths are remembered until :func:`release`, so the call miles makes per layer
    returns at once.
    """
    op_spec(op)
    implementation = import_module(f"{_SOURCE}._impl.{op}")
    model_params = {name: tuple(v) if isinstance(v, Iterator) else v for name, v in model_params.items()}
    key = _memo_key(op, device, model_params)
    if key is not None and key in _PREBUILT:
        return list(_PREBUILT[key])
    paths = tuple(implementation.prebuild(device=device, max_workers=max_workers, **model_params))
    if key is not None:
        _PREBUILT[key] = paths
    return list(paths)


def release(op: str | None = None) -> int:
    """Free the scratch pool (of every op, or of ``op``) and the caches of every imported implementation; forget
    what :func:`prebuild` remembered.  Returns the bytes freed from the pool (``torch.cuda.empty_cache()`` is the
    caller's)."""
    names = OPS if op is None else (op_spec(op).name,)
    for key in [key for key in _PREBUILT if op is None or key[0] == op]:
        del _PREBUILT[key]
    freed = workspace.release(op)
    for name in names:
        implementation = sys.modules.get(f"{_SOURCE}._impl.{name}")
        if implementation is not None:
            implementation.release()
    return freed
