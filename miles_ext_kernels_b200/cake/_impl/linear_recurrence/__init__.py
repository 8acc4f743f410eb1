"""The implementation of ``cake.linear_recurrence``."""

from ..._runtime import loader

loader.install_op("linear_recurrence")

from .ops import (  # noqa: E402
    check_supported,
    gated_linear_recurrence,
    gated_linear_recurrence_step,
    prebuild,
    release,
)

__all__ = ["check_supported", "gated_linear_recurrence", "gated_linear_recurrence_step", "prebuild", "release"]
