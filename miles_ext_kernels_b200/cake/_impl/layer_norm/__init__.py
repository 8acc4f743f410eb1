"""The implementation of ``cake.layer_norm``."""

from ..._runtime import loader

loader.install_op("layer_norm")

from .ops import check_supported, layer_norm, prebuild, release  # noqa: E402

__all__ = ["check_supported", "layer_norm", "prebuild", "release"]
