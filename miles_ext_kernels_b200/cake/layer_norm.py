"""LayerNorm over the last dimension, forward and backward, with the reduction of the weight's and the bias's gradients,
on hand-written sm_100a kernels; on request the backward works from an 8-bit checkpoint of the normalised rows.

An op of this package, without a counterpart in the reference and without a miles argument that selects it: call it in
the place of ``torch.nn.functional.layer_norm``.  Both variants (``det``, ``fast``) run the same kernels: the parameter
gradients are summed in a fixed order, so identical inputs give identical bits.

Importing this module imports neither torch nor the implementation.
"""

from ._runtime.spec import OpSpec, lazy_exports

OP = OpSpec(
    name="layer_norm",
    summary="LayerNorm over rows of any width, forward + backward, optional 8-bit checkpoint",
    variants=("det", "fast"),
    packages=("libmek_b200",),
    exports=("check_supported", "layer_norm"),
)

__all__, __getattr__, __dir__ = lazy_exports(__name__, OP)
