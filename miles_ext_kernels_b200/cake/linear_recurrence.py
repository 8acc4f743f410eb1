"""The gated linear recurrence ``h[t] = exp(g[t]) h[t-1] + x[t]`` per channel, over long or packed sequences, forward and
backward, and its single-token step on a pool of states, on hand-written sm_100a kernels.

An op of this package, without a counterpart in the reference and without a miles argument that selects it: the
element-wise sibling of the gated delta rule (``cake.gdn``), with the same conventions -- ``g`` is a log decay in nats,
sequences are packed by ``cu_seqlens``, states are FP32.  Both variants (``det``, ``fast``) run the same kernels: states
are folded in token order whatever the timing, so identical inputs give identical bits.

Importing this module imports neither torch nor the implementation.
"""

from ._runtime.spec import OpSpec, lazy_exports

OP = OpSpec(
    name="linear_recurrence",
    summary="gated linear recurrence per channel, forward + backward + single-token step",
    variants=("det", "fast"),
    packages=("libmek_b200",),
    exports=("check_supported", "gated_linear_recurrence", "gated_linear_recurrence_step"),
)

__all__, __getattr__, __dir__ = lazy_exports(__name__, OP)
