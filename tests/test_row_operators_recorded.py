"""What follows a call besides the backward: forward mode is refused instead of losing its tangents, and a trace holds the
operator instead of its empty output."""

from __future__ import annotations

import warnings

import pytest
import torch
from torch.autograd import forward_ad

BF16 = torch.bfloat16


def operators():
    from miles_ext_kernels_b200.cake.gated_rmsnorm import rmsnorm_silu_gate
    from miles_ext_kernels_b200.cake.layer_norm import layer_norm
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence

    w, b = torch.randn(128, device="cuda").to(BF16), torch.randn(128, device="cuda").to(BF16)
    h0 = torch.randn(1, 128, device="cuda")
    cu = torch.tensor([0, 70, 200], device="cuda")
    return {
        "layer_norm": lambda x, z: layer_norm(x, w, b),
        "layer_norm without parameters": lambda x, z: layer_norm(x),
        "layer_norm with a checkpoint": lambda x, z: layer_norm(x, w, b, checkpoint="e4m3"),
        "gated_rmsnorm": lambda x, z: rmsnorm_silu_gate(x, z, w),
        "gated_rmsnorm with a checkpoint": lambda x, z: rmsnorm_silu_gate(x, z, w, checkpoint="e4m3"),
        "recurrence": lambda x, z: gated_linear_recurrence(x, -z.abs(), h0)[0],
        "recurrence with states": lambda x, z: gated_linear_recurrence(x, -z.abs(), h0, True),
        "packed recurrence": lambda x, z: gated_linear_recurrence(x, -z.abs(), None, True, cu),
    }


NAMES = ("layer_norm", "layer_norm without parameters", "layer_norm with a checkpoint", "gated_rmsnorm",
         "gated_rmsnorm with a checkpoint", "recurrence", "recurrence with states", "packed recurrence")


def inputs(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return tuple(torch.randn(1, 200, 128, device="cuda", generator=gen).to(BF16) for _ in range(2))


def tensors(out):
    return [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name):
    op, (x, z) = operators()[name], inputs(0)
    want = tensors(op(x, z))
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            op(forward_ad.make_dual(x, torch.ones_like(x)), z)
        got = tensors(op(x, z))  # nothing to follow
        assert all(torch.equal(a, b) and forward_ad.unpack_dual(a).tangent is None for a, b in zip(got, want))
    for transform in (lambda: torch.func.jvp(lambda t: op(t, z), (x,), (x,)),
                      lambda: torch.func.vmap(lambda t: op(t[None], z))(x)):
        with pytest.raises(RuntimeError):
            transform()


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_trace_holds_the_operator(name):
    op = operators()[name]
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(lambda x, z: tuple(tensors(op(x, z))), inputs(1), check_trace=False)
        for seed in (2, 3):
            x, z = inputs(seed)
            for got, want in zip(traced(x, z), tensors(op(x, z))):
                assert torch.equal(got, want)
        leaves = [t.requires_grad_() for t in inputs(4)]
        again = [t.detach().requires_grad_() for t in leaves]
        for (first, ours) in ((traced(*leaves)[0], leaves), (tensors(op(*again))[0], again)):
            first.float().square().sum().backward()
        for a, b in zip(leaves, again):
            assert (a.grad is None) == (b.grad is None) and (a.grad is None or torch.equal(a.grad, b.grad))


@pytest.mark.gpu
def test_the_step_refuses_both():
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence_step as step

    x, g, pool = (torch.randn(3, 64, device="cuda") for _ in range(3))
    slots = torch.arange(3, device="cuda")
    kept, want = pool.clone(), pool.clone()
    y = step(x, g, want, slots)
    with forward_ad.dual_level():
        for dual in ((1, 0, 0), (0, 1, 0), (0, 0, 1)):
            given = [forward_ad.make_dual(t, torch.ones_like(t)) if d else t for t, d in zip((x, g, pool), dual)]
            with pytest.raises(ValueError, match="forward-mode"):
                step(*given, slots)
        assert torch.equal(pool, kept)
        assert torch.equal(step(x, g, pool, slots), y) and torch.equal(pool, want)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with pytest.raises(ValueError, match="trace"):
            torch.jit.trace(lambda a, b: step(a, b, pool, slots), (x, g), check_trace=False)
    assert torch.equal(pool, want)
