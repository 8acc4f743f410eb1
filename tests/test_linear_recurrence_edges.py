"""The gated linear recurrence where autograd, tracing and its own borders meet it (GPU)."""

from __future__ import annotations

import pytest
import torch

BF16, FP32 = torch.bfloat16, torch.float32


def make(batch, tokens, channels, seed=0, dtype=BF16):
    gen = torch.Generator(device="cuda").manual_seed(seed * 131 + tokens)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    return randn(batch, tokens, channels).to(dtype), -0.1 * randn(batch, tokens, channels).abs()


@pytest.mark.gpu
def test_a_pool_that_a_graph_has_saved_and_that_is_then_stepped():
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence, gated_linear_recurrence_step as step

    x, g = make(4, 40, 64)
    pool = torch.randn(4, 64, device="cuda")
    g.requires_grad_()
    y, _ = gated_linear_recurrence(x, g, pool)
    y.float().sum().backward(retain_graph=True)  # the pool is as it was
    version = pool._version
    with torch.no_grad():
        step(x[:, 0], g[:, 0], pool)
        assert pool._version == version + 1
        step(x[:, 0], g[:, 0], pool[:3][:, :], torch.tensor([2, -1, 0, 1], device="cuda"))  # a view of it
        assert pool._version == version + 2
        step(x[:0, 0], g[:0, 0], pool)
        assert pool._version == version + 2  # nothing was changed
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()
    with torch.inference_mode():
        pool = torch.zeros(4, 64, device="cuda")  # has no version
        assert torch.equal(step(x[:, 0], g[:, 0], pool), x[:, 0])
