"""Dense operands that start off a 16-byte boundary -- views into flat buffers, gradients handed over as slices -- of the
short convolution, the gated delta rule and KDA: copied by the host (CPU), the same bits as from aligned ones (GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

BF16 = torch.bfloat16


def moved(t, offset=1):
    """``t``'s values, dense, ``offset`` elements into a flat buffer."""
    return torch.empty(t.numel() + offset, device=t.device, dtype=t.dtype)[offset:].view(t.shape).copy_(t)


def test_the_host_copies_them():
    from miles_ext_kernels_b200.cake._impl.gdn import ops

    x = torch.randn(2, 5, 3, 128).bfloat16()
    for offset in (0, 1, 4, 8):
        for packed in (ops._packed, ops._rows):
            got = packed(moved(x, offset))
            assert got.data_ptr() % 16 == 0 and torch.equal(got, x.view(10, 3, 128))
    assert ops._rows(x).data_ptr() == x.data_ptr()


def test_the_library_refuses_rows_of_the_convolution_that_are_not_aligned():
    from miles_ext_kernels_b200.cake._runtime import loader

    lib, p = loader.load_library(), ctypes.c_void_p
    for odd in range(3):
        x, prev, y = (p(64 + (2 if k == odd else 0)) for k in range(3))
        assert lib.mek_conv1d_fwd(x, prev, p(64), 1, p(64), y, 4, 8, None) == 1 and "aligned" in lib.last_error()
    for odd in range(6):
        x, prev, after, dy, dy_after, dx = (p(64 + (8 if k == odd else 0)) for k in range(6))
        assert lib.mek_conv1d_bwd(x, prev, after, p(64), 1, dy, dy_after, p(64), dx, None, None, 0, 4, 8, None) == 1
        assert "aligned" in lib.last_error()


def gradients(op, inputs, outputs):
    leaves = [t.detach().requires_grad_(t.is_floating_point()) for t in inputs]
    out = op(*leaves)
    out = out if isinstance(out, tuple) else (out,)
    grads = torch.autograd.grad(out, [t for t in leaves if t.requires_grad], outputs)
    return [t.detach() for t in out] + list(grads)


def compare(op, inputs, outputs):
    want = gradients(op, inputs, outputs)
    for offset in (1, 3):
        for k in range(len(inputs)):
            got = gradients(op, [moved(t, offset) if j == k else t for j, t in enumerate(inputs)], outputs)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (k, offset)
        for k in range(len(outputs)):
            got = gradients(op, inputs, [moved(t, offset) if j == k else t for j, t in enumerate(outputs)])
            assert all(torch.equal(a, b) for a, b in zip(got, want)), ("gradient", k, offset)


def randn(*shape, seed=0, dtype=BF16):
    gen = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(*shape, device="cuda", generator=gen).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("policy", ["bf16", "fp32"])
def test_the_convolution(policy):
    from miles_ext_kernels_b200.cake.conv1d import causal_conv1d

    cu = torch.tensor([0, 40, 41, 130], device="cuda")
    compare(lambda x, w: causal_conv1d(x, w, cu, silu_grad_preactivation=policy), [randn(1, 130, 72), randn(72, 4)],
            [randn(1, 130, 72, seed=1)])


@pytest.mark.gpu
@pytest.mark.parametrize("l2norm", [True, False])
def test_the_gated_delta_rule(l2norm):
    from miles_ext_kernels_b200.cake import gdn

    tokens, heads, value_heads = 150, 2, 4
    unit = lambda t: torch.nn.functional.normalize(t.float(), dim=-1).to(BF16)  # noqa: E731
    inputs = [unit(randn(1, tokens, heads, 128)), unit(randn(1, tokens, heads, 128, seed=1)),
              randn(1, tokens, value_heads, 128, seed=2), -0.3 * randn(1, tokens, value_heads, dtype=torch.float32).abs(),
              randn(1, tokens, value_heads, seed=3).sigmoid(), randn(2, value_heads, 128, 128, dtype=torch.float32)]
    cu = torch.tensor([0, 70, tokens], device="cuda", dtype=torch.int32)
    compare(lambda q, k, v, g, beta, h0: gdn.chunk_gated_delta_rule(
        q, k, v, g=g, beta=beta, initial_state=h0, output_final_state=True, use_qk_l2norm_in_kernel=l2norm, cu_seqlens=cu),
        inputs, [randn(1, tokens, value_heads, 128, seed=4), randn(2, value_heads, 128, 128, seed=5, dtype=torch.float32)])


@pytest.mark.gpu
def test_kda():
    from miles_ext_kernels_b200.cake import kda

    tokens, heads = 150, 2
    unit = lambda t: torch.nn.functional.normalize(t.float(), dim=-1).to(BF16)  # noqa: E731
    inputs = [unit(randn(tokens, heads, 128)), unit(randn(tokens, heads, 128, seed=1)), randn(tokens, heads, 128, seed=2),
              -0.3 * randn(tokens, heads, 128, seed=3, dtype=torch.float32).abs(), randn(tokens, heads, seed=4).sigmoid()]
    cu = torch.tensor([0, 70, tokens], device="cuda", dtype=torch.int32)
    compare(lambda q, k, v, g, beta: kda.chunk_kda(q, k, v, g, beta, cu), inputs, [randn(tokens, heads, 128, seed=5)])
