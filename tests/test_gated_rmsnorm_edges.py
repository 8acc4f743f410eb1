"""The gated RMSNorm's operands where they start at odd addresses: refusals of the C ABI and the host's copies (CPU), the
same bits as from aligned operands (GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

EPS = 1e-6
BF16 = torch.bfloat16


def test_the_library_refuses_dense_operands_that_are_not_aligned():
    from miles_ext_kernels_b200.cake._runtime import loader

    lib, p, i64 = loader.load_library(), ctypes.c_void_p, ctypes.c_int64
    rows = [i64(2), 1, i64(128), i64(0), i64(128), i64(0), ctypes.c_float(EPS), None]

    def at(odd, *names):  # a pointer per name, two bytes off for the odd one
        return [p(64 + (2 if name == odd else 0)) for name in names]

    for odd in ("weight", "y"):
        x, z, w, y = at(odd, "x", "z", "weight", "y")
        assert lib.mek_gated_rmsnorm_fwd(x, z, w, y, *rows) == 1 and "aligned" in lib.last_error(), odd
        assert lib.mek_gated_rmsnorm_fwd_keep(x, z, w, y, p(64), p(64), p(64), p(64), *rows) == 1, odd
        assert "aligned" in lib.last_error()
    for odd in ("dy", "weight", "dx", "dz"):
        dy, w, dx, dz = at(odd, "dy", "weight", "dx", "dz")
        assert lib.mek_gated_rmsnorm_bwd(dy, p(64), p(64), w, dx, dz, None, None, *rows) == 1, odd
        assert "aligned" in lib.last_error()
        assert lib.mek_gated_rmsnorm_bwd_kept(dy, p(64), p(64), p(64), p(64), w, dx, dz, None, None, i64(2), None) == 1, odd
        assert "aligned" in lib.last_error()


def test_the_host_aligns_what_lies_at_an_odd_address():
    from miles_ext_kernels_b200.cake._impl.rows import aligned

    flat = torch.arange(600, dtype=torch.float32).bfloat16()
    for offset in (0, 1, 5, 8):
        view = flat[offset : offset + 512].view(4, 128)
        got = aligned(view)
        assert torch.equal(got, view) and got.data_ptr() % 16 == 0 and got.is_contiguous()
        assert (got.data_ptr() == view.data_ptr()) == (view.data_ptr() % 16 == 0)
    turned = aligned(flat[:512].view(128, 4).t())
    assert turned.is_contiguous() and torch.equal(turned, flat[:512].view(128, 4).t())


def make(tokens, heads, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed * 31 + tokens)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen).bfloat16()  # noqa: E731
    return randn(tokens, heads, 128), randn(tokens, heads, 128), 1 + 0.5 * randn(128), randn(tokens, heads, 128)


def run(x, z, w, dy, checkpoint):
    from miles_ext_kernels_b200.cake.gated_rmsnorm import rmsnorm_silu_gate

    leaves = [t.detach().requires_grad_() for t in (x, z, w)]
    y = rmsnorm_silu_gate(*leaves, EPS, checkpoint=checkpoint)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def moved(t, offset):
    """``t``'s values, contiguous, `offset` elements into a flat buffer."""
    flat = torch.empty(t.numel() + offset, device=t.device, dtype=t.dtype)
    view = flat[offset:].view(t.shape)
    view.copy_(t)
    return view


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("offset", [1, 4, 7])
def test_a_weight_and_a_gradient_at_odd_addresses(checkpoint, offset):
    x, z, w, dy = make(37, 3)
    want = run(x, z, w, dy, checkpoint)
    assert moved(w, offset).data_ptr() % 16 != 0 and moved(dy, offset).is_contiguous()
    for got in (run(x, z, moved(w, offset), dy, checkpoint), run(x, z, w, moved(dy, offset), checkpoint)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_the_gradient_of_a_concatenation_of_flat_outputs(checkpoint):
    """The backward of a 1-D cat hands the norm a slice of the whole gradient, here from an odd element on."""
    from miles_ext_kernels_b200.cake.gated_rmsnorm import rmsnorm_silu_gate

    x, z, w, dy = make(5, 2, seed=1)
    leaves = [t.detach().requires_grad_() for t in (x, z, w)]
    other = torch.zeros(3, device="cuda", dtype=BF16, requires_grad=True)
    whole = torch.cat([other, rmsnorm_silu_gate(*leaves, EPS, checkpoint=checkpoint).flatten()])
    got = torch.autograd.grad(whole, leaves, torch.cat([torch.zeros(3, device="cuda", dtype=BF16), dy.flatten()]))
    assert all(torch.equal(a, b) for a, b in zip(got, run(x, z, w, dy, checkpoint)[1:]))


def test_rows_that_cannot_be_read_in_place_are_copied():
    from miles_ext_kernels_b200.cake._impl.gated_rmsnorm.ops import _rows_view

    flat = torch.randn(4000).bfloat16()
    views = [flat[offset : offset + 3 * 2 * 128].view(3, 2, 128) for offset in (0, 1, 3, 4)]  # dense, at odd addresses
    views += [v.view(-1, 128) for v in views]
    views += [flat[: 2 * 1159].view(2, 1159)[:1, 8:136], flat.as_strided((1, 2, 128), (1159, 128, 1), 8),  # one token only
              flat.as_strided((2, 1, 128), (256, 1159, 1)), flat.as_strided((2, 3, 128), (1159, 128, 1), 1)]
    for view in views:
        t, heads, token_stride, head_stride = _rows_view(view, "x")
        assert heads == (1 if view.dim() == 2 else view.shape[1])
        assert t.data_ptr() % 16 == 0 and token_stride % 8 == 0 and head_stride % 8 == 0
        rows = t.as_strided((view.shape[0], heads, 128), (token_stride, head_stride, 1))
        assert torch.equal(rows.reshape(view.shape), view)


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_x_and_z_at_odd_addresses(checkpoint):
    x, z, w, dy = make(37, 3, seed=2)
    want = run(x, z, w, dy, checkpoint)
    for got in (run(moved(x, 1), z, w, dy, checkpoint), run(x, moved(z, 3), w, dy, checkpoint)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = torch.randn(2, 1159, device="cuda").bfloat16()[:1, 8:136]  # one row of a projection of odd width
    got = run(one, one, w, dy[:1, 0], checkpoint)
    assert all(torch.equal(a, b) for a, b in zip(got, run(one.clone(), one.clone(), w, dy[:1, 0], checkpoint)))


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_a_second_derivative_is_refused(checkpoint):
    from miles_ext_kernels_b200.cake.gated_rmsnorm import rmsnorm_silu_gate

    x, z, w, dy = make(6, 2, seed=3)
    leaves = [t.requires_grad_() for t in (x, z, w)]
    y = rmsnorm_silu_gate(*leaves, EPS, checkpoint=checkpoint)
    grads = torch.autograd.grad(y, leaves, dy.requires_grad_(), create_graph=True)
    first = [g.detach() for g in grads]
    assert all(torch.equal(a, b) for a, b in zip(first, run(x, z, w, dy.detach(), checkpoint)[1:]))
    # other paths of the sum have a second derivative; this one's must not be left out of it without a word
    penalty = sum(g.float().square().sum() for g in grads) + x.float().pow(3).sum()
    with pytest.raises(RuntimeError, match="once_differentiable"):
        penalty.backward()
