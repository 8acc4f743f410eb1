"""The ops of a recurrent layer as one run: LayerNorm, projections, the short convolution, the gated linear recurrence,
the gated output norm -- forward and backward, with and without 8-bit checkpoints, against the same layer in plain
64-bit torch that rounds where the ops round; then token by token with the step (GPU)."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

BF16 = torch.bfloat16
pytestmark = pytest.mark.gpu


class Rounded(torch.autograd.Function):
    """A value on its way through BF16; its gradient goes the same way."""

    @staticmethod
    def forward(ctx, t):
        return t.to(BF16).double()

    @staticmethod
    def backward(ctx, d):
        return d.to(BF16).double()


def e4m3(t, power=None):
    power = 1.0 if power is None else power
    return (t / power).float().to(torch.float8_e4m3fn).double() * power


class PlainNorm(torch.autograd.Function):
    """LayerNorm whose backward takes the normalised rows as the checkpoint holds them."""

    @staticmethod
    def forward(ctx, x, w, b, keep):
        rstd = 1 / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + 1e-5)
        unit = (x - x.mean(-1, keepdim=True)) * rstd
        ctx.save_for_backward(e4m3(unit) if keep else unit, rstd, w)
        return unit * w + b

    @staticmethod
    def backward(ctx, dy):
        unit, rstd, w = ctx.saved_tensors
        dn = dy * w
        dx = rstd * (dn - dn.mean(-1, keepdim=True) - unit * (dn * unit).mean(-1, keepdim=True))
        return dx, (dy * unit).flatten(0, -2).sum(0), dy.flatten(0, -2).sum(0), None


class PlainGatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, w, keep):
        rstd = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        n = x * rstd
        y = n * w * F.silu(z)
        if keep:
            mantissa, exponent = torch.frexp(z.abs().amax(-1, keepdim=True))
            n, z = e4m3(n), e4m3(z, torch.ldexp(torch.ones_like(mantissa), exponent - 9 + (mantissa > 0.875)))
        ctx.save_for_backward(n, z, w, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        n, z, w, rstd = ctx.saved_tensors
        s = torch.sigmoid(z)
        dn = dy * z * s * w
        dx = rstd * (dn - n * (dn * n).mean(-1, keepdim=True))
        return dx, dy * n * w * s * (1 + z * (1 - s)), (dy * z * s * n).flatten(0, -2).sum(0), None


def plain_layer(p, x, h0, lengths, keep):
    p = {k: v.double() for k, v in p.items()}
    r = Rounded.apply
    x = x.double()
    normed = r(PlainNorm.apply(x, p["ln_w"], p["ln_b"], keep))
    inner, gate, z = (r(normed @ p[k]) for k in ("w_in", "w_gate", "w_z"))
    g = -F.softplus(gate) * p["rate"]
    outs, states, start = [], [], 0
    for i, n in enumerate(lengths):
        part = inner[0, start : start + n]
        padded = torch.cat([part.new_zeros(3, part.shape[1]), part])
        conv = r(F.silu(sum(p["taps"][:, k] * padded[k : k + n] for k in range(4))))
        h = h0[i].double()
        for t in range(n):
            h = g[0, start + t].exp() * h + conv[t]
            outs.append(h)
        states.append(h)
        start += n
    y = r(torch.stack(outs))[None]
    heads = y.unflatten(-1, (-1, 128))
    gated = r(PlainGatedNorm.apply(heads, z.unflatten(-1, (-1, 128)), p["norm_w"], keep))
    return x + r(gated.flatten(-2) @ p["w_out"]), torch.stack(states)


def layer(p, x, h0, cu, checkpoint):
    from miles_ext_kernels_b200.cake.conv1d import causal_conv1d
    from miles_ext_kernels_b200.cake.gated_rmsnorm import rmsnorm_silu_gate
    from miles_ext_kernels_b200.cake.layer_norm import layer_norm
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence

    normed = layer_norm(x, p["ln_w"], p["ln_b"], checkpoint=checkpoint)
    inner, gate, z = (normed @ p[k] for k in ("w_in", "w_gate", "w_z"))
    g = -F.softplus(gate.float()) * p["rate"]
    conv = causal_conv1d(inner, p["taps"], cu)
    y, final = gated_linear_recurrence(conv, g, h0, output_final_state=True, cu_seqlens=cu)
    heads = y.unflatten(-1, (-1, 128))
    gated = rmsnorm_silu_gate(heads, z.unflatten(-1, (-1, 128)), p["norm_w"], checkpoint=checkpoint)
    return x + gated.flatten(-2) @ p["w_out"], final


def make(lengths, width=256, inner=384, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    p = {
        "ln_w": (1 + 0.1 * randn(width)).to(BF16), "ln_b": (0.1 * randn(width)).to(BF16),
        "w_in": (randn(width, inner) / width**0.5).to(BF16), "w_gate": (randn(width, inner) / width**0.5).to(BF16),
        "w_z": (randn(width, inner) / width**0.5).to(BF16), "w_out": (randn(inner, width) / inner**0.5).to(BF16),
        "taps": 0.5 * randn(inner, 4), "norm_w": (1 + 0.1 * randn(128)).to(BF16),
        "rate": torch.exp(-4 * torch.rand(inner, device="cuda", generator=gen)),
    }
    total = sum(lengths)
    x = randn(1, total, width).to(BF16)
    return p, x, randn(len(lengths), inner), randn(1, total, width).to(BF16)


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_a_layer_s_training_step(checkpoint):
    lengths = [130, 1, 77, 200]
    p, x, h0, dy = make(lengths)
    cu = torch.tensor([0, *lengths], device="cuda").cumsum(0).int()
    outcome = []
    for run in (lambda q, a, h: layer(q, a, h, cu, checkpoint), lambda q, a, h: plain_layer(q, a, h, lengths, checkpoint is not None)):
        q = {k: v.clone().requires_grad_() for k, v in p.items()}
        a, h = x.clone().requires_grad_(), h0.clone().requires_grad_()
        y, final = run(q, a, h)
        grads = torch.autograd.grad((y, final), [a, h, *q.values()], (dy.to(y.dtype), torch.ones_like(final)))
        outcome.append({"y": y, "final": final, **dict(zip(["dx", "dh0", *("d" + k for k in q)], grads))})
    got, want = outcome
    for name in want:
        w, g = want[name].double(), got[name].double()
        # a value passes at most 16 roundings to BF16 (eight operations, forward and backward), each off by at most 2^-9
        # of it on root mean square (half a step is 2^-8 at most, 2^-9.4 on average); independent ones add as squares
        assert (g - w).norm() <= 16**0.5 * 2.0**-9 * 2 * w.norm(), (name, float((g - w).norm() / w.norm()))


def test_prefill_and_steps_continue_one_another():
    from miles_ext_kernels_b200.cake.layer_norm import layer_norm
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence, gated_linear_recurrence_step

    p, x, _, _ = make([40, 40, 40], seed=1)
    rows = x.view(3, 40, -1)
    with torch.no_grad():
        normed = layer_norm(rows, p["ln_w"], p["ln_b"])
        one_by_one = torch.stack([layer_norm(rows[:, t], p["ln_w"], p["ln_b"]) for t in range(40)], 1)
        assert torch.equal(normed, one_by_one)  # a row does not depend on its batch
        inner, gate = normed @ p["w_in"], normed @ p["w_gate"]
        g = -F.softplus(gate.float()) * p["rate"]
        whole, last = gated_linear_recurrence(inner, g, output_final_state=True)
        _, state = gated_linear_recurrence(inner[:, :25], g[:, :25], output_final_state=True)
        pool = torch.zeros(8, state.shape[1], device="cuda")
        slots = torch.tensor([6, 1, 4], device="cuda")
        pool[slots] = state
        for t in range(25, 40):
            y = gated_linear_recurrence_step(inner[:, t], g[:, t], pool, slots)
            # both round the same FP32 state up to its last bits
            assert (y.float() - whole[:, t].float()).abs().max() <= 2.0**-8 * whole[:, t].float().abs().max()
        assert torch.allclose(pool[slots], last, rtol=1e-5, atol=1e-5)
