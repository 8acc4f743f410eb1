"""The gated RMSNorm's 8-bit checkpoint: refusals (CPU); the codes, and the gradients computed from them, against 64 bits,
with gates of every size, rows of zeros, gates that are not finite, the gate in place or copied, captured graphs (GPU)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import rows_oracle as R

EPS = 1e-6


FLUSH = 2.0**-126  # a sigmoid below it may come out as zero


def sigmoid_error(z, s):
    """What a term with one sigmoid may be off by, relative.  CUDA's programming guide bounds __expf(z) by
    2 + floor(1.173 |z|) ulp and __fdividef by 2 ulp (an ulp is at most 2^-23 of the value); s = 1 / (1 + e) passes on
    (1 - s) of e's relative error; the sum, and up to twelve FP32 products and sums of a term, add half an ulp each.
    The guide has __fdividef(x, y) give zero for 2^126 < y < 2^128, and 1 / infinity is zero: FLUSH is added for that."""
    return ((2 + 1.173 * z.abs()) * (1 - s) + 2 + 13 / 2) * 2.0**-23


def test_the_checkpoint_argument_and_the_library_s_checks():
    import ctypes

    from miles_ext_kernels_b200.cake._runtime import loader
    from miles_ext_kernels_b200.cake.gated_rmsnorm import rmsnorm_silu_gate

    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="checkpoint must be one of"):
        rmsnorm_silu_gate(x, x, x[0], checkpoint="fp8")
    with pytest.raises(ValueError, match="CUDA tensors"):
        rmsnorm_silu_gate(x, x, x[0], checkpoint="e4m3")
    lib, p, i64 = loader.load_library(), ctypes.c_void_p, ctypes.c_int64
    kept = [p(64), p(64), p(64), p(64)]
    tail = [i64(1), 1, i64(128), i64(0), i64(128), i64(0), ctypes.c_float(EPS), None]
    for k in range(4):
        some = [None if i == k else a for i, a in enumerate(kept)]
        assert lib.mek_gated_rmsnorm_fwd_keep(p(64), p(64), p(64), p(64), *some, *tail) == 1 and "null" in lib.last_error()
        assert lib.mek_gated_rmsnorm_bwd_kept(p(64), *some, p(64), p(64), p(64), None, None, i64(1), None) == 1
    assert lib.mek_gated_rmsnorm_fwd_keep(p(64), p(64), p(64), p(64), p(68), *kept[1:], *tail) == 1
    assert "aligned" in lib.last_error()
    assert lib.mek_gated_rmsnorm_bwd_kept(p(64), *kept, p(64), p(64), p(64), None, None, i64(0), None) == 1
    assert lib.mek_gated_rmsnorm_bwd_kept(p(64), *kept, p(64), p(64), p(64), p(64), None, i64(1), None) == 1


def make(tokens, heads, seed=0, gate=1.0, pad=8):
    gen = torch.Generator(device="cuda").manual_seed(seed * 997 + tokens * 7 + heads)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    x = (randn(tokens, heads, 128) * (0.1 + randn(tokens, heads, 1).abs())).bfloat16()
    projection = (randn(tokens, 2 * heads * 128 + pad) * gate).bfloat16()
    z = projection[:, heads * 128 : 2 * heads * 128].unflatten(-1, (heads, 128))
    return x, z, (1 + 0.5 * randn(128)).bfloat16(), randn(tokens, heads, 128).bfloat16()


def run(x, z, w, dy, checkpoint="e4m3"):
    from miles_ext_kernels_b200.cake.gated_rmsnorm import rmsnorm_silu_gate

    leaves = [t.detach().requires_grad_() for t in (x, z, w)]
    y = rmsnorm_silu_gate(*leaves, EPS, checkpoint=checkpoint)
    kept = y.grad_fn.saved_tensors
    y.backward(dy)
    return {"y": y.detach(), "dx": leaves[0].grad, "dz": leaves[1].grad, "dw": leaves[2].grad}, kept


def check(got, kept, x, z, w, dy):
    codes_n, codes_z, exponent, rstd = (t.double() if t.dtype == torch.float32 else t for t in kept[:4])
    x, z, w, dy = (t.double().reshape(-1, 128) if t.dim() > 1 else t.double() for t in (x, z, w, dy))
    true_rstd = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
    assert ((rstd[:, None] / true_rstd - 1).abs() <= 32 * R.U32).all()
    n = x * true_rstd
    assert R.e4m3_misses(codes_n, n, 32 * R.U32 * n.abs()) == 0
    finite = torch.isfinite(z)
    most = torch.where(finite, z, 0.0).abs().amax(-1)
    power = 2.0 ** (exponent.double() - 127)
    assert (most <= 448 * power).all() and ((most > 224 * power) | (exponent == 1)).all()  # the smallest that fits
    scaled = torch.where(finite, z / power[:, None], 0.0)
    value = codes_z.view(torch.float8_e4m3fn).double()
    assert torch.equal(value.isnan(), ~finite)
    # z / 2^e is exact: each code is the nearest, ties to even, as torch rounds it
    assert torch.equal(torch.where(finite, value, 0.0), scaled.float().to(torch.float8_e4m3fn).double())
    # the gradients of these codes
    n, z, rstd = codes_n.view(torch.float8_e4m3fn).double(), value * power[:, None], rstd[:, None]
    s = torch.sigmoid(z)
    a = dy * z * s
    dn = a * w
    dot = (dn * n).mean(-1, keepdim=True)
    dx = rstd * (dn - n * dot)
    term = sigmoid_error(z, s)
    # (the mean of 128 terms: eight in a lane and four shuffles, half an ulp each)
    dx_slack = rstd * (dn.abs() * term + n.abs() * ((dn * n).abs() * (term + 14 * R.U32)).mean(-1, keepdim=True))
    dx_slack = dx_slack + rstd * (dy * z * w).abs() * FLUSH
    dz = dy * n * w * s * (1 + z * (1 - s))
    # 1 - s is off by s's own error s term, and by half an ulp of one
    dz_slack = (dy * n * w * s).abs() * ((1 + z.abs() * (1 - s)) * term + z.abs() * (s * term + R.U32))
    dz_slack = dz_slack + (dy * n * w).abs() * (1 + z.abs()) * FLUSH
    dw = (a * n).sum(0)
    rows = dy.shape[0]
    for name, want, slack in (("dx", dx, dx_slack), ("dz", dz, dz_slack), ("dw", dw, ((a * n).abs() * (term + 512 * R.U32)).sum(0))):
        if name == "dw" and not torch.isfinite(want).all():
            continue
        have = got[name].reshape(want.shape)
        assert R.misses(have, want, slack) == 0, name
        if rows > 2 and torch.isfinite(want).all():
            assert R.misses((have.double() * 1.02).to(have.dtype), want, slack) > 0, f"{name}: the gate is too loose"


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [8, 3])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 12), (7, 16), (33, 5), (1031, 12), (4099, 4)])
@pytest.mark.parametrize("gate", [1.0, 30.0, 1e-30])
def test_codes_and_gradients_against_64_bits(tokens, heads, gate, pad):
    x, z, w, dy = make(tokens, heads, gate=gate, pad=pad)
    got, kept = run(x, z, w, dy)
    check(got, kept, x, z, w, dy)
    plain, _ = run(x, z, w, dy, checkpoint=None)
    assert torch.equal(got["y"], plain["y"])  # what is kept does not change the output
    again, _ = run(x, z, w, dy)
    assert all(torch.equal(got[n], again[n]) for n in got)
    flat, _ = run(x.reshape(-1, 128), z.reshape(-1, 128), w, dy.reshape(-1, 128))
    assert all(torch.equal(flat[n].view(got[n].shape), got[n]) for n in got)


@pytest.mark.gpu
def test_rows_of_zeros_powers_of_two_and_values_that_are_not_finite():
    x, z, w, dy = make(40, 2, seed=1)
    x, z = x.clone(), z.clone()
    x[3], z[5] = 0, 0
    z[7, 0] = torch.linspace(-448, 448, 128, device="cuda").bfloat16()  # the format's own range, and just outside
    z[8, 0], z[9, 0] = z[7, 0] * 1.0078125, z[7, 0] * 2.0**-100
    z[10, 0, :3] = torch.tensor([2.0**-133, 0.0, -(2.0**-133)])  # among BF16's subnormals
    z[10, 0, 3:] = 0
    got, kept = run(x, z, w, dy)
    check(got, kept, x, z, w, dy)
    clean = got
    z[12, 1, 5], z[13, 1, 6], x[14, 0, 7] = math.inf, math.nan, math.nan
    got, kept = run(x, z, w, dy)
    values = kept[1].view(torch.float8_e4m3fn).float().view(40, 2, 128)
    assert values[12, 1, 5].isnan() and values[13, 1, 6].isnan() and int(values.isnan().sum()) == 2
    rows = [r for r in range(40) if r not in (12, 13, 14)]
    for n in ("y", "dx", "dz"):
        assert torch.equal(got[n][rows], clean[n][rows]), n
    assert int(got["dz"][12, 1].isnan().sum()) == 1  # the other gates of the row keep their gradients


@pytest.mark.gpu
def test_memory_empty_calls_and_captured_graphs():
    from miles_ext_kernels_b200.cake.gated_rmsnorm import rmsnorm_silu_gate

    x, z, w, dy = make(2048, 16, seed=2)
    n = x.numel()
    leaf = w.clone().requires_grad_()
    held = []
    for checkpoint in (None, "e4m3"):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        inputs = [x * 2, z * 2]
        y = rmsnorm_silu_gate(*inputs, leaf, EPS, checkpoint=checkpoint)
        del inputs
        held.append(torch.cuda.memory_allocated() - before)
        del y
    assert held[0] >= 6 * n and held[1] <= 4 * n + 5 * n // 128 + 65536
    got, _ = run(x[:0], z[:0], w, dy[:0])
    assert got["y"].shape == (0, 16, 128) and got["dw"].abs().sum() == 0
    want, _ = run(x, z, w, dy)
    leaves = [t.clone().requires_grad_() for t in (x, z, w)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rmsnorm_silu_gate(*leaves, EPS, checkpoint="e4m3")
        dx, dz, dw = torch.autograd.grad(y, leaves, dy)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for name, t in (("y", y), ("dx", dx), ("dz", dz), ("dw", dw)):
        assert torch.equal(t.detach(), want[name]), name
