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


def top_and_bottom():
    """Gates whose decays reach both ends of FP32: up to the largest finite one, down past the smallest normal one."""
    top = torch.linspace(88.0, 88.7228, 500)  # e^88.7228 = 3.4028e38
    return torch.cat([top, -top, torch.linspace(-86.97, 88.0, 700), torch.tensor([-87.0, -200.0, -float("inf"), 89.0, 1e30])])


@pytest.mark.gpu
def test_decays_at_both_ends_of_fp32():
    """One token from the state 1 (and, backwards, from the gradient 1): the decay itself.  It may be off by the rounding of
    log 2, |n| 2e-9 for a gate of n log 2, and three half steps; below e^-86.98 it may be zero."""
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence, gated_linear_recurrence_step as step

    g = top_and_bottom().cuda()
    want = g.double().exp()
    h0, x = torch.ones(1, g.numel(), device="cuda"), torch.zeros(1, 1, g.numel(), device="cuda")
    leaves = [t.requires_grad_() for t in (x, g[None, None].clone(), h0)]
    y, _ = gated_linear_recurrence(*leaves)
    _, dg, dh0 = torch.autograd.grad(y, leaves, torch.ones_like(y))
    with torch.no_grad():
        pool = torch.ones(1, g.numel(), device="cuda")
        stepped = step(x[0], g[None], pool)
    # (clamped, or the gate of minus infinity would make 0 * infinity of its bound, which is 0)
    bound = want * (3 * 2.0**-24 + g.double().abs().clamp(max=200) / 0.693 * 2e-9) + torch.where(g < -86.98, 1.67e-38, 0.0).double()
    for got in (y, dg, dh0, stepped, pool):
        got = got.detach().flatten().double()
        over = want > torch.finfo(FP32).max
        assert torch.equal(got[over].isinf(), torch.ones_like(got[over]).bool()) and int(over.sum()) == 2
        assert ((got - want).abs() <= bound)[~over].all()
        assert (got[g <= -87.0] == 0).all()


def growth(kind, tokens, channels):
    """Gates that grow past FP32's range inside a tile, and where there is something to grow."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.zeros(1, tokens, channels, device="cuda")
    dy = torch.zeros(1, tokens, channels, device="cuda")
    g = torch.full((1, tokens, channels), 8.0 if kind == "in a warp" else 1.0, device="cuda")
    randn = lambda n: torch.randn(n, channels, device="cuda", generator=gen)  # noqa: E731
    if kind == "closed after it":  # what grew is gone behind a gate of minus infinity
        g[:, 150] = -float("inf")
        g[:, 151:] = -0.1
        x[:, 150:], dy[:, 170:] = randn(tokens - 150), randn(tokens - 170)
    elif kind == "closed before it":
        g[:, :40] = -0.1
        g[:, 40] = -float("inf")
        x[:, :20], dy[:, :30] = randn(20), randn(30)
        g[:, 41:] = 2.0
    else:
        reach = 8 if kind == "in a warp" else 60
        x[:, -reach:], dy[:, :reach] = randn(reach), randn(reach)
    return x, g, dy


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [64, 33, 640, 12800])
@pytest.mark.parametrize("kind", ["in a tile", "in a warp", "closed after it", "closed before it"])
def test_growth_of_nothing_is_nothing(kind, channels):
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence
    from oracle import rows_oracle as R

    tokens = 900
    x, g, dy = growth(kind, tokens, channels)
    leaves = [t.clone().requires_grad_() for t in (x, g)]
    y, final = gated_linear_recurrence(*leaves, output_final_state=True)
    dl = torch.zeros_like(final)
    if kind == "closed after it":
        dl.normal_()
    dx, dg = torch.autograd.grad((y, final), leaves, (dy, dl))
    some = slice(0, 70)  # the channels are alike
    want = R.linear_recurrence(x[0, :, some], g[0, :, some], [tokens], None, dy[0, :, some], dl[:, some])
    for name, got in (("y", y[0]), ("final", final), ("dx", dx[0]), ("dg", dg[0])):
        got = got.detach()
        assert torch.isfinite(got).all(), name
        assert R.misses(got[:, some], *want[name]) == 0, name


PACKED = [
    ([1], 0), ([0, 5], 0), ([1] * 70, 0), ([3] * 200, 5), ([0, 0, 3, 0, 0, 130, 0, 1, 16, 0], 0), ([16, 16, 32, 64], 7),
    ([300, 2, 255], 40), ([0] * 45 + [20] + [0] * 45, 0), ([7, 0, 5, 1, 2, 0, 0, 1, 200, 9, 300, 1, 1], 130), ([513], 600),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,tail", PACKED)
@pytest.mark.parametrize("channels,dtype,gdtype", [(128, BF16, FP32), (128, BF16, BF16), (72, torch.float16, torch.float16),
                                                   (64, FP32, BF16), (64, FP32, FP32)])
def test_packed_sequences_that_come_by_boxes(lengths, tail, channels, dtype, gdtype):
    """Channels that TMA can address: several boundaries in a warp, empty sequences, tokens behind the last one, and gates
    of 16 bits, whose gradients take the place of decays."""
    import test_linear_recurrence as base

    total = sum(lengths) + tail
    x, g, h0, dy, dl = base.make(1, total, channels, dtype, gdtype, len(lengths), seed=21)
    if tail:
        x[:, total - tail :], dy[:, total - tail :] = float("nan"), float("inf")
    cu = torch.tensor([0] + lengths, device="cuda").cumsum(0).int()
    base.check(base.run(x, g, h0, dy, dl, cu), x, g, h0, dy, dl, lengths, str(lengths)[:40], tail)
    base.check(base.run(x, g, None, dy, None, cu, final=False), x, g, None, dy, None, lengths, "no states", tail)


@pytest.mark.gpu
@pytest.mark.parametrize("gdtype", [FP32, BF16])
@pytest.mark.parametrize("kind", ["mixed", "open"])
@pytest.mark.parametrize("chains", [1, 16, 20, 30, 50, 100, 400])
def test_every_depth_of_the_look_back(chains, kind, gdtype):
    """How far a block looks back follows from the number of chains (channel blocks x batch rows): 48 tiles, 5 x 8, ... 8, four by
    one warp.  With open gates a state carried wrongly would show; a chain has the bits that it has alone."""
    import test_linear_recurrence as base

    tokens, batch = 128 * 14 + 37, 2 if chains % 20 == 0 else 1
    channels = 64 * chains // batch
    x, g, h0, dy, dl = base.make(batch, tokens, channels, BF16, gdtype, batch, kind, seed=22)
    got = base.run(x, g, h0, dy, dl)
    for row, block in {(0, 0), (batch - 1, channels // 64 - 1)}:
        some, one = slice(64 * block, 64 * block + 64), slice(row, row + 1)
        part = [t[one][..., some].contiguous() for t in (x, g, h0, dy, dl)]
        mine = {n: t[one][..., some].contiguous() for n, t in got.items()}
        base.check(mine, *part, [tokens], f"{chains} chains")
        alone = base.run(*part)
        assert all(torch.equal(mine[n], alone[n]) for n in alone)


@pytest.mark.gpu
def test_a_gradient_at_an_odd_address():
    import test_linear_recurrence as base

    x, g, h0, dy, dl = base.make(2, 200, 64, BF16, BF16, 2, seed=23)
    want = base.run(x, g, h0, dy, dl)
    for offset in (1, 4):
        flat = torch.empty(dy.numel() + offset, device="cuda", dtype=BF16)
        states = torch.empty(dl.numel() + 1, device="cuda")
        moved, moved_states = flat[offset:].view(dy.shape).copy_(dy), states[1:].view(dl.shape).copy_(dl)
        got = base.run(x, g, h0, moved, moved_states)
        assert moved.is_contiguous() and all(torch.equal(got[n], want[n]) for n in want)
