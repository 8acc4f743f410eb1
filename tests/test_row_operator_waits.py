"""Waits of the row operators that run out: the kernels are not sent what they wait for, give up after a short limit and
return; what was computed from it is NaN, the rest is as it was, and the next call is right.  Nothing faults: no copy is in
flight and no lane stays behind."""

from __future__ import annotations

import ctypes
from contextlib import contextmanager

import pytest
import torch

BF16, FP32 = torch.bfloat16, torch.float32
TILE, WARP = 128, 16
WORDS = 1 << 8


def _set(limit_ns, rows_served, tiles_withheld):
    from miles_ext_kernels_b200.cake._runtime import loader

    lib = loader.load_library()
    lib.check(lib.mek_selftest_row_waits(ctypes.c_int64(limit_ns), ctypes.c_int64(rows_served),
                                         ctypes.c_uint32(tiles_withheld)))


@contextmanager
def withheld(rows_served=-1, tiles=0, limit_ns=2_000_000):
    try:
        _set(limit_ns, rows_served, tiles)
        yield
        torch.cuda.synchronize()
    finally:
        _set(-1, -1, 0)


def test_the_limit_is_at_most_a_second():
    with pytest.raises(ValueError, match="one second"):
        _set(1_000_000_001, -1, 0)
    _set(-1, -1, 0)


def sequence(tokens, channels, seed=0, dtype=BF16):
    gen = torch.Generator(device="cuda").manual_seed(seed + tokens)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    x, dy = randn(1, tokens, channels).to(dtype), randn(1, tokens, channels).to(dtype)
    return x, -0.02 * randn(1, tokens, channels).abs(), dy


def recurrence(x, g, h0, dy, dl, cu=None, forward=None, backward=None):
    """One step with what each direction is not sent."""
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence

    leaves = [t.detach().requires_grad_() for t in (x, g, h0)]
    with withheld(**(forward or {})):
        y, final = gated_linear_recurrence(*leaves, output_final_state=True, cu_seqlens=cu)
    with withheld(**(backward or {})):
        dx, dg, dh0 = torch.autograd.grad((y, final), leaves, (dy, dl))
    return {"y": y.detach(), "final": final.detach(), "dx": dx, "dg": dg, "dh0": dh0}


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [64, 640, 12800, 66])  # eight warps look back, some of them far, or one warp; plain loads
def test_words_that_do_not_come(channels):
    """The state cannot leave a tile: the tiles behind it are NaN, up to the next sequence's start."""
    tokens = 5 * TILE + 40
    x, g, dy = sequence(tokens, channels)
    cuts = torch.tensor([0, 3 * TILE + 20, tokens], device="cuda", dtype=torch.int32)
    h0, dl = torch.randn(2, channels, device="cuda"), torch.randn(2, channels, device="cuda")
    want = recurrence(x, g, h0, dy, dl, cuts)
    got = recurrence(x, g, h0, dy, dl, cuts, forward=dict(tiles=WORDS))
    second = 3 * TILE + 20  # the second sequence starts in tile 3
    right = [*range(0, TILE), *range(second, 4 * TILE)]
    lost = [*range(TILE, second), *range(4 * TILE, tokens)]
    assert torch.equal(got["y"][:, right], want["y"][:, right]) and got["y"][:, lost].isnan().all()
    assert got["final"].isnan().all()
    got = recurrence(x, g, h0, dy, dl, cuts, backward=dict(tiles=WORDS))
    right = [*range(3 * TILE, second), *range(5 * TILE, tokens)]
    lost = [*range(0, 3 * TILE), *range(second, 5 * TILE)]
    for n in ("dx", "dg"):
        assert torch.equal(got[n][:, right], want[n][:, right]) and got[n][:, lost].isnan().all(), n
    assert got["dh0"].isnan().all() and torch.equal(got["y"], want["y"])
    again = recurrence(x, g, h0, dy, dl, cuts)
    assert all(torch.equal(again[n], want[n]) for n in want)


LAYOUTS = {
    "one": [3 * TILE + 70],
    "two in a warp": [TILE + 53, 200],  # starts and ends inside the warp that is kept back
    "many in a warp": [TILE + 50, 3, 1, 4, 0, 130, 20],
    "at its borders": [48, 16, 64, 48, 100],
    "short": [5] * 40,
}


@pytest.mark.gpu
@pytest.mark.parametrize("gdtype", [FP32, BF16])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_tokens_that_do_not_come(layout, gdtype):
    """One warp's tokens of every tile: NaN, like all that follows from them inside their sequence."""
    warp, channels, lengths = 3, 128, LAYOUTS[layout]
    tokens = sum(lengths)
    x, g, dy = sequence(tokens, channels, seed=1)
    g = g.to(gdtype)
    cuts = torch.tensor([0] + lengths, device="cuda").cumsum(0).int()
    n = len(lengths)
    h0, dl = torch.randn(n, channels, device="cuda"), torch.randn(n, channels, device="cuda")
    want = recurrence(x, g, h0, dy, dl, cuts)
    kept_back = lambda t: t % TILE // WARP == warp  # noqa: E731
    spans = [(sum(lengths[:i]), sum(lengths[: i + 1])) for i in range(n)]
    state, adjoint, before = [False] * tokens, [False] * tokens, [False] * tokens
    for lo, hi in spans:
        bad = inside = False
        for t in range(lo, hi):
            inside = inside and t % TILE != 0  # the backward starts each tile from the forward's state
            before[t] = inside or kept_back(t)
            bad, inside = bad or kept_back(t), inside or kept_back(t)
            state[t] = bad
        bad = False
        for t in reversed(range(lo, hi)):
            bad = bad or kept_back(t)
            adjoint[t] = bad
    assert any(state) and any(adjoint)

    def check(got, n, lost):
        lost = torch.tensor(lost, device="cuda")
        where = lost[None, :, None] if got[n].dim() == 3 else lost[:, None]
        assert torch.equal(got[n].isnan(), where.expand_as(got[n])), n
        assert torch.equal(torch.where(where, 0, got[n]), torch.where(where, 0, want[n])), n

    got = recurrence(x, g, h0, dy, dl, cuts, forward=dict(tiles=1 << warp))
    check(got, "y", state)
    check(got, "final", [hi > lo and state[hi - 1] for lo, hi in spans])
    got = recurrence(x, g, h0, dy, dl, cuts, backward=dict(tiles=1 << warp))
    check(got, "dx", adjoint)
    check(got, "dg", [a or b for a, b in zip(adjoint, before)])
    check(got, "dh0", [hi > lo and adjoint[lo] for lo, hi in spans])
    again = recurrence(x, g, h0, dy, dl, cuts)
    assert all(torch.equal(again[n], want[n]) for n in want)


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("width,dtype", [(1024, BF16), (4096, BF16), (16384, BF16), (2048, FP32), (8192, FP32)])
def test_rows_that_do_not_come(width, dtype, checkpoint):
    """Streamed rows from one row on: their outputs are NaN, and so are the parameters' gradients, which need every row."""
    from miles_ext_kernels_b200.cake.layer_norm import layer_norm

    rows, served = 1500, 700
    gen = torch.Generator(device="cuda").manual_seed(width)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(dtype)  # noqa: E731
    x, w, b, dy = randn(rows, width), randn(width), randn(width), randn(rows, width)

    def step(forward=None, backward=None):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        with withheld(**(forward or {})):
            y = layer_norm(*leaves, checkpoint=checkpoint)
        with withheld(**(backward or {})):
            return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = step()
    y, dx, dw, _ = step(forward=dict(rows_served=served))
    for got, ref in ((y, want[0]), (dx, want[1])):  # the statistics and the codes of those rows are NaN as well
        assert torch.equal(got[:served], ref[:served]) and got[served:].isnan().all()
    assert dw.isnan().all()
    y, dx, dw, db = step(backward=dict(rows_served=served))
    assert torch.equal(y, want[0]) and torch.equal(dx[:served], want[1][:served]) and dx[served:].isnan().all()
    assert dw.isnan().all() and db.isnan().all()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
