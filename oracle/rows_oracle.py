"""Plain 64-bit forms of the row operators, written from their definitions: LayerNorm and its 8-bit checkpoint, the gated
linear recurrence."""

from __future__ import annotations

import torch

__all__ = ["U32", "e4m3_misses", "half_step", "layer_norm", "layer_norm_bwd", "linear_recurrence", "misses"]

U32 = 2.0**-24  # half a step of FP32, relative


def half_step(dtype: torch.dtype) -> float:
    """The largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def misses(got: torch.Tensor, want: torch.Tensor, slack: torch.Tensor) -> int:
    """How many values of ``got`` are further from the 64-bit ``want`` than one rounding to their type, half its smallest
    subnormal step and ``slack``; non-finite values have to be alike."""
    got64, info = got.double(), torch.finfo(got.dtype)
    bound = half_step(got.dtype) * (want.abs() + slack) + info.smallest_normal * half_step(got.dtype) * 2 + slack
    fine = torch.isfinite(want)
    bad = torch.where(fine, ~((got64 - want).abs() <= bound), torch.isfinite(got64))
    return int(bad.sum())


def e4m3_misses(codes: torch.Tensor, want: torch.Tensor, slack: torch.Tensor) -> int:
    """How many e4m3 codes (uint8) stand for a value further from ``want`` than half a step -- 2^-4 of the value, 2^-10
    among the subnormals -- and ``slack``."""
    value = codes.view(torch.float8_e4m3fn).double()
    return int((~((value - want).abs() <= (want.abs() + slack) * 2.0**-4 + 2.0**-10 + slack)).sum())


def layer_norm(x, weight, bias, eps):
    """``(y, unit, rstd, unit_slack, y_slack)`` in 64 bits; the slacks bound what FP32 sums and products may add: a mean
    is a sum of C terms whose partial sums round at most 64 times along any path (16 in a thread's registers, ten levels
    of shuffles, 32 warps), each by half a step of the terms' absolute mean."""
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = 1 / torch.sqrt(centred.square().mean(-1, keepdim=True) + eps)
    unit = centred * rstd
    slack = 64 * U32 * ((x.abs().mean(-1, keepdim=True) + x.abs()) * rstd + unit.abs())
    # an offset mean moves the variance too: by its own error squared, which the first term covers, and by the
    # centred values' relative error, twice
    slack = slack + unit.abs() * 64 * U32 * 2 * (x.abs().mean(-1, keepdim=True) * rstd)
    w = 1.0 if weight is None else weight.double()
    b = 0.0 if bias is None else bias.double()
    y = unit * w + b
    y_slack = slack * abs(w) + 2 * U32 * y.abs()
    return y, unit, rstd, slack, y_slack


def layer_norm_bwd(dy, unit, rstd, weight, unit_slack):
    """``{name: (value, slack)}`` of dx, dw, db for the given normalised rows."""
    dy = dy.double()
    w = 1.0 if weight is None else weight.double()
    dn = dy * w
    m1, m2 = dn.mean(-1, keepdim=True), (dn * unit).mean(-1, keepdim=True)
    dx = rstd * (dn - m1 - unit * m2)
    size = dn.abs() + dn.abs().mean(-1, keepdim=True) + unit.abs() * (dn * unit).abs().mean(-1, keepdim=True)
    dx_slack = rstd * (64 * U32 * size + unit_slack * m2.abs() + unit.abs() * (dn.abs() * unit_slack).mean(-1, keepdim=True))
    dx_slack = dx_slack + dx.abs() * 64 * U32
    # a block adds its rows' terms one after the other, at most 512 of them in the tests
    dw, db = (dy * unit).sum(0), dy.sum(0)
    dw_slack = 512 * U32 * (dy * unit).abs().sum(0) + (dy.abs() * unit_slack).sum(0)
    return {"dx": (dx, dx_slack), "dw": (dw, dw_slack), "db": (db, 512 * U32 * dy.abs().sum(0))}


def linear_recurrence(x, g, lengths, h0=None, dy=None, d_final=None):
    """``{name: (value, slack)}`` of the packed tokens ``x``, ``g [T, C]`` of consecutive sequences of ``lengths``, token by
    token in 64 bits.  The slack follows the sizes: with m the sum of magnitudes that the state could have (no
    cancellation), a step adds at most 6 half steps of FP32 to what it carries over -- a decay within 3 half steps of
    exp(g), its product and the fold's -- and 2 to the new state.  A decay below 2^-125.5 counts as zero, which takes
    away less than 2^-125.5 = 1.663e-38 of what the step carries over (2^-126 = 1.1755e-38, times 2^0.5), and no
    more than the decay itself."""
    total, channels = x.shape
    x, a = x.double(), g.double().exp()
    n = len(lengths)
    h0 = x.new_zeros(n, channels) if h0 is None else h0.double()
    y, dy_slack = torch.zeros_like(x), torch.zeros_like(x)
    before, before_slack = torch.zeros_like(x), torch.zeros_like(x)
    final, final_slack = h0.clone(), torch.zeros_like(h0)
    start = 0
    spans = []
    for i, length in enumerate(lengths):
        spans.append((start, start + length))
        h, m, e = h0[i], h0[i].abs(), torch.zeros_like(h0[i])
        for t in range(start, start + length):
            before[t], before_slack[t] = h, e
            e = a[t] * (e + 6 * U32 * m) + a[t].clamp(max=1.67e-38) * m
            h, m = a[t] * h + x[t], a[t] * m + x[t].abs()
            e = e + 2 * U32 * m
            y[t], dy_slack[t] = h, e
        final[i], final_slack[i] = h, e
        start += length
    out = {"y": (y, dy_slack), "final": (final, final_slack)}
    if dy is None:
        return out
    dy = dy.double()
    d_final = torch.zeros_like(h0) if d_final is None else d_final.double()
    dx, dg, dx_slack, dg_slack = (torch.zeros_like(x) for _ in range(4))
    dh0, dh0_slack = d_final.clone(), torch.zeros_like(h0)
    for i, (lo, hi) in enumerate(spans):
        c, m, e = d_final[i], d_final[i].abs(), torch.zeros_like(d_final[i])
        for t in range(hi - 1, lo - 1, -1):
            dh, m = dy[t] + c, dy[t].abs() + m
            e = e + 2 * U32 * m
            dx[t], dx_slack[t] = dh, e
            c = a[t] * dh
            e, m = a[t] * (e + 6 * U32 * m) + a[t].clamp(max=1.67e-38) * m, a[t] * m
            dg[t] = c * before[t]
            dg_slack[t] = e * before[t].abs() + c.abs() * before_slack[t] + e * before_slack[t] + 4 * U32 * dg[t].abs()
        dh0[i], dh0_slack[i] = c, e
    out.update(dx=(dx, dx_slack), dg=(dg, dg_slack), dh0=(dh0, dh0_slack))
    return out
