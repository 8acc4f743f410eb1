"""Plain 64-bit forms of the row operators, written from their definitions: LayerNorm and its 8-bit checkpoint."""

from __future__ import annotations

import torch

__all__ = ["U32", "e4m3_misses", "half_step", "layer_norm", "layer_norm_bwd", "misses"]

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
