"""LayerNorm where its rows or its gradient meet the borders of the accesses: widths whose codes bulk copies cannot move,
and gradients at odd addresses, against 64 bits (GPU)."""

from __future__ import annotations

import pytest
import torch

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("width,dtype,param", [
    (520, BF16, BF16), (1000, BF16, FP32), (1000, FP16, FP16), (2056, BF16, BF16), (4104, BF16, None), (8200, BF16, BF16),
    (16376, FP16, FP32), (516, FP32, FP32), (1004, FP32, BF16), (2052, FP32, FP32), (4100, FP32, None), (8196, FP32, FP32)])
def test_checkpoints_of_widths_that_are_no_multiple_of_16(width, dtype, param):
    """Rows of wide accesses whose 8-bit codes do not start on 16 bytes: loaded, not streamed, by 128 threads and more."""
    import test_layer_norm as base

    for rows in (1, 203, 700):
        x, w, b, dy = base.make(rows, width, dtype, param, seed=31)
        got = base.run(x, w, b, dy, checkpoint="e4m3")
        base.check(got, x, w, b, dy, codes=base.codes_of(x, w, b), what=f"{rows} x {width}")
        assert torch.equal(got["y"], base.run(x, w, b, dy)["y"])
        again = base.run(x, w, b, dy, checkpoint="e4m3")
        assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("width,dtype", [(64, BF16), (1024, BF16), (4096, BF16), (16384, FP16), (2048, FP32), (20000, BF16)])
def test_a_gradient_and_parameters_at_odd_addresses(width, dtype, checkpoint):
    import test_layer_norm as base

    x, w, b, dy = base.make(150, width, dtype, dtype, seed=32)

    def moved(t, offset=1):
        return torch.empty(t.numel() + offset, device="cuda", dtype=t.dtype)[offset:].view(t.shape).copy_(t)

    codes = base.codes_of(x, w, b) if checkpoint else None
    base.check(base.run(x, w, b, moved(dy), checkpoint=checkpoint), x, w, b, dy, codes=codes, what="dy")
    base.check(base.run(x, moved(w), moved(b, 3), dy, checkpoint=checkpoint), x, w, b, dy, codes=codes, what="w, b")
    x_off = moved(x)  # a forward of one-element accesses and, with dy as it was, what its backward makes of it
    codes = base.codes_of(x_off, w, b) if checkpoint else None
    base.check(base.run(x_off, w, b, dy, checkpoint=checkpoint), x, w, b, dy, codes=codes, what="x")
