"""LayerNorm: the op's declaration and refusals (CPU); the kernels against plain 64-bit forms at widths of every kernel
shape and alignment, parameters of each type or none, strided and offset rows, the 8-bit checkpoint, rows that are not
finite, other streams, captured graphs (GPU).  Tolerances: one rounding to the output's type plus a bound on what FP32
sums may add, derived in the oracle."""

from __future__ import annotations

import pytest
import torch

from oracle import rows_oracle as R

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def test_the_op_declaration_and_its_refusals():
    import miles_ext_kernels_b200 as package
    from miles_ext_kernels_b200 import cake
    from miles_ext_kernels_b200.cake import layer_norm

    assert "layer_norm" in cake.OPS
    op = cake.op_spec("layer_norm")
    assert op.variants == ("det", "fast") and set(op.exports) == {"check_supported", "layer_norm"}
    assert not op.has_variant_flag  # no miles argument selects it
    package.configure(cake_layer_norm_variant="fast")
    assert cake.variant("layer_norm") == "fast"
    package.configure()
    with pytest.raises(ValueError, match="BF16, FP16 or FP32 rows"):
        layer_norm.check_supported(64, torch.float64)
    with pytest.raises(ValueError, match="weight and bias"):
        layer_norm.check_supported(64, BF16, torch.float64)
    with pytest.raises(ValueError, match="rows of 1 to"):
        layer_norm.check_supported(0, BF16)
    with pytest.raises(ValueError, match="rows of 1 to"):
        layer_norm.check_supported(200705, BF16, checkpoint="e4m3")
    f, x = layer_norm.layer_norm, torch.zeros(2, 8)
    for match, call in (
        ("checkpoint must be one of", lambda: f(x, checkpoint="int8")),
        (r"weight must be \[8\]", lambda: f(x, torch.ones(7))),
        (r"bias must be \[8\]", lambda: f(x, None, torch.ones(1, 8))),
        ("one type", lambda: f(x, torch.ones(8), torch.ones(8, dtype=BF16))),
        ("BF16, FP16 or FP32 rows", lambda: f(x.double())),
        ("weight and bias", lambda: f(x, torch.ones(8, dtype=torch.float64))),
        ("rows of 1 to", lambda: f(torch.zeros(2, 0))),
        ("at least one dimension", lambda: f(torch.tensor(1.0))),
        ("must be a CUDA tensor", lambda: f(x)),
    ):
        with pytest.raises(ValueError, match=match):
            call()


def test_the_library_checks_its_arguments_without_a_gpu():
    import ctypes

    from miles_ext_kernels_b200.cake._runtime import loader

    lib = loader.load_library()
    i64, p = ctypes.c_int64, ctypes.c_void_p
    args = lambda **k: [p(64), k.get("type", 0), None, None, 0, p(64), None, None, p(64) if k.get("codes") else None,  # noqa: E731
                        i64(k.get("rows", 1)), i64(k.get("width", 8)), i64(k.get("stride", 8)), ctypes.c_float(1e-5), None]
    assert lib.mek_layer_norm_fwd(*args(type=3)) == 2 and "element type" in lib.last_error()
    assert lib.mek_layer_norm_fwd(*args(rows=0)) == 1 and "rows=0" in lib.last_error()
    assert lib.mek_layer_norm_fwd(*args(width=1 << 25)) == 1
    assert lib.mek_layer_norm_fwd(*args(stride=-8)) == 1 and "negative" in lib.last_error()
    assert lib.mek_layer_norm_fwd(*args(codes=True, width=200705)) == 2
    assert lib.mek_layer_norm_fwd(None, *args()[1:]) == 1 and "null" in lib.last_error()
    none = [None] * 16
    assert lib.mek_layer_norm_bwd(*none) == 1
    assert lib.mek_layer_norm_partial_rows(i64(0), i64(8), 0) == 0
    for width in (1, 8, 100, 4096, 16384, 40000):
        assert 1 <= lib.mek_layer_norm_partial_rows(i64(1 << 20), i64(width), 2) <= 148 * 16


def make(rows, width, dtype, param, seed=0, offset=0.3):
    gen = torch.Generator(device="cuda").manual_seed(seed * 977 + rows * 31 + width)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    x = (randn(rows, width) * (0.5 + randn(width).abs()) + offset).to(dtype)
    w = (1 + 0.2 * randn(width)).to(param) if param is not None else None
    b = (0.3 * randn(width)).to(param) if param is not None else None
    return x, w, b, randn(rows, width).to(dtype)


def run(x, w, b, dy, eps=1e-5, checkpoint=None):
    from miles_ext_kernels_b200.cake.layer_norm import layer_norm

    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves, eps, checkpoint=checkpoint)
    assert y.dtype == x.dtype and y.shape == x.shape
    y.backward(dy)
    out = {"y": y.detach(), "dx": leaves[0].grad}
    if w is not None:
        out["dw"] = leaves[1].grad
    if b is not None:
        out["db"] = leaves[2].grad
    return out


def codes_of(x, w, b, eps=1e-5):
    from miles_ext_kernels_b200.cake._impl.layer_norm import ops

    return ops._forward(x, w, b, eps, True, True)[1][1]


def check(got, x, w, b, dy, eps=1e-5, codes=None, what=""):
    width = x.shape[-1]
    x, dy = x.reshape(-1, width), dy.reshape(-1, width)
    y, unit, rstd, slack, y_slack = R.layer_norm(x, w, b, eps)
    assert R.misses(got["y"].reshape(-1, width), y, y_slack) == 0, f"{what} y"
    if codes is not None:
        assert R.e4m3_misses(codes, unit, slack) == 0, f"{what} codes"
        unit, slack = codes.view(torch.float8_e4m3fn).double(), torch.zeros_like(unit)
    for name, (want, allow) in R.layer_norm_bwd(dy, unit, rstd, w, slack).items():
        if name in got:
            have = got[name].reshape(want.shape)
            assert R.misses(have, want, allow) == 0, f"{what} {name}"
            if want.abs().max() > 0 and name == "dx" and width > 2:
                assert R.misses((have.double() * 1.02).to(have.dtype), want, allow) > 0, f"{what} {name}: the gate is too loose"


WIDTHS = (1, 2, 7, 32, 128, 250, 256, 257, 512, 1000, 1024, 1157, 2048, 2304, 4096, 5000, 8192, 10007, 16384, 20000, 40008)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,param", [(BF16, BF16), (BF16, FP32), (FP16, FP16), (FP32, FP32), (FP32, None)])
@pytest.mark.parametrize("width", WIDTHS)
def test_against_64_bits_at_every_kernel_shape(width, dtype, param):
    for rows in (1, 5, 331):
        x, w, b, dy = make(rows, width, dtype, param)
        got = run(x, w, b, dy)
        check(got, x, w, b, dy, what=f"{rows} x {width}")
        again = run(x, w, b, dy)
        for name in got:
            assert torch.equal(got[name], again[name]), name  # fixed-order sums: the same bits


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", [(32771, 128), (4099, 1157), (5000, 4096), (70001, 16)])
def test_many_rows(rows, width):
    x, w, b, dy = make(rows, width, BF16, FP32, seed=1)
    check(run(x, w, b, dy), x, w, b, dy, what=f"{rows} x {width}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,param", [(BF16, BF16), (FP16, FP32), (FP32, FP32), (BF16, None)])
@pytest.mark.parametrize("width", (1, 7, 128, 257, 1024, 1157, 4096, 8192, 16384, 40008))
def test_the_8_bit_checkpoint(width, dtype, param):
    for rows in (1, 203):
        x, w, b, dy = make(rows, width, dtype, param, seed=2)
        got = run(x, w, b, dy, checkpoint="e4m3")
        assert torch.equal(got["y"], run(x, w, b, dy)["y"])  # what is kept does not change the output
        check(got, x, w, b, dy, codes=codes_of(x, w, b), what=f"{rows} x {width}")


@pytest.mark.gpu
def test_the_checkpoint_keeps_eight_bits_and_lets_the_input_go():
    from miles_ext_kernels_b200.cake.layer_norm import layer_norm

    rows, width = 4096, 4096
    x = torch.randn(rows, width, device="cuda", dtype=BF16).requires_grad_()
    torch.cuda.synchronize()
    held = []
    for checkpoint in (None, "e4m3"):
        before = torch.cuda.memory_allocated()
        doubled = x * 2  # an activation that only the norm needs
        y = layer_norm(doubled, checkpoint=checkpoint)
        del doubled
        held.append(torch.cuda.memory_allocated() - before)
        del y
    n = rows * width
    assert held[0] >= 4 * n and held[1] <= 3 * n + 64 * 1024


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_strided_offset_and_higher_dimensional_rows(dtype):
    width = 512
    x, w, b, dy = make(330, width, dtype, FP32, seed=3)
    want = run(x, w, b, dy)
    for pad, offset in ((8, 0), (8, 8), (3, 1), (40, 16)):
        wide = torch.full((330, width + pad), float("nan"), device="cuda", dtype=dtype)
        view = wide[:, offset : offset + width] if offset + width <= width + pad else wide[:, :width]
        view.copy_(x)
        got = run(view, w, b, dy)
        for name in ("y", "dx"):
            if (width + pad) % 8 == 0 and offset % 8 == 0:
                assert torch.equal(got[name], want[name]), (name, pad, offset)
        check(got, x, w, b, dy, what=f"pad {pad} offset {offset}")
    cube = x.view(2, 3, 55, width)
    got = run(cube, w, b, dy.view(cube.shape))
    assert all(torch.equal(got[n].reshape(want[n].shape), want[n]) for n in want)
    turned = cube.transpose(0, 1)  # leading dimensions that do not merge
    got = run(turned, w, b, dy.view(cube.shape).transpose(0, 1))
    for n in ("y", "dx"):
        assert torch.equal(got[n].transpose(0, 1).reshape(330, width), want[n]), n
    columns = x.t().contiguous().t()  # unit stride across the rows
    got = run(columns, w, b, dy)
    assert all(torch.equal(got[n], want[n]) for n in want)
    assert run(x[:, 0, None].expand(330, 16), None, None, dy[:, :16])["y"].abs().max() < 1e-1  # equal elements
    one = run(x[0], w, b, dy[0])  # a single row without leading dimensions
    assert one["y"].shape == (width,) and torch.equal(one["y"], want["y"][0])


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_rows_with_nothing_in_them_and_rows_that_are_not_finite(checkpoint):
    for width in (128, 1157, 4096):
        x, w, b, dy = make(20, width, BF16, BF16, seed=4)
        clean = run(x, w, b, dy, checkpoint=checkpoint)
        x[3] = 0
        x[5] = 7.0
        x[8, 1] = float("nan")
        x[11, 2] = float("inf")
        x[14, 0] = torch.finfo(BF16).min
        got = run(x, w, b, dy, checkpoint=checkpoint)
        assert torch.equal(got["y"][3], b) and torch.equal(got["y"][5], b)  # unit = 0
        assert got["y"][8].isnan().all() and got["y"][11].isnan().all()
        fine = [r for r in range(20) if r not in (3, 5, 8, 11, 14)]
        for name in ("y", "dx"):
            assert torch.equal(got[name][fine], clean[name][fine]), name
        assert torch.isfinite(got["dx"][3]).all()
        assert torch.equal(got["db"], clean["db"])  # does not read x


@pytest.mark.gpu
def test_empty_rows_missing_parameters_and_partial_gradients():
    from miles_ext_kernels_b200.cake.layer_norm import layer_norm

    x, w, b, dy = make(40, 96, BF16, FP32, seed=5)
    got = run(x[:0], w, b, dy[:0])
    assert got["y"].shape == (0, 96) and got["dw"].abs().sum() == 0 and got["db"].abs().sum() == 0
    for weight, bias in ((w, None), (None, b), (None, None)):
        check(run(x, weight, bias, dy), x, weight, bias, dy)
    full = run(x, w, b, dy)
    for wants in ((True, False, False), (False, True, False), (False, False, True), (True, False, True)):
        leaves = [t.detach().requires_grad_(flag) for t, flag in zip((x, w, b), wants)]
        layer_norm(*leaves).backward(dy)
        for leaf, flag, name in zip(leaves, wants, ("dx", "dw", "db")):
            assert (leaf.grad is not None) == flag and (not flag or torch.equal(leaf.grad, full[name])), (wants, name)
    with torch.no_grad():
        assert torch.equal(layer_norm(x.requires_grad_(), w, b), full["y"])
    x = x.detach().requires_grad_()
    y = layer_norm(x, w, b)
    (grad,) = torch.autograd.grad(y, x, dy.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_offsets_past_32_bits(checkpoint):
    """2.2 G elements a tensor: the last rows against the same rows on their own."""
    rows, width = 540_672, 4096
    x = torch.empty(rows, width, device="cuda", dtype=BF16).normal_()
    dy = torch.empty_like(x).normal_()
    w, b = torch.randn(width, device="cuda").to(BF16), torch.randn(width, device="cuda").to(BF16)
    assert x.numel() > 1 << 31
    got = run(x, w, b, dy, checkpoint=checkpoint)
    tail = run(x[-300:], w, b, dy[-300:], checkpoint=checkpoint)
    for name in ("y", "dx"):
        assert torch.equal(got[name][-300:], tail[name]), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 4097])
def test_rows_side_by_side_in_a_warp(rows, dtype):
    """Narrow rows share warps; the last warp's places may be empty, and a row's neighbours do not reach it."""
    for width in (3, 24, 64, 100, 128):
        x, w, b, dy = make(rows, width, dtype, FP32, seed=9)
        got = run(x, w, b, dy)
        check(got, x, w, b, dy, what=f"{rows} x {width}")
        if rows > 2:
            x[1] = float("nan")
            bad = run(x, w, b, dy)
            others = [r for r in range(rows) if r != 1]
            assert torch.equal(bad["y"][others], got["y"][others]) and torch.equal(bad["dx"][others], got["dx"][others])
            assert torch.equal(bad["db"], got["db"]) and bad["dw"].isnan().all()


@pytest.mark.gpu
def test_against_differences_of_the_forward():
    x, w, b, dy = make(3, 37, FP32, FP32, seed=6)
    got = run(x, w, b, dy)
    gen = torch.Generator(device="cuda").manual_seed(0)
    x64, w64, b64 = x.double(), w.double(), b.double()
    loss = lambda x_, w_, b_: float((R.layer_norm(x_, w_, b_, 1e-5)[0] * dy.double()).sum())  # noqa: E731
    for name, at, h in (("dx", x64, 1e-5), ("dw", w64, 1e-5), ("db", b64, 1e-5)):
        way = torch.randn(at.shape, device="cuda", generator=gen, dtype=torch.float64)
        moved = [dict(dx=(x64 + s * h * way, w64, b64), dw=(x64, w64 + s * h * way, b64), db=(x64, w64, b64 + s * h * way))[name]
                 for s in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * h)
        # central differences in 64 bits: h^2 of the third derivative and 1e-16 / h of rounding; the gradient is FP32
        scale = float((got[name].double() * way).abs().sum())
        assert abs(float((got[name].double() * way).sum()) - slope) <= 1e-5 * scale + 1e-6, name


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_other_streams_the_pool_and_captured_graphs(checkpoint):
    import miles_ext_kernels_b200 as package
    from miles_ext_kernels_b200.cake.layer_norm import layer_norm

    x, w, b, dy = make(600, 1000, BF16, BF16, seed=7)
    want = run(x, w, b, dy, checkpoint=checkpoint)
    package.configure(cake_workspace_pool_bytes=1 << 28)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, w, b, dy, checkpoint=checkpoint)
        again = run(x, w, b, dy, checkpoint=checkpoint)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) and torch.equal(again[n], want[n]) for n in want)

    graphs = []
    for k in range(2):  # two graphs that could share scratch, replayed in turn and at once
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        grad = dy.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer_norm(*leaves, checkpoint=checkpoint)
            dx, dw, db = torch.autograd.grad(y, leaves, grad)
        graphs.append((graph, leaves, grad, {"y": y, "dx": dx, "dw": dw, "db": db}))
    x2, w2, b2, dy2 = make(600, 1000, BF16, BF16, seed=8)
    want2 = run(x2, w2, b2, dy2, checkpoint=checkpoint)
    with torch.no_grad():
        for leaf, t in zip(graphs[1][1], (x2, w2, b2)):
            leaf.copy_(t)
        graphs[1][2].copy_(dy2)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    for (_, _, _, out), ref in zip(graphs, (want, want2)):
        assert all(torch.equal(out[n].detach(), ref[n]) for n in ref)
