"""The gated linear recurrence: its declaration and refusals (CPU); the kernels against the token-by-token form in 64
bits at lengths around a warp's and a tile's tokens, odd widths, every pair of types, packed sequences with empty ones
and tokens behind the last, initial and final states with their gradients, strided operands, decays of zero and one,
sequences that are not finite, other streams, captured graphs; the single-token step with padding and repeated slots
(GPU).  Tolerances: one rounding to the output's type plus a bound the oracle carries along the recurrence."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import rows_oracle as R

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def test_the_op_declaration_and_its_refusals():
    import miles_ext_kernels_b200 as package
    from miles_ext_kernels_b200 import cake
    from miles_ext_kernels_b200.cake import linear_recurrence as op

    assert "linear_recurrence" in cake.OPS
    spec = cake.op_spec("linear_recurrence")
    assert set(spec.exports) == {"check_supported", "gated_linear_recurrence", "gated_linear_recurrence_step"}
    assert spec.variants == ("det", "fast") and not spec.has_variant_flag
    package.configure(cake_linear_recurrence_variant="fast")
    assert cake.variant("linear_recurrence") == "fast"
    package.configure()
    with pytest.raises(ValueError, match="BF16, FP16 or FP32"):
        op.check_supported(64, torch.float64)
    with pytest.raises(ValueError, match="BF16, FP16 or FP32"):
        op.check_supported(64, BF16, torch.int32)
    with pytest.raises(ValueError, match="channels"):
        op.check_supported(0, BF16)
    f, x = op.gated_linear_recurrence, torch.zeros(1, 4, 8)
    cu = torch.tensor([0, 2, 4])
    for match, call in (
        (r"x must be \[B, T", lambda: f(x[0], x[0])),
        ("g must have x's shape", lambda: f(x, x[:, :, :1])),
        ("BF16, FP16 or FP32", lambda: f(x.double(), x)),
        ("channels", lambda: f(torch.zeros(1, 4, 0), torch.zeros(1, 4, 0))),
        ("at least one batch row", lambda: f(torch.zeros(0, 4, 8), torch.zeros(0, 4, 8))),
        ("packs the sequences of one row", lambda: f(torch.zeros(2, 4, 8), torch.zeros(2, 4, 8), cu_seqlens=cu)),
        ("cu_seqlens must be", lambda: f(x, x, cu_seqlens=cu[:1])),
        ("cu_seqlens must be", lambda: f(x, x, cu_seqlens=cu.float())),
        ("initial_state must be", lambda: f(x, x, torch.zeros(2, 8))),
        ("initial_state must be", lambda: f(x, x, torch.zeros(1, 8, dtype=BF16))),
        ("initial_state must be", lambda: f(x, x, torch.zeros(1, 8), cu_seqlens=cu)),
        ("must be a CUDA tensor", lambda: f(x, x)),
    ):
        with pytest.raises(ValueError, match=match):
            call()
    s, x, pool = op.gated_linear_recurrence_step, torch.zeros(3, 8), torch.zeros(5, 8)
    for match, call in (
        (r"x must be \[rows", lambda: s(x[0], x[0], pool)),
        ("g must have x's shape", lambda: s(x, x[:2], pool)),
        ("BF16, FP16 or FP32", lambda: s(x, x.double(), pool)),
        ("state must be FP32", lambda: s(x, x, pool[:, :4])),
        ("state must be FP32", lambda: s(x, x, pool.bfloat16())),
        ("state must be FP32", lambda: s(x, x, pool[:0])),
        ("need as many states", lambda: s(x, x, pool[:2])),
        ("state_indices must be", lambda: s(x, x, pool, torch.zeros(2, dtype=torch.int32))),
        ("state_indices must be", lambda: s(x, x, pool, torch.zeros(3))),
        ("has no gradient", lambda: s(x.clone().requires_grad_(), x, pool)),
        ("must be a CUDA tensor", lambda: s(x, x, pool)),
    ):
        with pytest.raises(ValueError, match=match):
            call()


def test_the_library_checks_its_arguments_without_a_gpu():
    import ctypes

    from miles_ext_kernels_b200.cake._runtime import loader

    lib = loader.load_library()
    i64, p = ctypes.c_int64, ctypes.c_void_p
    assert lib.mek_linear_recurrence_tile() >= 1

    def fwd(x=64, x_type=0, batch=1, tokens=4, channels=8, cu=None, seqs=1):
        return lib.mek_linear_recurrence_fwd(p(x), x_type, p(64), 2, p(64), i64(batch), i64(tokens), i64(channels), i64(0),
                                             i64(8), i64(0), i64(8), p(cu), i64(seqs), None, None, None, None)

    assert fwd(x=None) == 1 and "null" in lib.last_error()
    assert fwd(x_type=5) == 2 and "element type" in lib.last_error()
    assert fwd(tokens=0) == 1 and fwd(channels=0) == 1 and fwd(batch=0) == 1
    assert fwd(cu=64, batch=2) == 1 and "one batch row" in lib.last_error()
    assert fwd(tokens=1 << 20) == 1 and "no room" in lib.last_error()
    assert fwd(tokens=1 << 30, channels=1 << 23) == 1 and "tiles" in lib.last_error()
    step = lambda rows, pool, slots=None: lib.mek_linear_recurrence_step(  # noqa: E731
        p(64), 0, p(64), 0, p(64), p(slots), 0, p(64), i64(rows), i64(pool), i64(8), i64(8), i64(8), i64(8), None)
    assert step(0, 1) == 1 and step(1, 0) == 1 and step(4, 3) == 1


def gates(kind, shape, gen):
    """Log decays: ``mixed`` memories of 1 to 1,000 tokens, ``closed`` (mostly no memory), ``open`` (a = 1 exactly and a
    little growth), ``edge``: zeros of the decay, the smallest decays, none."""
    u = torch.rand(*shape, device="cuda", generator=gen)
    if kind == "mixed":
        rate = torch.exp(torch.rand(shape[-1], device="cuda", generator=gen) * math.log(1e-3))
        return -torch.nn.functional.softplus(torch.randn(*shape, device="cuda", generator=gen)) * rate
    if kind == "closed":
        return -30 * u
    if kind == "open":
        return torch.where(u < 0.7, 0.0, 0.01 * u)
    return torch.where(u < 0.3, -math.inf, torch.where(u < 0.6, -86.0 - 20 * u, torch.where(u < 0.8, -1e-6 * u, 0.0)))


def make(batch, tokens, channels, dtype, gdtype, sequences, kind="mixed", seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7 + tokens * 131 + channels)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    x = randn(batch, tokens, channels).to(dtype)
    g = gates(kind, (batch, tokens, channels), gen).to(gdtype)
    return x, g, randn(sequences, channels), randn(batch, tokens, channels).to(dtype), randn(sequences, channels)


def run(x, g, h0, dy, d_final, cu=None, final=True):
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence

    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, g, h0)]
    y, last = gated_linear_recurrence(*leaves, output_final_state=final, cu_seqlens=cu)
    assert y.shape == x.shape and y.dtype == x.dtype and (last is not None) == final
    outs, grads = ([y, last], [dy, d_final]) if final else ([y], [dy])
    torch.autograd.backward(outs, grads)
    got = {"y": y.detach(), "dx": leaves[0].grad, "dg": leaves[1].grad}
    if final:
        got["final"] = last.detach()
    if h0 is not None:
        got["dh0"] = leaves[2].grad
    return got


def check(got, x, g, h0, dy, d_final, lengths, what="", tail=0):
    channels = x.shape[-1]
    flat = lambda t: t.reshape(-1, channels)  # noqa: E731
    used = x.shape[0] * x.shape[1] - tail
    want = R.linear_recurrence(flat(x)[:used], flat(g)[:used], lengths, h0, flat(dy)[:used], d_final if "final" in got else None)
    for name, value in got.items():
        ref, slack = want[name]
        value = flat(value) if name in ("y", "dx", "dg") else value
        if name in ("y", "dx", "dg"):
            assert tail == 0 or value[used:].abs().max() == 0, f"{what} {name}: tokens behind the last sequence"
            value = value[:used]
        assert R.misses(value, ref, slack) == 0, f"{what} {name}"
        if name in ("y", "dx") and ref.numel() > 50:
            assert R.misses((value.double() * 1.02).to(value.dtype), ref, slack) > 0, f"{what} {name}: the gate is too loose"


TYPES = [(BF16, FP32), (BF16, BF16), (FP16, FP32), (FP16, FP16), (FP32, FP32), (FP32, BF16), (BF16, FP16)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gdtype", TYPES)
@pytest.mark.parametrize("batch,tokens,channels", [(1, 1, 1), (3, 2, 5), (1, 15, 64), (2, 16, 66), (1, 17, 130), (1, 127, 63),
                                                   (2, 128, 64), (1, 129, 33), (3, 257, 70), (1, 700, 200)])
def test_dense_batches_against_64_bits(batch, tokens, channels, dtype, gdtype):
    x, g, h0, dy, dl = make(batch, tokens, channels, dtype, gdtype, batch)
    got = run(x, g, h0, dy, dl)
    check(got, x, g, h0, dy, dl, [tokens] * batch)
    again = run(x, g, h0, dy, dl)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["closed", "open", "edge"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_decays_of_zero_and_one(kind, dtype):
    x, g, h0, dy, dl = make(2, 300, 96, dtype, FP32, 2, kind)
    check(run(x, g, h0, dy, dl), x, g, h0, dy, dl, [300] * 2, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,tail", [
    ([1], 0), ([0, 5], 0), ([5, 0], 0), ([1] * 70, 0), ([0, 0, 3, 0, 0, 130, 0, 1, 16, 0], 0), ([128, 128, 1], 0),
    ([16, 16, 32, 64], 7), ([300, 2, 255], 40), ([0] * 45 + [20] + [0] * 45, 0), ([0, 0], 3), ([513], 600), ([3] * 200, 5),
])
@pytest.mark.parametrize("channels,dtype,gdtype", [(70, BF16, FP32), (33, FP32, FP32)])
def test_packed_sequences(lengths, tail, channels, dtype, gdtype):
    total = sum(lengths) + tail
    x, g, h0, dy, dl = make(1, total, channels, dtype, gdtype, len(lengths), seed=1)
    if tail:  # whatever lies behind the last sequence stays there
        x[:, total - tail :], dy[:, total - tail :] = math.nan, math.inf
    cu = torch.tensor([0] + lengths, device="cuda").cumsum(0)
    got = run(x, g, h0, dy, dl, cu.int())
    check(got, x, g, h0, dy, dl, lengths, str(lengths)[:40], tail)
    wide = run(x, g, h0, dy, dl, cu)  # int64 boundaries
    assert all(torch.equal(got[n], wide[n]) for n in got)
    bare = run(x, g, None, dy, None, cu.int(), final=False)
    check(bare, x, g, None, dy, None, lengths, "no states", tail)


@pytest.mark.gpu
def test_packed_sequences_have_the_bits_of_each_on_its_own_where_tiles_agree():
    lengths = [256, 128, 384]
    x, g, h0, dy, dl = make(1, sum(lengths), 128, BF16, FP32, 3, seed=2)
    cu = torch.tensor([0, 256, 384, 768], dtype=torch.int32, device="cuda")
    got = run(x, g, h0, dy, dl, cu)
    for i in range(3):
        part = slice(int(cu[i]), int(cu[i + 1]))
        alone = run(x[:, part], g[:, part], h0[i : i + 1], dy[:, part], dl[i : i + 1])
        for n in ("y", "dx", "dg"):
            assert torch.equal(got[n][:, part], alone[n]), n
        for n in ("final", "dh0"):
            assert torch.equal(got[n][i : i + 1], alone[n]), n


@pytest.mark.gpu
def test_nothing_of_a_sequence_reaches_another():
    lengths = [40, 200, 7, 150]
    x, g, h0, dy, dl = make(1, sum(lengths), 64, FP32, FP32, 4, seed=3)
    cu = torch.tensor([0] + lengths, device="cuda").cumsum(0).int()
    clean = run(x, g, h0, dy, dl, cu)
    x[0, 60, 3], g[0, 61, 4], dy[0, 100, 5] = math.inf, math.nan, math.nan
    got = run(x, g, h0, dy, dl, cu)
    for n in ("y", "dx", "dg"):
        for rows in (slice(0, 40), slice(240, None)):
            assert torch.equal(got[n][:, rows], clean[n][:, rows]), n
    for n in ("final", "dh0"):
        assert torch.equal(got[n][[0, 2, 3]], clean[n][[0, 2, 3]]), n
    assert got["y"][0, 60, 3].isinf() and got["y"][0, 239, 4].isnan() and got["dx"][0, 40, 5].isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,channels", [(BF16, 128), (FP32, 37)])
def test_strided_and_higher_dimensional_operands(dtype, channels):
    x, g, h0, dy, dl = make(2, 150, channels, dtype, FP32, 2, seed=4)
    want = run(x, g, h0, dy, dl)
    wide = torch.full((2, 153, 3 * channels + 1), math.nan, device="cuda", dtype=dtype)
    view = wide[:, 2:152, channels : 2 * channels]
    view.copy_(x)
    gates_wide = torch.full((150, 2, channels + 4), math.nan, device="cuda")
    gview = gates_wide.transpose(0, 1)[:, :, 1 : channels + 1]
    gview.copy_(g)
    got = run(view, gview, h0, dy, dl)
    assert all(torch.equal(got[n], want[n]) for n in want)
    turned = run(x.transpose(1, 2).contiguous().transpose(1, 2), g, h0, dy, dl)  # channels not contiguous: copied
    assert all(torch.equal(turned[n], want[n]) for n in want)
    if channels % 2 == 0:
        heads = (2, 150, 2, channels // 2)
        got = run(x.view(heads), g.view(heads), h0.view(2, 2, -1), dy.view(heads), dl.view(2, 2, -1))
        assert all(torch.equal(got[n].reshape(want[n].shape), want[n]) for n in want)
        shared = g[:, :, None, : channels // 2].expand(heads)  # one gate for both heads
        leaf = g[:, :, : channels // 2].clone().requires_grad_()
        from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence

        y, _ = gated_linear_recurrence(x.view(heads), leaf[:, :, None].expand(heads))
        y.backward(dy.view(heads))
        alone = run(x.view(heads), shared, None, dy.view(heads), None, final=False)
        assert torch.equal(leaf.grad, alone["dg"].sum(2))
    flat = gview.expand(2, 150, channels)
    assert torch.equal(run(x[:, :1].expand(2, 150, channels), flat, h0, dy, dl)["y"],
                       run(x[:, :1].repeat(1, 150, 1), g, h0, dy, dl)["y"])


@pytest.mark.gpu
def test_calls_without_tokens_and_partial_gradients():
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence

    x, g, h0, dy, dl = make(2, 200, 40, BF16, FP32, 2, seed=5)
    empty = x[:, :0].detach().requires_grad_()
    state = h0.clone().requires_grad_()
    y, final = gated_linear_recurrence(empty, g[:, :0], state, output_final_state=True)
    assert y.shape == (2, 0, 40) and torch.equal(final, h0)
    final.backward(dl)
    assert torch.equal(state.grad, dl)
    full = run(x, g, h0, dy, dl)
    for wants in ((1, 0, 0), (0, 1, 0), (0, 0, 1)):
        leaves = [t.detach().requires_grad_(bool(w)) for t, w in zip((x, g, h0), wants)]
        outs = gated_linear_recurrence(*leaves, output_final_state=True)
        torch.autograd.backward(outs, (dy, dl))
        for leaf, w, n in zip(leaves, wants, ("dx", "dg", "dh0")):
            assert (leaf.grad is not None) == bool(w) and (not w or torch.equal(leaf.grad, full[n])), n
    with torch.no_grad():
        y, final = gated_linear_recurrence(x.requires_grad_(), g, h0, True)
    assert torch.equal(y, full["y"]) and torch.equal(final, full["final"]) and not y.requires_grad
    leaves = [t.detach().requires_grad_() for t in (x, g, h0)]
    _, final = gated_linear_recurrence(*leaves, output_final_state=True)
    final.backward(dl)  # only the final state is used
    check({"final": final.detach(), "dx": leaves[0].grad, "dg": leaves[1].grad, "dh0": leaves[2].grad}, x, g, h0,
          torch.zeros_like(dy), dl, [200] * 2)
    y, _ = gated_linear_recurrence(x.detach().requires_grad_(), g)
    (grad,) = torch.autograd.grad(y, y.grad_fn.next_functions[0][0].variable, dy.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@pytest.mark.gpu
def test_against_differences_of_the_forward():
    x, g, h0, dy, dl = make(1, 140, 6, FP32, FP32, 1, seed=6)
    got = run(x, g, h0, dy, dl)
    gen = torch.Generator(device="cuda").manual_seed(1)

    def loss(x_, g_, h_):
        out = R.linear_recurrence(x_[0], g_[0], [140], h_)
        return float((out["y"][0] * dy[0].double()).sum() + (out["final"][0] * dl.double()).sum())

    base = {"dx": x.double(), "dg": g.double(), "dh0": h0.double()}
    for name, at in base.items():
        way, h = torch.randn(at.shape, device="cuda", generator=gen, dtype=torch.float64), 1e-6
        ends = [loss(*(v + s * h * way if n == name else v for n, v in base.items())) for s in (1, -1)]
        slope = (ends[0] - ends[1]) / (2 * h)
        scale = float((got[name].double() * way).abs().sum())
        assert abs(float((got[name].double() * way).sum()) - slope) <= 1e-5 * scale + 1e-5, name


@pytest.mark.gpu
def test_long_sequences_on_few_channels():
    """Hundreds of tiles in one chain."""
    for channels, tokens in ((3, 30011), (64, 16384)):
        x, g, h0, dy, dl = make(1, tokens, channels, FP32, FP32, 1, seed=7)
        check(run(x, g, h0, dy, dl), x, g, h0, dy, dl, [tokens], f"{tokens} x {channels}")


@pytest.mark.gpu
def test_other_streams_the_pool_and_captured_graphs():
    import miles_ext_kernels_b200 as package
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence

    sets = [make(2, 1500, 200, BF16, FP32, 2, seed=s) for s in (8, 9)]
    wants = [run(*s) for s in sets]
    package.configure(cake_workspace_pool_bytes=1 << 28)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [run(*sets[0]) for _ in range(2)]
    here = run(*sets[1])
    torch.cuda.current_stream().wait_stream(side)
    for n in wants[0]:
        assert torch.equal(got[0][n], wants[0][n]) and torch.equal(got[1][n], wants[0][n]) and torch.equal(here[n], wants[1][n])
    graphs = []
    for _ in range(2):
        x, g, h0, dy, dl = (t.clone() for t in sets[0])
        leaves = [t.requires_grad_() for t in (x, g, h0)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, final = gated_linear_recurrence(*leaves, output_final_state=True)
            dx, dg, dh0 = torch.autograd.grad((y, final), leaves, (dy, dl))
        graphs.append((graph, [*leaves, dy, dl], dict(y=y, final=final, dx=dx, dg=dg, dh0=dh0)))
    with torch.no_grad():
        for have, new in zip(graphs[1][1], sets[1]):
            have.copy_(new)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    for (_, _, out), want in zip(graphs, wants):
        assert all(torch.equal(out[n].detach(), want[n]) for n in want)


@pytest.mark.gpu
def test_time_major_operands_and_a_backward_run_twice():
    """[T, B, C] memory behind [B, T, C] views: the token stride is the larger one."""
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence

    x, g, h0, dy, dl = make(3, 300, 128, BF16, BF16, 3, seed=13)
    want = run(x, g, h0, dy, dl)
    views = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, g, dy)]
    assert views[0].stride(0) == 128 and views[0].stride(1) == 3 * 128
    got = run(views[0], views[1], h0, views[2], dl)
    assert all(torch.equal(got[n], want[n]) for n in want)
    leaves = [t.clone().requires_grad_() for t in (x, g, h0)]
    outs = gated_linear_recurrence(*leaves, output_final_state=True)
    for _ in range(2):
        grads = torch.autograd.grad(outs, leaves, (dy, dl), retain_graph=True)
        assert all(torch.equal(a, want[n]) for a, n in zip(grads, ("dx", "dg", "dh0")))


@pytest.mark.gpu
def test_many_chains_and_many_short_sequences():
    """More chains than blocks (one warp looks back), batches of one tile, a batch of two tokens."""
    for batch, tokens, channels in ((40, 300, 1024), (300, 100, 64), (700, 2, 192)):
        x, g, h0, dy, dl = make(batch, tokens, channels, BF16, FP32, batch, seed=14)
        got = run(x, g, h0, dy, dl)
        for rows in (slice(0, 2), slice(batch - 2, batch)):
            part = {n: t[rows] for n, t in got.items()}
            check(part, x[rows], g[rows], h0[rows], dy[rows], dl[rows], [tokens] * 2, f"{batch} x {tokens} x {channels}")
        again = run(x, g, h0, dy, dl)
        assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """2.2 G elements a tensor; closed gates make the last tokens independent of the ones before."""
    tokens, channels = 540_672, 4096
    x = torch.empty(1, tokens, channels, device="cuda", dtype=BF16).normal_()
    g = torch.full((1, tokens, channels), -200.0, device="cuda", dtype=BF16)
    dy = torch.empty_like(x).normal_()
    assert x.numel() > 1 << 31
    got = run(x, g, None, dy, None, final=False)
    assert torch.equal(got["y"], x) and torch.equal(got["dx"], dy) and got["dg"].abs().max() == 0


# ---- the single-token step -------------------------------------------------------------------------------------------
def step_reference(x, g, state, slots):
    """Row after row in 64 bits: ``(y, state, y slack, state slack)``."""
    state, slack = state.double().clone(), torch.zeros_like(state, dtype=torch.float64)
    y, y_slack = torch.zeros(x.shape, dtype=torch.float64, device=x.device), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for r, slot in enumerate(slots):
        if 0 <= slot < state.shape[0]:
            a = g[r].double().exp()
            slack[slot] = a * slack[slot] + 6 * R.U32 * a * state[slot].abs() + 2 * R.U32 * (a * state[slot].abs() + x[r].double().abs())
            state[slot] = a * state[slot] + x[r].double()
            y[r], y_slack[r] = state[slot], slack[slot]
    return y, state, y_slack, slack


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gdtype", TYPES)
@pytest.mark.parametrize("rows,pool,channels", [(1, 1, 1), (1, 7, 64), (5, 9, 66), (33, 40, 1031), (300, 512, 128)])
def test_the_step_against_64_bits(rows, pool, channels, dtype, gdtype):
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence_step as step

    x, g, _, _, _ = make(1, rows, channels, dtype, gdtype, 1, seed=10)
    x, g = x[0], g[0]
    gen = torch.Generator().manual_seed(rows)
    state = torch.randn(pool, channels, device="cuda")
    order = torch.randperm(pool, generator=gen)[:rows].tolist()
    padded = [(-1 if r % 5 == 3 else s) for r, s in enumerate(order)]
    outside = [(pool + 3 if r % 7 == 2 else s) for r, s in enumerate(padded)]
    repeated = [outside[r // 3] for r in range(rows)]
    for slots in (None, order, padded, outside, repeated, [order[0]] * rows):
        for index in (torch.int32, torch.int64):
            pooled = state.clone()
            at = None if slots is None else torch.tensor(slots, device="cuda", dtype=index)
            y = step(x, g, pooled, at)
            ref = step_reference(x, g, state, range(rows) if slots is None else slots)
            assert y.dtype == dtype and R.misses(y, ref[0], ref[2]) == 0, slots
            assert R.misses(pooled, ref[1], ref[3]) == 0, slots
            untouched = sorted(set(range(pool)) - set(range(rows) if slots is None else slots))
            assert torch.equal(pooled[untouched], state[untouched])  # left as they were


@pytest.mark.gpu
def test_the_step_continues_a_sequence_and_reads_strided_rows():
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence, gated_linear_recurrence_step as step

    x, g, h0, dy, dl = make(4, 60, 96, BF16, FP32, 4, seed=11)
    _, prefill = gated_linear_recurrence(x[:, :50], g[:, :50], h0, True)
    wide = torch.full((6, 2, 96), 5.0, device="cuda")
    pool = wide[:, 1]  # slots inside a wider buffer
    slots = torch.tensor([3, 0, 5, 2], device="cuda", dtype=torch.int32)
    pool[slots.long()] = prefill
    ys = [step(x[:, t], g[:, t], pool, slots) for t in range(50, 60)]
    want = R.linear_recurrence(x.reshape(-1, 96), g.reshape(-1, 96), [60] * 4, h0)
    y, slack = (t.view(4, 60, 96)[:, 50:] for t in want["y"])
    assert R.misses(torch.stack(ys, 1), y, slack) == 0
    assert R.misses(pool[slots.long()], *want["final"]) == 0
    assert (wide[:, 0] == 5).all() and (pool[[1, 4]] == 5).all()
    heads = torch.zeros(6, 4, 24, device="cuda")
    y = step(x[:, 0].view(4, 4, 24), g[:, 0].view(4, 4, 24), heads, slots)
    assert y.shape == (4, 4, 24) and torch.equal(heads[slots.long()].to(BF16), y)
    assert step(x[:0, 0], g[:0, 0], pool).shape == (0, 96)
    with pytest.raises(ValueError, match="dense inside its slot"):
        step(x[:, 0], g[:, 0], torch.zeros(96, 6, device="cuda").t(), slots)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gdtype", [(BF16, FP32), (FP32, FP16)])
@pytest.mark.parametrize("channels", [2056, 2060])
def test_a_large_step_with_wide_and_narrow_accesses(channels, dtype, gdtype):
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence_step as step

    rows, pool = 530, 600
    x, g, _, _, _ = make(1, rows, channels, dtype, gdtype, 1, seed=16)
    state = torch.randn(pool, channels, device="cuda")
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(4))[:rows]
    order[7], order[300], order[529], order[8] = order[2], order[2], order[100], -1
    pooled = state.clone()
    y = step(x[0], g[0], pooled, order.cuda())
    ref = step_reference(x[0], g[0], state, order.tolist())
    assert R.misses(y, ref[0], ref[2]) == 0 and R.misses(pooled, ref[1], ref[3]) == 0


@pytest.mark.gpu
def test_the_step_on_a_pool_past_32_bits():
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence_step as step

    pool = torch.zeros(540_000, 4096, device="cuda")
    assert pool.numel() > 1 << 31
    x, g, _, _, _ = make(1, 3, 4096, BF16, FP32, 1, seed=15)
    slots = torch.tensor([539_999, 3, 530_001], device="cuda")
    y = step(x[0], g[0], pool, slots)
    assert torch.equal(y, x[0]) and torch.equal(pool[slots].to(BF16), x[0]) and int((pool != 0).any(1).sum()) == 3


@pytest.mark.gpu
def test_the_step_in_a_captured_graph():
    from miles_ext_kernels_b200.cake.linear_recurrence import gated_linear_recurrence_step as step

    x, g, _, _, _ = make(1, 8, 256, BF16, FP32, 1, seed=12)
    x, g = x[0], g[0]
    pool = torch.randn(20, 256, device="cuda")
    slots = torch.arange(8, device="cuda", dtype=torch.int32)
    want, reference = pool.clone(), []
    for shift in (0, 5, 12):
        reference.append(step(x, g, want, slots + shift))
    graph = torch.cuda.CUDAGraph()
    mine = pool.clone()
    with torch.cuda.graph(graph):
        y = step(x, g, mine, slots)
    for shift, ref in zip((0, 5, 12), reference):
        slots.copy_(torch.arange(8, device="cuda") + shift)
        graph.replay()
        assert torch.equal(y, ref)
    assert torch.equal(mine, want)
