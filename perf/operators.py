"""The operators of a recurrent training layer with their real sizes: what each reads, computes and writes, in plain
torch and through the package's entry points.

Three families, which one layer runs one after the other:

* ``layer_norm`` -- LayerNorm over the last dimension, forward and backward with the reduction of the weight's and the
  bias's gradients, keeping either the input or an 8-bit checkpoint of the normalised rows for the backward;
* ``gated_norm`` -- the SiLU-gated RMSNorm over rows of 128 with its two inputs kept as 8-bit checkpoints;
* ``recurrence`` -- the gated linear recurrence ``h[t] = exp(g[t]) h[t-1] + x[t]`` per channel over long or packed
  sequences, forward and backward, and ``step``, its form for single tokens on a pool of states.

``run`` computes them in elementary torch operations in 32 bits, or calls the package where ``own`` is true.  ``exact``
computes the same values in 64 bits, written apart: the statistics in one expression per definition, the recurrence
block by block instead of by doubling.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # eight sequences' next tokens through a norm of a 2,048-wide model: only latency counts
        dict(name="ln_decode", op="layer_norm", rows=8, width=2048, dtype="bf16", weight="bf16", checkpoint=False,
             backward=False),
        # a training step's 32,768 tokens of a 4,096-wide model
        dict(name="ln_train", op="layer_norm", rows=32768, width=4096, dtype="bf16", weight="bf16", checkpoint=False,
             backward=True),
        # an odd width in full precision, as a probe or a small encoder has it
        dict(name="ln_odd_fp32", op="layer_norm", rows=4099, width=1157, dtype="fp32", weight="fp32", checkpoint=False,
             backward=True),
        # a wide model's training step, the normalised rows kept in 8 bits
        dict(name="ln_8bit", op="layer_norm", rows=16384, width=8192, dtype="bf16", weight="bf16", checkpoint=True,
             backward=True),
        # the output norm of a small layer, 8-bit checkpoints, the gate inside a wider projection
        dict(name="gate_8bit_small", op="gated_norm", tokens=1031, heads=12),
        # the output norm of a training step: 32,768 tokens of 32 heads
        dict(name="gate_8bit_train", op="gated_norm", tokens=32768, heads=32),
        # a training step of a recurrent layer: 4 sequences of 8,192 tokens, 4,096 channels, FP32 gates
        dict(name="glr_train", op="recurrence", batch=4, tokens=8192, docs=0, channels=4096, dtype="bf16", gate="fp32",
             backward=True),
        # 65,536 packed tokens of 24 documents with initial and final states and gates in the model's type
        dict(name="glr_packed", op="recurrence", batch=1, tokens=65536, docs=24, channels=2048, dtype="bf16",
             gate="bf16", backward=True),
        # one long sequence on few channels: a rank's share of the channels
        dict(name="glr_long", op="recurrence", batch=1, tokens=262144, docs=0, channels=512, dtype="bf16", gate="fp32",
             backward=True),
        # a prompt's prefill, forward only, odd sizes in full precision
        dict(name="glr_odd_prefill", op="recurrence", batch=3, tokens=1031, docs=0, channels=1157, dtype="fp32",
             gate="fp32", backward=False),
        # one sequence's next token
        dict(name="step_one", op="step", rows=1, slots=64, channels=4096, dtype="bf16", gate="fp32"),
        # a full serving batch's next tokens on a pool of states
        dict(name="step_batch", op="step", rows=1024, slots=2048, channels=4096, dtype="bf16", gate="fp32"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm", "gated_norm", "recurrence", "recurrence", "step"])
    if op == "layer_norm":
        width = _log_uniform(rng, 64, 16384)
        if rng.random() < 0.6:
            width = max(64, width // 64 * 64)
        rows = _log_uniform(rng, 1, max(2, min(65536, (1 << 27) // width)))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if dtype == "fp32":
            rows = max(1, rows // 2)
        # a checkpoint's codes flip with the last bit of FP32 statistics, which FP32 parameters' gradients would show
        checkpoint = dtype != "fp32" and rng.random() < 0.4
        return dict(op=op, rows=rows, width=width, dtype=dtype, weight=dtype if checkpoint else rng.choice([dtype, "fp32"]),
                    checkpoint=checkpoint, backward=rng.random() < 0.75)
    if op == "gated_norm":
        return dict(op=op, tokens=_log_uniform(rng, 1, 32768), heads=rng.choice([1, 4, 12, 16, 24, 32]))
    if op == "recurrence":
        channels = _log_uniform(rng, 32, 8192)
        if rng.random() < 0.6:
            channels = max(32, channels // 32 * 32)
        total = _log_uniform(rng, 16, max(32, min(131072, (1 << 26) // channels)))
        docs = rng.choice([0, 0, 1, 5, 40])
        batch = 1 if docs else rng.choice([1, 2, 5])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return dict(op=op, batch=batch, tokens=max(1, total // batch), docs=docs, channels=channels, dtype=dtype,
                    gate=rng.choice(["fp32", dtype]), backward=rng.random() < 0.7)
    channels = _log_uniform(rng, 64, 8192)
    rows = _log_uniform(rng, 1, 1024)
    return dict(op=op, rows=rows, slots=rows + rng.randrange(1, 200), channels=channels,
                dtype=rng.choice(["bf16", "fp16", "fp32"]), gate=rng.choice(["fp32", "fp32", "bf16"]))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    op = case["op"]

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    def rand(*shape):
        return torch.rand(*shape, device=dev, generator=gen)

    def leaf(t):
        return t.requires_grad_(case.get("backward", True))

    s = dict(case)
    if op == "layer_norm":
        dtype, wtype, width = DTYPES[case["dtype"]], DTYPES[case["weight"]], case["width"]
        # residual-stream rows: a common offset and channels of unequal size
        s["x"] = leaf((randn(case["rows"], width) * (0.5 + rand(width)) + 0.3).to(dtype))
        s["w"] = leaf((1 + 0.2 * randn(width)).to(wtype))
        s["b"] = leaf((0.2 * randn(width)).to(wtype))
        s["dy"] = randn(case["rows"], width).to(dtype) if case["backward"] else None
    elif op == "gated_norm":
        tokens, heads = case["tokens"], case["heads"]
        s["x"] = leaf(randn(tokens, heads, 128).bfloat16())
        projection = randn(tokens, 2 * heads * 128).bfloat16()
        s["z"] = projection[:, heads * 128 :].unflatten(-1, (heads, 128)).requires_grad_()
        s["w"] = leaf((1 + 0.5 * randn(128)).bfloat16())
        s["dy"] = randn(tokens, heads, 128).bfloat16()
    else:
        channels = case["channels"]
        # decays of 1 to 1,000 tokens' memory, drawn per channel, modulated per token
        rate = torch.exp(rand(channels) * math.log(1e-3))
        if op == "recurrence":
            batch, tokens, docs = case["batch"], case["tokens"], case["docs"]
            s["x"] = leaf(randn(batch, tokens, channels).to(DTYPES[case["dtype"]]))
            gate = torch.nn.functional.softplus(randn(batch, tokens, channels))
            s["g"] = leaf(gate.mul_(rate).neg_().to(DTYPES[case["gate"]]))
            del gate
            if docs:
                cuts = torch.Generator().manual_seed(seed)
                inner = torch.randint(0, tokens + 1, (docs - 1,), generator=cuts).sort().values
                cu = torch.cat([torch.zeros(1, dtype=torch.int64), inner, torch.tensor([tokens])])
                full = (cu[1:] > cu[:-1]).nonzero().flatten()
                s["cu"] = cu.to(dev, torch.int32)
                # the documents that hold tokens, their first and last tokens
                s["full"], s["first"], s["last"] = (t.to(dev) for t in (full, cu[:-1][full], cu[1:][full] - 1))
            else:
                s["cu"] = None
                s["full"] = torch.arange(batch, device=dev)
                s["first"] = s["full"] * tokens
                s["last"] = s["first"] + tokens - 1
            sequences = docs or batch
            s["h0"] = leaf(randn(sequences, channels))
            s["dy"] = randn(batch, tokens, channels).to(DTYPES[case["dtype"]]) if case["backward"] else None
            s["dht"] = randn(sequences, channels) if case["backward"] else None
        else:
            rows, slots = case["rows"], case["slots"]
            s["x"] = randn(rows, channels).to(DTYPES[case["dtype"]])
            s["g"] = (torch.nn.functional.softplus(randn(rows, channels)) * -rate).to(DTYPES[case["gate"]])
            s["state"] = randn(slots, channels)
            s["slots_of"] = torch.randperm(slots, device=dev, generator=gen)[:rows].to(torch.int32)
    return s


def _e4m3(t):
    return t.to(torch.float8_e4m3fn).float()


def _layer_norm(s, backward, checkpoint):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    unit = centred * rstd
    y = (unit * w + b).to(s["x"].dtype)
    if not backward:
        return y
    if checkpoint:
        unit = _e4m3(unit)
    dy = s["dy"].float()
    dn = dy * w
    dx = rstd * (dn - dn.mean(-1, keepdim=True) - unit * (dn * unit).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": (dy * unit).sum(0).to(s["w"].dtype),
            "db": dy.sum(0).to(s["b"].dtype)}


def _scaled_e4m3(z):
    """Rows in e4m3 under a power of two: the smallest that brings the row's largest magnitude to at most 448."""
    mantissa, exponent = torch.frexp(z.abs().amax(-1, keepdim=True))
    exponent = (exponent - 9 + (mantissa > 0.875)).clamp(min=-126)
    return torch.ldexp(_e4m3(torch.ldexp(z, -exponent)), exponent)


def _gated_norm(s):
    x, z, w, dy = s["x"].float(), s["z"].float(), s["w"].float(), s["dy"].float()
    rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    n = x * rstd
    y = n * w * (z * torch.sigmoid(z))
    n, z = _e4m3(n), _scaled_e4m3(z)
    sig = torch.sigmoid(z)
    a = dy * z * sig
    dn = a * w
    dx = rstd * (dn - n * (dn * n).mean(-1, keepdim=True))
    dz = dy * n * w * sig * (1 + z * (1 - sig))
    dw = (a * n).sum((0, 1))
    return {"y": y.bfloat16(), "dx": dx.bfloat16(), "dz": dz.bfloat16(), "dw": dw.bfloat16()}


def _scan(a, b):
    """``h[t] = a[t] h[t-1] + b[t]`` along the first dimension by doubling: log2(T) passes, no torch operation scans."""
    step = 1
    while step < b.shape[0]:
        b = torch.cat([b[:step], torch.addcmul(b[step:], a[step:], b[:-step])])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _recurrence(s, backward):
    shape, channels = s["x"].shape, s["channels"]
    x = s["x"].float().reshape(-1, channels)
    # rounded from 64 bits: a 32-bit exponential is biased next to one, which adds up over a thousand tokens' memory
    a = torch.exp(s["g"].double().reshape(-1, channels)).float()
    h0, first, last, full = s["h0"], s["first"], s["last"], s["full"]
    into = x.index_add(0, first, a[first] * h0[full])
    h = _scan(a.index_fill(0, first, 0.0), into)
    final = h0.index_copy(0, full, h[last])
    y = h.to(s["x"].dtype).view(shape)
    if not backward:
        return {"y": y, "final": final}
    before = torch.cat([h[:1], h[:-1]]).index_copy(0, first, h0[full])
    grad = s["dy"].float().reshape(-1, channels).index_add(0, last, s["dht"][full])
    after = torch.cat([a[1:], a[:1]]).index_fill(0, last, 0.0)
    dx = _scan(after.flip(0), grad.flip(0)).flip(0)
    dg = dx * a * before
    dh0 = s["dht"].index_copy(0, full, (a * dx)[first])
    return {"y": y, "final": final, "dx": dx.to(s["x"].dtype).view(shape), "dg": dg.to(s["g"].dtype).view(shape),
            "dh0": dh0}


def _step(s):
    slots = s["slots_of"].long()
    h = torch.exp(s["g"].float()) * s["state"][slots] + s["x"].float()
    s["state"].index_copy_(0, slots, h)
    return {"y": h.to(s["x"].dtype), "state": s["state"]}


def run(s):
    op = s["op"]
    if own:
        from miles_ext_kernels_b200.cake import gated_rmsnorm, layer_norm, linear_recurrence

        if op == "layer_norm":
            y = layer_norm.layer_norm(s["x"], s["w"], s["b"], 1e-5, checkpoint="e4m3" if s["checkpoint"] else None)
            if not s["backward"]:
                return y
            dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
            return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
        if op == "gated_norm":
            y = gated_rmsnorm.rmsnorm_silu_gate(s["x"], s["z"], s["w"], 1e-6, checkpoint="e4m3")
            dx, dz, dw = torch.autograd.grad(y, (s["x"], s["z"], s["w"]), s["dy"])
            return {"y": y.detach(), "dx": dx, "dz": dz, "dw": dw}
        if op == "recurrence":
            y, final = linear_recurrence.gated_linear_recurrence(
                s["x"], s["g"], initial_state=s["h0"], output_final_state=True, cu_seqlens=s["cu"])
            if not s["backward"]:
                return {"y": y, "final": final}
            dx, dg, dh0 = torch.autograd.grad((y, final), (s["x"], s["g"], s["h0"]), (s["dy"], s["dht"]))
            return {"y": y.detach(), "final": final.detach(), "dx": dx, "dg": dg, "dh0": dh0}
        y = linear_recurrence.gated_linear_recurrence_step(s["x"], s["g"], s["state"], state_indices=s["slots_of"])
        return {"y": y, "state": s["state"]}
    with torch.no_grad():
        if op == "layer_norm":
            return _layer_norm(s, s["backward"], s["checkpoint"])
        if op == "gated_norm":
            return _gated_norm(s)
        if op == "recurrence":
            return _recurrence(s, s["backward"])
        return _step(s)


def work(case):
    """Each call's inputs read once and its outputs written once; a backward call's inputs are the incoming gradients
    and what the forward had to keep (the rows, or their 8-bit checkpoint, which the forward writes too)."""
    op = case["op"]
    if op == "layer_norm":
        n, e = case["rows"] * case["width"], BYTES[case["dtype"]]
        params = 2 * case["width"] * BYTES[case["weight"]]
        if not case["backward"]:
            return {"bytes": 2 * e * n + params, "flops": 8 * n}
        kept = 2 if case["checkpoint"] else e  # written and read again, or read again
        return {"bytes": (4 * e + kept) * n + 3 * params + 8 * case["rows"], "flops": 20 * n}
    if op == "gated_norm":
        n = case["tokens"] * case["heads"] * 128
        # x, z, y; dy, dx, dz in bf16, two checkpoints written and read
        return {"bytes": (6 * 2 + 4) * n + 10 * case["tokens"] * case["heads"], "flops": 40 * n}
    if op == "recurrence":
        n = case["batch"] * case["tokens"] * case["channels"]
        e, eg = BYTES[case["dtype"]], BYTES[case["gate"]]
        states = (case["docs"] or case["batch"]) * case["channels"] * 4
        if not case["backward"]:
            return {"bytes": (2 * e + eg) * n + 2 * states, "flops": 3 * n}
        return {"bytes": (5 * e + 3 * eg) * n + 5 * states, "flops": 11 * n}
    n = case["rows"] * case["channels"]
    return {"bytes": (2 * BYTES[case["dtype"]] + BYTES[case["gate"]] + 8) * n + 4 * case["rows"], "flops": 3 * n}


def _blocks64(a, b, block=128):
    """The recurrence in 64 bits: every block of tokens from a zero state, all blocks side by side, then the blocks'
    ends one after the other, then the state that entered each block carried through its products of decays."""
    total, channels = b.shape
    count = -(-total // block)
    pad = count * block - total
    a = torch.cat([a, a.new_ones(pad, channels)]).view(count, block, channels)
    b = torch.cat([b, b.new_zeros(pad, channels)]).view(count, block, channels)
    local, decay = torch.empty_like(b), torch.empty_like(a)
    h, p = torch.zeros_like(b[:, 0]), torch.ones_like(a[:, 0])
    for i in range(block):
        h = a[:, i] * h + b[:, i]
        p = a[:, i] * p
        local[:, i], decay[:, i] = h, p
    state = torch.zeros_like(h)
    carry = torch.zeros_like(b[0, 0])
    for j in range(count):
        state[j] = carry
        carry = decay[j, -1] * carry + local[j, -1]
    return (local + decay * state[:, None]).view(-1, channels)[:total]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    to8 = lambda t: t.float().to(torch.float8_e4m3fn).double()  # noqa: E731
    if op == "layer_norm":
        x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
        var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
        sd = (var + 1e-5).sqrt()
        unit = (x - mean) / sd
        y = unit * w + b
        del x
        if not case["backward"]:
            return y
        if case["checkpoint"]:
            unit = to8(unit)
        dy = s["dy"].double()
        dw, db = torch.einsum("rc,rc->c", dy, unit), dy.sum(0)
        dy = dy.mul_(w)
        width = case["width"]
        dx = (dy - dy.sum(-1, keepdim=True) / width - unit * (torch.einsum("rc,rc->r", dy, unit)[:, None] / width)) / sd
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if op == "gated_norm":
        x, z, w, dy = (s[k].double() for k in ("x", "z", "w", "dy"))
        rms = (x.square().sum(-1, keepdim=True) / 128 + 1e-6).sqrt()
        n = x / rms
        y = n * w * z / (1 + torch.exp(-z))
        n = to8(n)
        # the power of two: the exponent is the smallest whose multiple 448 reaches the row's largest magnitude
        power = torch.ceil(torch.log2(z.abs().amax(-1, keepdim=True).clamp(min=1e-300) / 448)).clamp(min=-126)
        z = to8(z / torch.exp2(power)) * torch.exp2(power)
        gate = 1 / (1 + torch.exp(-z))
        upstream = dy * w * (z * gate)
        dx = (upstream - n * ((upstream * n).sum(-1, keepdim=True) / 128)) / rms
        dz = dy * (n * w) * (gate + z * gate * (1 - gate))
        dw = torch.einsum("thc,thc,thc->c", dy, z * gate, n)
        return {"y": y, "dx": dx, "dz": dz, "dw": dw}
    if op == "recurrence":
        shape, channels = s["x"].shape, case["channels"]
        x = s["x"].double().view(-1, channels)
        a = s["g"].double().view(-1, channels).exp()
        h0, first, last, full = s["h0"].double(), s["first"], s["last"], s["full"]
        b = x.clone()
        b[first] += a[first] * h0[full]
        cut = a.clone()
        cut[first] = 0
        h = _blocks64(cut, b)
        final = h0.clone()
        final[full] = h[last]
        out = {"y": h.view(shape), "final": final}
        if not case["backward"]:
            return out
        del b, cut, x
        grad = s["dy"].double().view(-1, channels).clone()
        grad[last] += s["dht"].double()[full]
        cut = a.roll(-1, 0)
        cut[last] = 0
        dx = _blocks64(cut.flip(0), grad.flip(0)).flip(0)
        del cut, grad
        dh0 = s["dht"].double().clone()
        dh0[full] = a[first] * dx[first]
        before = h.roll(1, 0)
        before[first] = h0[full]
        out.update(dx=dx.view(shape), dg=(dx * a * before).view(shape), dh0=dh0)
        return out
    slots = s["slots_of"].long()
    h = s["g"].double().exp() * s["state"].double()[slots] + s["x"].double()
    state = s["state"].double()
    state[slots] = h
    return {"y": h, "state": state}
