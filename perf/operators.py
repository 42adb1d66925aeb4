"""The operators of the dense MLP site and what is measured of them.

Three families, in the order a layer runs them:

* ``layer_norm``   layer norm over the last dimension, forward (serving) and forward + backward
                   (a training step: output, input gradient, weight and bias gradients),
* ``mlp``          the dense gated feed-forward block y = (silu(x Wg^T) * (x Wu^T)) Wd^T, forward
                   and forward + backward,
* ``fp8``          the 8-bit serving form: ``quantize`` (activations per 1 x 128, weights per
                   128 x 128 block, power-of-two scales, written and read back) and ``linear`` (the
                   matrix product of two quantised operands, plain or with the gate applied to its
                   two halves).

``run`` computes a case in its plain form (elementary torch operations in 32 bits, rounded once at the
end) or, with ``own`` set, through this package's operators.
"""
import math

import torch

own = False

BLOCK = 128
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
          "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
# largest finite value of an 8-bit type: 1.75 * 2^8 and 1.75 * 2^15
TOP_EXPONENT = {"e4m3": 8, "e5m2": 15}


def listed():
    return [
        # one decoded token in front of an MLP site, fp32 residual carrier: a launch's latency
        dict(name="ln_token", op="layer_norm", rows=1, cols=768, dtype="f32", train=False),
        # a training step's norm at the small model's width, 4 x 4096 tokens
        dict(name="ln_step", op="layer_norm", rows=16384, cols=768, dtype="bf16", train=True),
        # odd token count and odd width: no row but the first is aligned
        dict(name="ln_step_odd", op="layer_norm", rows=4099, cols=2047, dtype="f16", train=True),
        # fp32 activations at the large model's width
        dict(name="ln_step_f32", op="layer_norm", rows=16384, cols=2048, dtype="f32", train=True),
        # one decoded token through an uncarved large-model layer: bound by reading its weights
        dict(name="mlp_token", op="mlp", rows=1, d_model=2048, d_ff=5632, dtype="bf16", train=False),
        # an odd prefill block of the small model
        dict(name="mlp_prefill", op="mlp", rows=333, d_model=768, d_ff=2048, dtype="f16", train=False),
        # a training step of the small model, ragged batch
        dict(name="mlp_step", op="mlp", rows=4093, d_model=768, d_ff=2048, dtype="bf16", train=True),
        # a training step of the large model
        dict(name="mlp_step_large", op="mlp", rows=8192, d_model=2048, d_ff=5632, dtype="bf16", train=True),
        # a small decode batch against the 8-bit gate/up matrix, gate applied
        dict(name="fp8_tokens", op="fp8_linear", rows=4, cols=2048, out=11264, gated=True, x="e4m3", y="bf16"),
        # ragged everything: rows, outputs and a last block of 80 columns
        dict(name="fp8_ragged", op="fp8_linear", rows=1001, cols=2000, out=3333, gated=False, x="e5m2", y="f32"),
        # a prefill block through the 8-bit gate/up matrix, gate applied
        dict(name="fp8_prefill", op="fp8_linear", rows=8192, cols=2048, out=11264, gated=True, x="e4m3", y="bf16"),
        # the hidden block of that layer quantised in front of the down projection, and read back
        dict(name="fp8_quantize", op="fp8_quantize", rows=8192, cols=5632, block_rows=1, dtype="bf16", q="e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "mlp", "fp8_linear", "fp8_linear", "fp8_quantize"])
    if op == "layer_norm":
        cols = _log(rng, 16, 8192)
        return dict(op=op, rows=_log(rng, 1, 16384 * 2048 // max(cols, 2048)), cols=cols,
                    dtype=rng.choice(["f32", "bf16", "f16"]), train=rng.random() < 0.7)
    if op == "mlp":
        return dict(op=op, rows=_log(rng, 1, 8192), d_model=16 * _log(rng, 4, 128), d_ff=16 * _log(rng, 4, 352),
                    dtype=rng.choice(["bf16", "f16"]), train=rng.random() < 0.6)
    if op == "fp8_linear":
        gated = rng.random() < 0.5
        out = 256 * _log(rng, 1, 44) if gated else _log(rng, 16, 11264)
        return dict(op=op, rows=_log(rng, 1, 8192), cols=16 * _log(rng, 4, 128), out=out, gated=gated,
                    x=rng.choice(["e4m3", "e5m2"]), y=rng.choice(["bf16", "f16", "f32"]))
    return dict(op=op, rows=_log(rng, 1, 8192), cols=16 * _log(rng, 4, 352), block_rows=rng.choice([1, 128]),
                dtype=rng.choice(["bf16", "f16", "f32"]), q=rng.choice(["e4m3", "e5m2"]))


# ---- inputs ---------------------------------------------------------------------------------

def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _activations(gen, rows, cols):
    """Residual-stream like rows: normal with a spread of row magnitudes, a few large channels."""
    chan = torch.exp(0.5 * _randn(gen, cols))
    return _randn(gen, rows, cols) * chan * torch.exp(0.3 * _randn(gen, rows, 1))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    st = {"case": dict(case)}
    if case["op"] == "layer_norm":
        dt = DTYPES[case["dtype"]]
        rows, cols = case["rows"], case["cols"]
        st["x"] = (_activations(gen, rows, cols) + 0.2).to(dt)
        st["weight"] = 1.0 + 0.1 * _randn(gen, cols)
        st["bias"] = 0.1 * _randn(gen, cols)
        if case["train"]:
            st["dy"] = _randn(gen, rows, cols).to(dt)
            for k in ("x", "weight", "bias"):
                st[k].requires_grad_(True)
    elif case["op"] == "mlp":
        dt = DTYPES[case["dtype"]]
        d, f = case["d_model"], case["d_ff"]
        st["x"] = _randn(gen, case["rows"], d).to(dt)
        st["gate_up"] = (_randn(gen, 2 * f, d) * d ** -0.5).to(dt)
        st["down"] = (_randn(gen, d, f) * f ** -0.5).to(dt)
        if case["train"]:
            st["dy"] = _randn(gen, case["rows"], d).to(dt)
            for k in ("x", "gate_up", "down"):
                st[k].requires_grad_(True)
    elif case["op"] == "fp8_linear":
        nb = -(-case["cols"] // BLOCK)
        qx, qw = DTYPES[case["x"]], torch.float8_e4m3fn
        lift = 2.0 ** (TOP_EXPONENT[case["x"]] - 3)       # blocks fill their type's range up to their largest value
        st["x"] = (_randn(gen, case["rows"], case["cols"]) * lift).clamp(-7 * lift, 7 * lift).to(qx)
        st["x_scale"] = torch.exp2(torch.round(_randn(gen, case["rows"], nb))) / lift
        st["w"] = (_randn(gen, case["out"], case["cols"]) * 32).clamp(-224, 224).to(qw)
        # scales that another program chose: not powers of two
        st["w_scale"] = torch.exp(0.3 * _randn(gen, -(-case["out"] // BLOCK), nb)) / 32 * case["cols"] ** -0.5
        if own:
            import mortar_b200 as mb
            st["matrix"] = mb.Fp8Matrix(st["w"], st["w_scale"])
    else:
        st["x"] = _activations(gen, case["rows"], case["cols"]).to(DTYPES[case["dtype"]])
    return st


# ---- one pass -------------------------------------------------------------------------------

def _run_own(st):
    import mortar_b200 as mb
    case = st["case"]
    if case["op"] == "layer_norm":
        y = mb.ops.layer_norm(st["x"], st["weight"], st["bias"], eps=1e-5)
        if not case["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["dy"]))
    if case["op"] == "mlp":
        y = mb.ops.mlp_dense(st["x"], st["gate_up"], st["down"])
        if not case["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (st["x"], st["gate_up"], st["down"]), st["dy"]))
    if case["op"] == "fp8_linear":
        return mb.ops.linear_fp8(st["x"], st["matrix"], x_scale=st["x_scale"], swiglu=case["gated"],
                                 out_dtype=DTYPES[case["y"]])
    q, scale = mb.ops.quantize_fp8(st["x"], block_rows=case["block_rows"], dtype=DTYPES[case["q"]])
    return mb.ops.dequantize_fp8(q, scale, out_dtype=st["x"].dtype), scale


def _plain_layer_norm(st):
    x, w, b = st["x"].detach().float(), st["weight"].detach(), st["bias"].detach()
    dt, cols = st["x"].dtype, st["x"].shape[1]
    mean = x.sum(1, keepdim=True) / cols
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).sum(1, keepdim=True) / cols + 1e-5)
    xh = xc * rstd
    y = (xh * w + b).to(dt)
    if not st["case"]["train"]:
        return y
    dy = st["dy"].float()
    g = dy * w
    c1 = g.sum(1, keepdim=True) / cols
    c2 = (g * xh).sum(1, keepdim=True) / cols
    dx = ((g - c1 - xh * c2) * rstd).to(dt)
    return y, dx, (dy * xh).sum(0), dy.sum(0)


def _plain_mlp(st):
    dt = st["x"].dtype
    x, wgu, wd = (st[k].detach().float() for k in ("x", "gate_up", "down"))
    f = wd.shape[1]
    gu = x @ wgu.t()
    g, u = gu[:, :f], gu[:, f:]
    s = 1.0 / (1.0 + torch.exp(-g))
    a = g * s
    h = a * u
    y = (h @ wd.t()).to(dt)
    if not st["case"]["train"]:
        return y
    dy = st["dy"].float()
    dh = dy @ wd
    dgu = torch.cat([dh * u * (s + a * (1.0 - s)), dh * a], dim=1)
    return y, (dgu @ wgu).to(dt), (dgu.t() @ x).to(dt), (dy.t() @ h).to(dt)


def _plain_fp8_linear(st):
    case = st["case"]
    cols, out = case["cols"], case["out"]
    sx = st["x_scale"].repeat_interleave(BLOCK, 1)[:, :cols]
    sw = st["w_scale"].repeat_interleave(BLOCK, 0)[:out].repeat_interleave(BLOCK, 1)[:, :cols]
    y = (st["x"].float() * sx) @ (st["w"].float() * sw).t()
    if case["gated"]:
        g, u = y[:, :out // 2], y[:, out // 2:]
        y = g / (1.0 + torch.exp(-g)) * u
    return y.to(DTYPES[case["y"]])


def _plain_fp8_quantize(st):
    case = st["case"]
    x = st["x"].float()
    rows, cols = x.shape
    br, nb = case["block_rows"], -(-cols // BLOCK)
    rb = -(-rows // br)
    padded = torch.zeros(rb * br, nb * BLOCK, device=x.device)
    padded[:rows, :cols] = x
    tiles = padded.reshape(rb, br, nb, BLOCK)
    amax = tiles.abs().amax(dim=(1, 3))
    # the smallest power of two that brings the block into the type's range (1.75 * 2^top at most)
    mant, expo = torch.frexp(amax)                         # amax = mant * 2^expo, mant in [0.5, 1)
    e = expo - 1 - TOP_EXPONENT[case["q"]] + (mant > 0.875).int()
    e = torch.where(amax > 0, e, torch.zeros_like(e)).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(amax), e)
    q = torch.ldexp(tiles, -e[:, None, :, None]).to(DTYPES[case["q"]])
    back = torch.ldexp(q.float(), e[:, None, :, None]).reshape(rb * br, nb * BLOCK)[:rows, :cols]
    return back.to(st["x"].dtype), scale


_PLAIN = {"layer_norm": _plain_layer_norm, "mlp": _plain_mlp, "fp8_linear": _plain_fp8_linear,
          "fp8_quantize": _plain_fp8_quantize}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------

def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "e5m2": 1}
    if case["op"] == "layer_norm":
        n, e = case["rows"] * case["cols"], size[case["dtype"]]
        if case["train"]:       # x, dy in; y, dx out; weight, bias in, their gradients out; all fp32 but the rows
            return {"bytes": 4 * n * e + 16 * case["cols"], "flops": 20 * n}
        return {"bytes": 2 * n * e + 8 * case["cols"], "flops": 8 * n}
    if case["op"] == "mlp":
        m, d, f, e = case["rows"], case["d_model"], case["d_ff"], size[case["dtype"]]
        if case["train"]:
            return {"bytes": (4 * m * d + 6 * d * f) * e, "flops": 18 * m * d * f}
        return {"bytes": (2 * m * d + 3 * d * f) * e, "flops": 6 * m * d * f}
    if case["op"] == "fp8_linear":
        m, k, n = case["rows"], case["cols"], case["out"]
        nb = -(-k // BLOCK)
        n_out = n // 2 if case["gated"] else n
        return {"bytes": m * k + n * k + 4 * nb * (m + -(-n // BLOCK)) + m * n_out * size[case["y"]],
                "flops": 2 * m * n * k}
    m, k = case["rows"], case["cols"]
    blocks = -(-m // case["block_rows"]) * -(-k // BLOCK)
    # x read, its 8-bit values written, read again and written as the numbers that they stand for
    return {"bytes": m * k * (2 * size[case["dtype"]] + 2) + 8 * blocks, "flops": 4 * m * k}


# ---- the definition in 64 bits --------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "layer_norm":
        x, w, b = (st[k].detach().double().requires_grad_(case["train"]) for k in ("x", "weight", "bias"))
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + 1e-5) * w + b
        if not case["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), st["dy"].double()))
    if case["op"] == "mlp":
        x, wgu, wd = (st[k].detach().double().requires_grad_(case["train"]) for k in ("x", "gate_up", "down"))
        wg, wu = wgu.chunk(2, dim=0)
        gate = torch.einsum("md,fd->mf", x, wg)
        hidden = gate * torch.sigmoid(gate) * torch.einsum("md,fd->mf", x, wu)
        y = torch.einsum("mf,df->md", hidden, wd)
        if not case["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (x, wgu, wd), st["dy"].double()))
    if case["op"] == "fp8_linear":
        m, n, k = case["rows"], case["out"], case["cols"]
        acc = torch.zeros(m, n, device="cuda", dtype=torch.float64)
        row_block = torch.arange(n, device="cuda") // BLOCK
        for b in range(-(-k // BLOCK)):
            part = st["x"][:, b * BLOCK:(b + 1) * BLOCK].double() @ st["w"][:, b * BLOCK:(b + 1) * BLOCK].double().t()
            acc += part * st["x_scale"][:, b:b + 1].double() * st["w_scale"][row_block, b].double()[None, :]
        if case["gated"]:
            gate, up = acc.chunk(2, dim=1)
            acc = gate * torch.sigmoid(gate) * up
        return acc
    x = st["x"].double()
    rows, cols = x.shape
    br, rb, nb = case["block_rows"], -(-rows // case["block_rows"]), -(-cols // BLOCK)
    top = 1.75 * 2.0 ** TOP_EXPONENT[case["q"]]
    amax = torch.zeros(rb, nb, device="cuda", dtype=torch.float64)
    for b in range(nb):
        a = x[:, b * BLOCK:(b + 1) * BLOCK].abs().amax(1)
        amax[:, b] = torch.nn.functional.pad(a, (0, rb * br - rows)).reshape(rb, br).amax(1)
    scale = torch.where(amax > 0, torch.exp2(torch.ceil(torch.log2(amax / top))), torch.ones_like(amax))
    scale = torch.where(amax > scale * top, 2 * scale, scale)              # log2 is rounded: settle the border
    scale = torch.where((amax > 0) & (amax <= scale / 2 * top), scale / 2, scale).clamp(min=2.0 ** -126)
    per_row = scale.repeat_interleave(br, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    v = x / per_row
    # the nearest value of the 8-bit type, ties to even: a step is 2^(exponent - mantissa bits)
    bits, low = (3, -6) if case["q"] == "e4m3" else (2, -14)
    expo = (torch.frexp(v)[1] - 1).clamp(min=low)
    step = torch.ldexp(torch.ones_like(v), expo - bits)
    return torch.round(v / step) * step * per_row, scale
