"""The dense MLP site on the GPU against plain 64-bit implementations.

Tolerances are bounds, derived from the roundings the kernels make.  u = eps / 2 of the result's type is
the error of one rounding relative to the value; f = 2^-24 is that of one fp32 operation, and a sum of n
fp32 terms taken in parts of at most p terms and then over the parts is off by at most
(p + n / p + 1) f times the sum of the terms' magnitudes."""
import pytest
import torch

import mortar_b200 as mb

pytestmark = pytest.mark.gpu
ops = mb.ops
F = 2.0 ** -24
DEV = "cuda"
FLOATS = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def rand(*shape, seed=0, scale=1.0, dt=torch.float32):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dt)


def within(got, ref, bound, what=""):
    half = got.dtype == torch.float16
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    over = (got - ref).abs() - bound
    if half:
        # fp16 ends at 65504: from 65520 on, half a step further, a value rounds to infinity, and one whose bound reaches
        # over that border may
        inf = torch.isinf(got)
        assert bool((inf | (ref.abs() - bound < 65520)).all()) and bool((~inf | (ref.abs() + bound >= 65520)).all()), what
        assert torch.equal(got[inf].sign(), ref[inf].sign()), what
        over[inf] = 0
    assert not torch.isnan(got).any() and bool((over <= 0).all()), \
        f"{what}: off by {float((got - ref).abs().max()):.3e}, {float(over.max()):.3e} over its bound"


def errors_are_clear():
    assert ops.dense_error() == 0 and ops.linear_fp8_error() == 0


# ---- layer norm -------------------------------------------------------------------------------

def ln_ref(x, w, b, eps, dy=None):
    x = x.double()
    w = torch.ones(x.shape[-1], device=DEV, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    y = xh * w + b
    if dy is None:
        return y, xh, rstd, mean
    dy = dy.double()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return y, xh, rstd, mean, dx, dy * xh, dy


def ln_bounds(x, w, b, y, xh, rstd, dx, dy, dt):
    """Bounds on y and dx.  With c = log-depth and per-thread terms of a row's sums (<= cols / 16 + 32
    additions whatever the split), the mean is off by c f mean|x|, so xh by rstd times that, plus a few f of
    |xh|, plus what rstd is off relatively ((c + 8) f of the variance, half of it)."""
    cols = x.shape[-1]
    c = cols / 16 + 32
    x, wa = x.double(), (torch.ones(cols, device=DEV, dtype=torch.float64) if w is None else w.double().abs())
    dxh = F * (c * rstd * x.abs().mean(-1, keepdim=True) + (c + 16) * xh.abs() + 4 * rstd * x.abs())
    u = half_step(dt) * 1.01
    by = u * y.abs() + dxh * wa + 4 * F * ((xh * wa).abs() + y.abs())
    if dt == torch.float16:
        by = by + 2.0 ** -25                                   # half the smallest subnormal step
    if dy is None:
        return by, None
    g = (dy.double() * wa).abs()
    m1, m2 = g.mean(-1, keepdim=True), (g * xh.abs()).mean(-1, keepdim=True)
    bdx = u * dx.abs() + rstd * (F * (c + 16) * (g + m1 + xh.abs() * m2) + dxh * m2 +
                                 xh.abs() * (g * dxh).mean(-1, keepdim=True)) * 1.01
    if dt == torch.float16:
        bdx = bdx + 2.0 ** -25
    return by, bdx


LN_SHAPES = [(1, 1), (1, 768), (3, 5), (7, 64), (130, 768), (257, 1000), (33, 2047), (64, 2048), (5, 4096), (9, 8191),
             (3, 20011), (700, 16), (2049, 33)]


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("rows,cols", LN_SHAPES)
def test_layer_norm_and_its_gradients(rows, cols, dt):
    x = (rand(rows, cols, seed=1, scale=2.0) + 0.5).to(dt).requires_grad_()
    w = (1 + rand(cols, seed=2, scale=0.2)).requires_grad_()
    b = rand(cols, seed=3, scale=0.2).requires_grad_()
    dy = rand(rows, cols, seed=4, dt=dt)
    y = ops.layer_norm(x, w, b, 1e-5)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    ry, xh, rstd, _, rdx, tw, tb = ln_ref(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    by, bdx = ln_bounds(x.detach(), w.detach(), b.detach(), ry, xh, rstd, rdx, dy, dt)
    assert y.dtype == dt and dx.dtype == dt and dw.dtype == torch.float32
    within(y.detach(), ry, by, "y")
    within(dx, rdx, bdx, "dx")
    # sums over the rows: terms off by (cols / 16 + 48) f like xh, added in parts
    n = rows / 8 + 320
    xerr = F * ((cols / 16 + 48) * (xh.abs() + rstd * x.detach().double().abs().mean(-1, keepdim=True)))
    within(dw, tw.sum(0), F * n * tw.abs().sum(0) + (dy.double().abs() * xerr).sum(0) + 1e-30, "dw")
    within(db, tb.sum(0), F * n * tb.abs().sum(0) + 1e-30, "db")
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b, 1e-5), y)
    again = torch.autograd.grad(ops.layer_norm(x, w, b, 1e-5), (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db)))


def test_layer_norm_gradient_against_differences():
    """<dx, v> from the kernel against (loss(x + h v) - loss(x - h v)) / 2h of the 64-bit formula, whose own
    error at h = 1e-4 is below 1e-6 of the terms."""
    x, w, b = rand(11, 96, seed=5).requires_grad_(), (1 + rand(96, seed=6, scale=0.3)).requires_grad_(), rand(96, seed=7).requires_grad_()
    dy = rand(11, 96, seed=8)
    grads = torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), dy)
    loss = lambda *a: float((ln_ref(*a, 1e-5)[0] * dy.double()).sum())
    args = [t.detach().double() for t in (x, w, b)]
    for i, gr in enumerate(grads):
        v = rand(*args[i].shape, seed=20 + i).double()
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + 1e-4 * v, args[i] - 1e-4 * v
        num = (loss(*hi) - loss(*lo)) / 2e-4
        assert abs(float((gr.double() * v).sum()) - num) <= 1e-5 * float((gr.double() * v).abs().sum())


@pytest.mark.parametrize("dt", FLOATS)
def test_layer_norm_strided_offset_and_typed_inputs(dt):
    """Rows of a wider tensor, starting off 16 bytes; weight of the rows' type; no weight, no bias; a
    gradient that is broadcast (stride 0)."""
    base = rand(40, 300, seed=9, dt=dt)
    for off in (0, 1, 3, 8):
        x = base[:, off:off + 200]
        ry, xh, rstd, _ = ln_ref(x, None, None, 1e-5)
        by, _ = ln_bounds(x, None, None, ry, xh, rstd, None, None, dt)
        within(ops.layer_norm(x), ry, by, f"offset {off}")
    x = rand(2, 3, 64, seed=10, dt=dt).transpose(0, 1)
    ry, xh, rstd, _ = ln_ref(x, None, None, 1e-5)
    within(ops.layer_norm(x), ry, ln_bounds(x, None, None, ry, xh, rstd, None, None, dt)[0], "transposed")
    x = rand(6, 64, seed=11, dt=dt).requires_grad_()
    w = rand(64, seed=12, dt=dt).requires_grad_()
    dx, dw = torch.autograd.grad(ops.layer_norm(x, w).sum(), (x, w))
    assert dw.dtype == dt
    dy = torch.ones(6, 64, device=DEV, dtype=dt)
    ry, xh, rstd, _, rdx, tw, _ = ln_ref(x.detach(), w.detach(), None, 1e-5, dy)
    within(dx, rdx, ln_bounds(x.detach(), w.detach(), None, ry, xh, rstd, rdx, dy, dt)[1], "dx")
    assert ops.layer_norm(rand(0, 64, dt=dt)).shape == (0, 64)


def test_layer_norm_edges():
    # no rows: gradients of weight and bias are zeros
    x = rand(0, 64).requires_grad_()
    w, b = rand(64).requires_grad_(), rand(64).requires_grad_()
    dx, dw, db = torch.autograd.grad(ops.layer_norm(x, w, b).sum(), (x, w, b))
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    # a constant row has variance 0: y = bias; a far offset keeps the variance (two passes over the row)
    y = ops.layer_norm(torch.full((2, 48), 7.0, device=DEV), None, w.detach()[:48].contiguous())
    within(y, w.detach()[:48].expand(2, 48), 1e-6, "constant row")
    x = rand(4, 512, seed=13) + 4096.0
    ry, xh, rstd, _ = ln_ref(x, None, None, 1e-5)
    within(ops.layer_norm(x), ry, ln_bounds(x, None, None, ry, xh, rstd, None, None, torch.float32)[0], "offset row")
    # a NaN or an infinity stays in its row
    x = rand(3, 64, seed=14)
    clean = ops.layer_norm(x)
    x[1, 5] = float("inf")
    y = ops.layer_norm(x)
    assert torch.isnan(y[1]).any() and torch.equal(y[0], clean[0]) and torch.equal(y[2], clean[2])


# ---- the dense block ------------------------------------------------------------------------

def mlp_ref(x, gu, dn):
    x, gu, dn = x.double(), gu.double(), dn.double()
    f = dn.shape[1]
    s = x @ gu.t()
    g, u = s[:, :f], s[:, f:]
    sig = torch.sigmoid(g)
    return g, u, sig, g * sig * u, (g * sig * u) @ dn.t()


def mlp_grads_ref(dy, x, gu, dn):
    g, u, sig, h, y = mlp_ref(x, gu, dn)
    dy, x, gu, dn = dy.double(), x.double(), gu.double(), dn.double()
    dh = dy @ dn
    dg, du = dh * u * (sig + g * sig * (1 - sig)), dh * g * sig
    ds = torch.cat([dg, du], 1)
    return y, ds @ gu, ds.t() @ x, dy.t() @ h, (g, u, sig, h, dh, dg, du)


def mlp_bounds(dy, x, gu, dn, parts, dt):
    """Elementwise bounds.  The tensor cores add n products in fp32: at most n f of the magnitudes' sum.
    g and u are off by e_g, e_u from that (and kept in fp32); h = g sig(g) u moves by at most
    1.1 |u| e_g + |silu(g)| e_u (|silu'| <= 1.1) plus a rounding; dg by |dh| (|silu''| <= 0.5) etc."""
    g, u, sig, h, dh, dg, du = parts
    xa, gua, dna, dya = x.double().abs(), gu.double().abs(), dn.double().abs(), dy.double().abs()
    d, f, m = x.shape[1], dn.shape[1], x.shape[0]
    us = half_step(dt) * 1.01
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    es = F * (d + 2) * (xa @ gua.t())
    eg, eu = es[:, :f], es[:, f:]
    a, da = (g * sig).abs(), 1.1
    eh = us * h.abs() + 1.02 * (da * u.abs() * eg + a * eu) + 64 * F * h.abs() + tiny
    y = h @ dn.double().t()
    by = us * y.abs() + 1.01 * (eh @ dna.t()) + F * (f + 2) * (h.abs() @ dna.t()) + tiny
    kg, ku = eg, eu
    edh = F * (d + 2) * (dya @ dna)
    edg = us * dg.abs() + 1.02 * (edh * u.abs() * da + dh.abs() * (da * ku + 0.51 * u.abs() * kg)) + 64 * F * (dh * u).abs() + tiny
    edu = us * du.abs() + 1.02 * (edh * a + dh.abs() * da * kg) + 64 * F * du.abs() + tiny
    eds, ds = torch.cat([edg, edu], 1), torch.cat([dg, du], 1)
    dx, dgu, ddn = ds @ gu.double(), ds.t() @ x.double(), dy.double().t() @ h
    bdx = us * dx.abs() + 1.01 * (eds @ gua) + F * (2 * f + 2) * (ds.abs() @ gua) + tiny
    bdgu = us * dgu.abs() + 1.01 * (eds.t() @ xa) + F * (m + 2) * (ds.abs().t() @ xa) + tiny
    bddn = us * ddn.abs() + 1.01 * (dya.t() @ eh) + F * (m + 2) * (dya.t() @ h.abs()) + tiny
    return by, bdx, bdgu, bddn


def close_in_norm(got, ref, dt, roundings, what):
    """Independent roundings of relative size u each add up in squares: the whole result is off by at most
    u sqrt(roundings) of its norm (the elementwise bounds above allow every error the same sign)."""
    err = float((got.double() - ref).norm() / ref.norm().clamp(min=1e-300))
    assert err <= half_step(dt) * roundings ** 0.5, f"{what}: {err:.2e} of the norm"


MLP_SHAPES = [(1, 16, 16), (1, 768, 2048), (2, 64, 48), (5, 256, 512), (16, 80, 144), (17, 112, 272), (33, 144, 400),
              (64, 768, 2048), (127, 256, 512), (128, 256, 512), (129, 336, 528), (300, 528, 784), (1000, 272, 1040),
              (2049, 128, 256)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,d,f", MLP_SHAPES)
def test_mlp_dense_and_its_gradients(rows, d, f, dt):
    x = rand(rows, d, seed=1, dt=dt).requires_grad_()
    gu = rand(2 * f, d, seed=2, scale=d ** -0.5, dt=dt).requires_grad_()
    dn = rand(d, f, seed=3, scale=f ** -0.5, dt=dt).requires_grad_()
    dy = rand(rows, d, seed=4, dt=dt)
    y = ops.mlp_dense(x, gu, dn)
    grads = torch.autograd.grad(y, (x, gu, dn), dy)
    errors_are_clear()
    X, G, D = x.detach(), gu.detach(), dn.detach()
    *refs, parts = mlp_grads_ref(dy, X, G, D)
    bounds = mlp_bounds(dy, X, G, D, parts, dt)
    for name, got, ref, bound, n in zip(("y", "dx", "dgate_up", "ddown"), (y.detach(), *grads), refs, bounds,
                                        (2, 2, 2, 2)):
        assert got.dtype == dt
        within(got, ref, bound, name)
        if ref.numel() > 200:
            close_in_norm(got, ref, dt, n, name)
    with torch.no_grad():
        within(ops.mlp_dense(x, gu, dn), refs[0], bounds[0], "y without gradients")
    again = torch.autograd.grad(ops.mlp_dense(x, gu, dn), (x, gu, dn), dy)
    assert all(torch.equal(p, q) for p, q in zip(again, grads))
    # one gradient at a time gives the same values
    for i, t in enumerate((x, gu, dn)):
        only = torch.autograd.grad(ops.mlp_dense(*(s if j == i else s.detach() for j, s in enumerate((x, gu, dn)))), t, dy)
        within(only[0], refs[1 + i], bounds[1 + i], "alone")


@pytest.mark.parametrize("rows", [1, 2, 8, 9, 15, 16, 24, 31, 32, 40, 63, 65])
def test_mlp_dense_every_small_batch(rows):
    dt, d, f = torch.bfloat16, 208, 336
    x, gu, dn = rand(rows, d, seed=1, dt=dt), rand(2 * f, d, seed=2, scale=d ** -0.5, dt=dt), rand(d, f, seed=3, scale=f ** -0.5, dt=dt)
    dy = rand(rows, d, seed=4, dt=dt)
    *refs, parts = mlp_grads_ref(dy, x, gu, dn)
    within(ops.mlp_dense(x, gu, dn), refs[0], mlp_bounds(dy, x, gu, dn, parts, dt)[0], "y")
    errors_are_clear()


def test_mlp_dense_gradient_against_differences():
    """<grad, v> against central differences of the 64-bit formula (h = 1e-4: error below 1e-6 of the terms);
    the gradient itself is off by at most its norm bound, 2 u of the norm, which bounds <grad - ref, v>."""
    dt, rows, d, f = torch.float16, 24, 64, 96
    ts = [rand(rows, d, seed=1, dt=dt), rand(2 * f, d, seed=2, scale=0.2, dt=dt), rand(d, f, seed=3, scale=0.2, dt=dt)]
    dy = rand(rows, d, seed=4, dt=dt)
    leaves = [t.clone().requires_grad_() for t in ts]
    grads = torch.autograd.grad(ops.mlp_dense(*leaves), leaves, dy)
    loss = lambda a: float((mlp_ref(*a)[-1] * dy.double()).sum())
    for i, gr in enumerate(grads):
        v = rand(*ts[i].shape, seed=30 + i).double()
        hi, lo = [t.double() for t in ts], [t.double() for t in ts]
        hi[i], lo[i] = hi[i] + 1e-4 * v, lo[i] - 1e-4 * v
        num = (loss(hi) - loss(lo)) / 2e-4
        tol = 2 * half_step(dt) * float(gr.double().norm() * v.norm()) + 1e-6 * float((gr.double() * v).abs().sum())
        assert abs(float((gr.double() * v).sum()) - num) <= tol


def test_mlp_dense_strides_empty_and_3d():
    dt, d, f = torch.bfloat16, 96, 160
    big = rand(40, 2 * d + 8, seed=1, dt=dt)
    gu_big, dn = rand(2 * f, d + 16, seed=2, scale=d ** -0.5, dt=dt), rand(f, d, seed=3, scale=f ** -0.5, dt=dt).t()
    for off in (0, 8, 3):
        x, gu = big[:, off:off + d], gu_big[:, off:off + d]
        refs = mlp_ref(x, gu, dn)
        *_, parts = mlp_grads_ref(x, x, gu, dn)
        by = mlp_bounds(x, x, gu, dn, parts, dt)[0]
        within(ops.mlp_dense(x, gu, dn), refs[-1], by, f"offset {off}")
        within(ops.mlp_dense(x.reshape(2, 20, d), gu, dn).reshape(40, d), refs[-1], by, "3d")
    x = torch.empty(0, d, device=DEV, dtype=dt).requires_grad_()
    gu, dn = gu_big[:, :d].contiguous().requires_grad_(), dn.contiguous().requires_grad_()
    dx, dgu, ddn = torch.autograd.grad(ops.mlp_dense(x, gu, dn).sum(), (x, gu, dn))
    assert dx.shape == (0, d) and not dgu.any() and not ddn.any()


@pytest.mark.parametrize("rows", [1, 40, 200])
def test_mlp_dense_keeps_a_bad_row_to_itself(rows):
    """A NaN or infinity in one token reaches that token's output only; extreme gates saturate."""
    dt, d, f = torch.bfloat16, 64, 128
    x, gu, dn = rand(rows + 1, d, seed=1, dt=dt), rand(2 * f, d, seed=2, scale=0.2, dt=dt), rand(d, f, seed=3, scale=0.2, dt=dt)
    clean = ops.mlp_dense(x, gu, dn)
    x[rows, 3] = float("nan")
    y = ops.mlp_dense(x, gu, dn)
    assert torch.isnan(y[rows]).all() and torch.equal(y[:rows], clean[:rows])
    x = torch.full((rows, d), 30.0, device=DEV, dtype=dt)
    ref = mlp_ref(x, gu, dn)
    y = ops.mlp_dense(x, gu, dn).double()
    assert not torch.isnan(y).any()
    assert float((y - ref[-1]).norm() / ref[-1].norm()) <= 2 * half_step(dt)


# ---- 8-bit floating point ---------------------------------------------------------------------

def fp8_ref(x, block_rows, dtype):
    """Scales and dequantised values by definition, in 64 bits."""
    top = torch.finfo(dtype).max
    rows, cols = x.shape
    rb, nb = -(-rows // block_rows), -(-cols // 128)
    pad = torch.zeros(rb * block_rows, nb * 128, device=x.device, dtype=torch.float64)
    pad[:rows, :cols] = x.double()
    t = pad.reshape(rb, block_rows, nb, 128)
    amax = t.abs().amax((1, 3))
    e = torch.arange(-126, 128, device=x.device, dtype=torch.float64)
    scales = torch.exp2(e)                                                   # every candidate, smallest first
    fits = amax[..., None] <= scales * top
    scale = scales[fits.int().argmax(-1)]
    scale = torch.where(amax == 0, torch.ones_like(scale), scale)
    scale = torch.where(torch.isfinite(amax), scale, torch.full_like(scale, float("nan")))
    q = (t / scale[:, None, :, None]).float().to(dtype)                      # exact quotient, one rounding
    return scale, q.reshape(rb * block_rows, nb * 128)[:rows, :cols]


def same(a, b):
    """Equal values, NaN where the other has NaN."""
    a, b = a.double(), b.double()
    return a.shape == b.shape and bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("rows,cols,block_rows", [(1, 16, 1), (3, 144, 1), (129, 768, 1), (1000, 2000, 1), (1, 16, 128),
                                                  (128, 128, 128), (129, 144, 128), (333, 2000, 128)])
def test_quantize_fp8_is_exact(rows, cols, block_rows, dt, dtype):
    x = rand(rows, cols, seed=1) * torch.exp2(rand(rows, cols, seed=2).mul(3).round())
    x[:, : cols // 3] *= 448.0
    x = x.to(dt)
    q, s = ops.quantize_fp8(x, block_rows=block_rows, dtype=dtype)
    rs, rq = fp8_ref(x, block_rows, dtype)
    assert same(s, rs) and same(q, rq)                                       # fp16 inputs overflow to infinities: NaN blocks
    back = ops.dequantize_fp8(q, s, out_dtype=torch.float32)
    per = rs.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    assert same(back, rq.double() * per)
    for out in (torch.bfloat16, torch.float16):
        assert same(ops.dequantize_fp8(q, s, out_dtype=out), (rq.double() * per).float().to(out))


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_fp8_borders(block_rows, dtype):
    """Largest value exactly at a power of two times the type's largest, one step above it, ties, zeros,
    subnormal blocks, infinities and NaN."""
    top = torch.finfo(dtype).max
    n = 9 * block_rows
    x = rand(n, 256, seed=3, scale=0.01)
    rows = torch.arange(0, n, block_rows)
    x[:] = 0
    x[rows[0], 0] = top * 4
    x[rows[1], 0] = torch.nextafter(torch.tensor(top * 4), torch.tensor(float("inf")))
    x[rows[2], :16] = torch.tensor([top] + [1.0 + i / 32 for i in range(15)])            # ties of e4m3 and e5m2 at scale 1
    x[rows[3], 0] = 1e-42                                                                # a subnormal number
    x[rows[4], 3] = float("inf")
    x[rows[5], 130] = float("nan")
    x[rows[6], 7] = -top * 2.0 ** -100
    x[rows[7], 7] = 3.0e38
    q, s = ops.quantize_fp8(x, block_rows=block_rows, dtype=dtype)
    assert torch.isnan(s[4, 0]) and torch.isnan(s[5, 1]) and not torch.isnan(s[4, 1]) and not torch.isnan(s[5, 0])
    ok = torch.ones(9, dtype=torch.bool)
    ok[4] = ok[5] = False
    rs, rq = fp8_ref(x, block_rows, dtype)
    assert torch.equal(s.double()[ok], rs[ok])
    keep = ok.repeat_interleave(block_rows)
    assert torch.equal(q.float()[keep], rq.float()[keep])
    back = ops.dequantize_fp8(q, s, out_dtype=torch.float32)
    assert torch.isnan(back[4 * block_rows:5 * block_rows, :128]).all()


def test_quantize_fp8_strided_and_empty():
    base = rand(37, 400, seed=4, dt=torch.bfloat16)
    for off in (0, 1, 8):
        x = base[:, off:off + 272]
        q, s = ops.quantize_fp8(x)
        rs, rq = fp8_ref(x, 1, torch.float8_e4m3fn)
        assert torch.equal(s.double(), rs) and torch.equal(q.float(), rq.float())
    q, s = ops.quantize_fp8(base[:0, :272], block_rows=128)
    assert q.shape == (0, 272) and s.shape == (0, 3)
    assert ops.dequantize_fp8(q, s).shape == (0, 272)


def fp8_operands(rows, out, cols, xt, wt, seed=0):
    nb = -(-cols // 128)
    x = rand(rows, cols, seed=seed + 1, scale=20).to(xt)
    w = rand(out, cols, seed=seed + 2, scale=20).to(wt)
    xs = torch.exp(rand(rows, nb, seed=seed + 3)) / 20
    ws = torch.exp(rand(-(-out // 128), nb, seed=seed + 4)) / 20 * cols ** -0.5
    return x, xs, w, ws


def fp8_linear_ref(x, xs, w, ws):
    cols, out = x.shape[1], w.shape[0]
    xd = x.double() * xs.double().repeat_interleave(128, 1)[:, :cols]
    wd = w.double() * ws.double().repeat_interleave(128, 0)[:out].repeat_interleave(128, 1)[:, :cols]
    return xd @ wd.t(), xd.abs() @ wd.abs().t()


def fp8_bound(ref, mag, cols, out_dtype):
    """128 products a block added in fp32 (128 f), scaled (3 f) and added over the blocks."""
    return half_step(out_dtype) * 1.01 * ref.abs() + F * (128 + 3 + -(-cols // 128)) * mag + \
        (2.0 ** -25 if out_dtype == torch.float16 else 0.0)


FP8_SHAPES = [(1, 16, 16), (1, 3333, 2000), (3, 256, 128), (4, 512, 768), (8, 300, 144), (16, 1000, 400), (17, 128, 2000),
              (33, 129, 80), (64, 384, 272), (130, 640, 1024), (257, 515, 656), (1001, 1111, 2000)]


@pytest.mark.parametrize("xt,wt", [(torch.float8_e4m3fn, torch.float8_e4m3fn), (torch.float8_e5m2, torch.float8_e4m3fn),
                                   (torch.float8_e4m3fn, torch.float8_e5m2), (torch.float8_e5m2, torch.float8_e5m2)])
@pytest.mark.parametrize("rows,out,cols", FP8_SHAPES)
def test_linear_fp8(rows, out, cols, xt, wt):
    x, xs, w, ws = fp8_operands(rows, out, cols, xt, wt)
    m = mb.Fp8Matrix(w, ws)
    ref, mag = fp8_linear_ref(x, xs, w, ws)
    for od in FLOATS:
        y = ops.linear_fp8(x, m, x_scale=xs, out_dtype=od)
        assert y.dtype == od
        within(y, ref, fp8_bound(ref, mag, cols, od), str(od))
    assert torch.equal(ops.linear_fp8(x, m, x_scale=xs, out_dtype=od), y)
    errors_are_clear()


@pytest.mark.parametrize("rows,d_ff,cols", [(1, 128, 16), (1, 2048, 768), (2, 128, 768), (5, 384, 144), (16, 256, 2000),
                                            (40, 640, 400), (129, 256, 272), (515, 896, 1024)])
@pytest.mark.parametrize("xt", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_linear_fp8_with_the_gate(rows, d_ff, cols, xt):
    x, xs, w, ws = fp8_operands(rows, 2 * d_ff, cols, xt, torch.float8_e4m3fn, seed=9)
    m = mb.Fp8Matrix(w, ws)
    ref, mag = fp8_linear_ref(x, xs, w, ws)
    e = fp8_bound(ref, mag, cols, torch.float32) + F * ref.abs()
    g, u = ref[:, :d_ff], ref[:, d_ff:]
    h = g * torch.sigmoid(g) * u
    for od in FLOATS:
        y = ops.linear_fp8(x, m, x_scale=xs, swiglu=True, out_dtype=od)
        # silu moves by at most 1.1 of its argument's error; its own evaluation costs a few f of 1 + |g|
        bound = half_step(od) * 1.01 * h.abs() + 1.02 * (1.1 * u.abs() * e[:, :d_ff] + (g * torch.sigmoid(g)).abs() * e[:, d_ff:]) + \
            F * (16 + 4 * g.abs()) * h.abs() + (2.0 ** -25 if od == torch.float16 else 1e-37)
        within(y, h, bound, str(od))
    errors_are_clear()


def test_linear_fp8_quantises_and_takes_strides():
    dt = torch.bfloat16
    x = rand(6, 11, 272, seed=1, dt=dt)
    w = rand(200, 272, seed=2, dt=dt)
    m = mb.Fp8Matrix.from_dense(w)
    q, s = ops.quantize_fp8(x.reshape(66, 272))
    y = ops.linear_fp8(x, m)
    assert y.shape == (6, 11, 200) and y.dtype == dt
    assert torch.equal(y.reshape(66, 200), ops.linear_fp8(q, m, x_scale=s))
    assert torch.equal(m.to_dense(torch.float32).double(), fp8_linear_ref(torch.eye(272, device=DEV).to(q.dtype), torch.ones(272, 3, device=DEV), m.data, m.scale)[0].t())
    # rows of wider tensors
    wide = torch.zeros(66, 400, device=DEV, dtype=torch.uint8).view(q.dtype)
    wide[:, 16:288] = q
    swide = torch.zeros(66, 7, device=DEV)
    swide[:, 2:5] = s
    assert torch.equal(ops.linear_fp8(wide[:, 16:288], m, x_scale=swide[:, 2:5]), y.reshape(66, 200))
    wwide = torch.zeros(200, 304, device=DEV, dtype=torch.uint8).view(q.dtype)
    wwide[:, 16:288] = m.data
    assert torch.equal(ops.linear_fp8(q, mb.Fp8Matrix(wwide[:, 16:288], m.scale), x_scale=s), y.reshape(66, 200))
    assert ops.linear_fp8(q[:0], m, x_scale=s[:0]).shape == (0, 200)


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_linear_fp8_bad_values_stay_in_their_row(rows):
    x, xs, w, ws = fp8_operands(rows + 1, 256, 272, torch.float8_e4m3fn, torch.float8_e4m3fn, seed=3)
    m = mb.Fp8Matrix(w, ws)
    clean = ops.linear_fp8(x, m, x_scale=xs)
    xs[rows, 2] = float("nan")                                       # the short last block of one token
    y = ops.linear_fp8(x, m, x_scale=xs)
    assert torch.isnan(y[rows]).all() and torch.equal(y[:rows], clean[:rows])


# ---- together -------------------------------------------------------------------------------

def test_registered_operators_match_and_differentiate():
    ns = torch.ops.mortar_b200
    dt = torch.bfloat16
    x = rand(70, 128, seed=1, dt=dt).requires_grad_()
    w, b = rand(128, seed=2).requires_grad_(), rand(128, seed=3).requires_grad_()
    gu, dn = rand(512, 128, seed=4, scale=0.1, dt=dt).requires_grad_(), rand(128, 256, seed=5, scale=0.1, dt=dt).requires_grad_()
    dy = rand(70, 128, seed=6, dt=dt)
    leaves = (x, w, b, gu, dn)
    a = torch.autograd.grad(ops.mlp_dense(ops.layer_norm(x, w, b), gu, dn), leaves, dy)
    n, stats = ns.layer_norm(x, w, b, 1e-5)
    assert not stats.requires_grad
    y, hidden, sums = ns.mlp_dense(n, gu, dn)
    c = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    q, s = ns.quantize_fp8(x.detach(), 1, False)
    m = mb.Fp8Matrix.from_dense(gu)
    assert torch.equal(ns.linear_fp8(q, s, m.data, m.scale, True, dt), ops.linear_fp8(x.detach(), m, swiglu=True))
    assert torch.equal(ns.dequantize_fp8(q, s, dt), ops.dequantize_fp8(q, s))


def test_site_trains_and_is_served_in_8_bits():
    """Norm, block and 8-bit form as a user runs them: a training step by the module against the 64-bit
    composition, then the same weights served in 8 bits."""
    torch.manual_seed(0)
    site = mb.SwiGLUDense(256, 512, norm=True, device=DEV)
    x = rand(3, 50, 256, seed=1).requires_grad_()
    dy = rand(3, 50, 256, seed=2, dt=torch.bfloat16)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = site(x)
    y.backward(dy)
    assert all(p.grad is not None and p.grad.dtype == torch.float32 for p in site.parameters())
    xd = x.detach().double().requires_grad_()
    ws = [p.detach().double().requires_grad_() for p in (site.norm.weight, site.norm.bias, site.gate_up.weight, site.down.weight)]
    s = ln_ref_graph(xd, ws[0], ws[1], site.norm.eps) @ ws[2].t()
    yd = (torch.nn.functional.silu(s[..., :512]) * s[..., 512:]) @ ws[3].t()
    grads = torch.autograd.grad(yd, (xd, *ws), dy.double())
    # weights and the norm's output are rounded to bf16 too: 8 roundings at most meet in a gradient
    close_in_norm(y.detach(), yd.detach(), torch.bfloat16, 8, "y")
    for name, got, ref in zip(("x", "norm.weight", "norm.bias", "gate_up", "down"),
                              (x.grad, site.norm.weight.grad, site.norm.bias.grad, site.gate_up.weight.grad, site.down.weight.grad), grads):
        close_in_norm(got, ref, torch.bfloat16, 8, name)
    served = site.to_fp8()
    xb = x.detach().bfloat16()
    got = served(xb)
    # the same composition from the parts
    n = ops.layer_norm(xb, site.norm.weight, site.norm.bias, site.norm.eps).detach()
    gu, dn = mb.Fp8Matrix.from_dense(site.gate_up.weight), mb.Fp8Matrix.from_dense(site.down.weight)
    h = ops.linear_fp8(n, gu, swiglu=True)
    assert torch.equal(got, ops.linear_fp8(h, dn))
    # four tensors rounded to e4m3 on the way (2^-4 each at most, in squares)
    assert float((got.double() - yd.detach()).norm() / yd.detach().norm()) <= 2.0 ** -4 * 4 ** 0.5
    errors_are_clear()


def ln_ref_graph(x, w, b, eps):
    mean = x.mean(-1, keepdim=True)
    return (x - mean) / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps) * w + b


def test_streams_and_graphs():
    """A training step and a served step on a side stream, captured twice and replayed with new inputs, the
    two graphs' replays running at the same time on two streams."""
    dt = torch.bfloat16
    gu, dn = rand(512, 128, seed=1, scale=0.1, dt=dt), rand(128, 256, seed=2, scale=0.1, dt=dt)
    w, b = rand(128, seed=3), rand(128, seed=4)
    m8 = mb.Fp8Matrix.from_dense(gu)
    dy = rand(300, 128, seed=5, dt=dt)

    def step(x):
        x = x.detach().requires_grad_()
        ws = [t.detach().requires_grad_() for t in (w, b, gu, dn)]
        n = ops.layer_norm(x, ws[0], ws[1])
        y = ops.mlp_dense(n, ws[2], ws[3])
        return [y.detach(), ops.linear_fp8(n.detach(), m8, swiglu=True), *torch.autograd.grad(y, (x, *ws), dy)]

    xs = [rand(300, 128, seed=10 + i, dt=dt) for i in range(2)]
    want = [step(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want[0]))
    static = [torch.zeros_like(x) for x in xs]
    graphs, outs = [], []
    for st in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(st))
        graphs.append(g)
    for order in ((0, 1), (1, 0)):
        for st, i in zip(static, order):
            st.copy_(xs[i])
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for o, i in zip(outs, order):
            assert all(torch.equal(p, q) for p, q in zip(o, want[i]))
    errors_are_clear()


def test_broadcast_gradients_and_second_derivatives():
    """A gradient of stride 0 (from a sum) counts like one that is written out; create_graph is refused."""
    dt = torch.bfloat16
    x, gu, dn = (rand(40, 64, seed=1, dt=dt).requires_grad_(), rand(96, 64, seed=2, scale=0.2, dt=dt).requires_grad_(),
                 rand(64, 48, seed=3, scale=0.2, dt=dt).requires_grad_())
    a = torch.autograd.grad(ops.mlp_dense(x, gu, dn).sum(), (x, gu, dn))
    b = torch.autograd.grad(ops.mlp_dense(x, gu, dn), (x, gu, dn), torch.ones(40, 64, device=DEV, dtype=dt))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    for f in (lambda: ops.mlp_dense(x, gu, dn), lambda: ops.layer_norm(x)):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(f().sum(), x, create_graph=True)


def test_one_row_views_and_misaligned_weights():
    """Rows whose stride says nothing (one row, expanded or sliced), and 8-bit weights that start off 16 bytes."""
    dt = torch.bfloat16
    gu, dn = rand(96, 64, seed=2, scale=0.2, dt=dt), rand(64, 48, seed=3, scale=0.2, dt=dt)
    row = rand(1, 64, seed=1, dt=dt)
    want = ops.mlp_dense(row, gu, dn)
    views = [row[0], row.expand(3, 64), rand(5, 64, seed=1, dt=dt)[::5], torch.as_strided(row, (1, 64), (1, 1))]
    for v in views:
        y = ops.mlp_dense(v, gu, dn)
        assert y.shape == v.shape
        assert torch.equal(ops.layer_norm(v).reshape(-1, 64)[0], ops.layer_norm(v.contiguous().clone()).reshape(-1, 64)[0])
    assert torch.equal(ops.mlp_dense(views[0], gu, dn), want[0]) and torch.equal(ops.mlp_dense(views[3], gu, dn), want)
    flat = torch.zeros(64 * 128 + 16, device=DEV, dtype=torch.uint8)
    m = mb.Fp8Matrix.from_dense(rand(64, 128, seed=4))
    off = flat[4:4 + 64 * 128].view(m.data.dtype).reshape(64, 128)
    off.copy_(m.data)
    x = rand(7, 128, seed=5, dt=dt)
    assert off.data_ptr() % 16 == 4
    assert torch.equal(ops.linear_fp8(x, mb.Fp8Matrix(off, m.scale)), ops.linear_fp8(x, m))
    q, s = ops.quantize_fp8(x[:1])
    assert torch.equal(ops.linear_fp8(q[0], m, x_scale=s[0]), ops.linear_fp8(q, m, x_scale=s)[0])
    wide = torch.as_strided(s, (1, 1), (0, 1))
    assert torch.equal(ops.linear_fp8(q, m, x_scale=wide), ops.linear_fp8(q, m, x_scale=s))


def test_calls_from_a_new_thread():
    """A thread that has made no CUDA call yet (as autograd's do) can make these."""
    import threading
    dt = torch.bfloat16
    x, gu, dn = rand(200, 64, seed=1, dt=dt), rand(512, 64, seed=2, scale=0.2, dt=dt), rand(64, 256, seed=3, scale=0.2, dt=dt)
    m = mb.Fp8Matrix.from_dense(gu)
    q, s = ops.quantize_fp8(x)
    want = [ops.mlp_dense(x, gu, dn), ops.linear_fp8(q, m, x_scale=s, swiglu=True), ops.layer_norm(x)]
    got = []

    def work():
        got.extend([ops.mlp_dense(x, gu, dn), ops.linear_fp8(q, m, x_scale=s, swiglu=True), ops.layer_norm(x)])
        torch.cuda.current_stream().synchronize()

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert len(got) == 3 and all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("rows,d,f", [(256, 32, 16384), (512, 4096, 64), (8192, 32, 48)])
def test_mlp_dense_cut_reductions(rows, d, f):
    """Few tiles and long reductions: the products are cut and joined; the same bits every time."""
    dt = torch.bfloat16
    x = rand(rows, d, seed=1, dt=dt).requires_grad_()
    gu, dn = rand(2 * f, d, seed=2, scale=d ** -0.5, dt=dt).requires_grad_(), rand(d, f, seed=3, scale=f ** -0.5, dt=dt).requires_grad_()
    dy = rand(rows, d, seed=4, dt=dt)
    y = ops.mlp_dense(x, gu, dn)
    got = (y.detach(), *torch.autograd.grad(y, (x, gu, dn), dy))
    *refs, parts = mlp_grads_ref(dy, x.detach(), gu.detach(), dn.detach())
    for name, p, ref, bound in zip(("y", "dx", "dgate_up", "ddown"), got, refs, mlp_bounds(dy, x.detach(), gu.detach(), dn.detach(), parts, dt)):
        within(p, ref, bound, name)
        close_in_norm(p, ref, dt, 2, name)
    y = ops.mlp_dense(x, gu, dn)
    again = (y.detach(), *torch.autograd.grad(y, (x, gu, dn), dy))
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    errors_are_clear()


def test_calls_from_many_threads_at_once():
    """Threads on streams of their own call every operator at the same time, forward and backward."""
    import threading
    dt = torch.bfloat16
    gu, dn = rand(512, 128, seed=2, scale=0.2, dt=dt), rand(128, 256, seed=3, scale=0.2, dt=dt)
    w, b = rand(128, seed=4), rand(128, seed=5)
    m = mb.Fp8Matrix.from_dense(gu)
    xs = [rand(rows, 128, seed=rows, dt=dt) for rows in (1, 37, 300, 1111)]

    def step(x):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, gu, dn)]
        n = ops.layer_norm(*leaves[:3])
        y = ops.mlp_dense(n, *leaves[3:])
        return [y.detach(), ops.linear_fp8(n.detach(), m, swiglu=True), *torch.autograd.grad(y.square().sum(), leaves)]

    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    wrong, ran = [], []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = step(xs[i])
                torch.cuda.current_stream().synchronize()
                wrong.extend(k for k, (p, q) in enumerate(zip(got, want[i])) if not torch.equal(p, q))
        ran.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(ran) == list(range(len(xs))) and not wrong
    errors_are_clear()


def test_captured_training_step_beside_an_eager_graph():
    """A training step cannot be captured while a graph of the default stream holds the gradients of the same
    leaves (it is refused before anything is captured); a served step can, and so can the training step once
    that graph is gone."""
    dt = torch.bfloat16
    site = mb.modules.SwiGLUDense(64, 128, device=DEV, dtype=dt)
    x = rand(40, 64, seed=1, dt=dt)
    dy = rand(40, 64, seed=2, dt=dt)
    held = site(x)
    params = list(site.parameters())
    want = [held.detach().clone(), *torch.autograd.grad(held, params, dy, retain_graph=True)]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(graph):
            site(x)
    gu = site.gate_up.weight
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.mlp_dense(x, gu, site.down.weight.detach())
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = site(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want[0])
    del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = site(x)
        got = torch.autograd.grad(y, params, dy)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip((y.detach(), *got), want))
    errors_are_clear()


def test_negated_views():
    """Views that stand for the negative of what memory holds (the imaginary part of a conjugate)."""
    z = torch.complex(rand(9, 64, seed=1), rand(9, 64, seed=2))
    x = z.conj().imag
    assert x.is_neg()
    plain = (-z.imag).contiguous()
    assert torch.equal(ops.layer_norm(x), ops.layer_norm(plain))
    assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(ops.quantize_fp8(x), ops.quantize_fp8(plain)))
    w = z[0].conj().imag
    assert torch.equal(ops.layer_norm(plain, w, w), ops.layer_norm(plain, plain[0], plain[0]))
    one = torch._neg_view(rand(64, seed=3))
    assert torch.equal(ops.layer_norm(plain, one), ops.layer_norm(plain, one.resolve_neg()))
    packed = torch._neg_view(plain)
    assert packed.is_contiguous() and torch.equal(ops.layer_norm(packed), ops.layer_norm(packed.resolve_neg()))


def test_replaced_parts_of_a_matrix_are_refused():
    m = mb.Fp8Matrix.from_dense(rand(256, 256, seed=1))
    x = rand(5, 256, seed=2, dt=torch.bfloat16)
    for part, value in (("scale", m.scale[:1]), ("scale", m.scale.double()), ("scale", m.scale.cpu()), ("data", m.data[0]),
                        ("data", m.data.view(torch.uint8)), ("data", m.data.t())):
        keep = getattr(m, part)
        setattr(m, part, value)
        with pytest.raises(ValueError):
            ops.linear_fp8(x, m)
        setattr(m, part, keep)
    ops.linear_fp8(x, m)


def test_captured_step_of_cast_weights_beside_an_eager_graph():
    """The same where the operator does not see the leaf itself: fp32 weights that are cast on the way."""
    site = mb.modules.SwiGLUDense(64, 128, norm=True, device=DEV)
    x = rand(40, 64, seed=1, dt=torch.bfloat16)
    held = site(x)
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            site(x)
    weights = [p.detach().requires_grad_() for p in (site.gate_up.weight, site.down.weight)]
    cast = [w.to(torch.bfloat16) for w in weights]
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.mlp_dense(x, *cast)
    del held, cast
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(site(x).square().sum(), list(site.parameters()))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, torch.autograd.grad(site(x).square().sum(), list(site.parameters()))))
    errors_are_clear()


@pytest.mark.parametrize("rows,out,cols", [(300, 10200, 272), (520, 13000, 144), (257, 18944, 128), (4000, 4736, 96)])
def test_linear_fp8_rounds_of_whole_and_half_tiles(rows, out, cols):
    """More tiles than run at once, the last of them cut in two (80, 153, 148 and 304 tiles of 256 x 256)."""
    test_linear_fp8(rows, out, cols, torch.float8_e4m3fn, torch.float8_e4m3fn)
    if out % 256 == 0:
        test_linear_fp8_with_the_gate(rows, out // 2, cols, torch.float8_e5m2)


@pytest.mark.parametrize("d_ff", [128 * 40, 128 * 75])
def test_linear_fp8_gate_of_whole_and_half_tiles(d_ff):
    test_linear_fp8_with_the_gate(300, d_ff, 400, torch.float8_e4m3fn)


@pytest.mark.parametrize("rows,d,f", [(2100, 528, 2064), (5000, 1040, 400), (1030, 2576, 1296)])
def test_mlp_dense_tiles_of_both_widths(rows, d, f):
    """Launches whose tiles fill the machine and launches whose do not, ragged in every direction: of the first shape
    gate/up, dh and the gradients run on tiles of 256 columns and down on 128, of the second only dh on 128."""
    test_mlp_dense_cut_reductions(rows, d, f)


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_fp8_rows_off_32_bytes(dt, block_rows):
    """Rows that start on 16 but not on 32 bytes, read and written."""
    e = dt.itemsize
    x = rand(130, 416, seed=1, dt=dt)[:, :400].contiguous()
    per16 = 16 // e
    wide = torch.zeros(130, 400 + per16, device=DEV, dtype=dt)
    views = [wide[:, :400], wide[:, per16:]]
    want = ops.quantize_fp8(x, block_rows=block_rows)
    for v in views:
        v.copy_(x)
        got = ops.quantize_fp8(v, block_rows=block_rows)
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(got, want))
    back = ops.dequantize_fp8(*want, out_dtype=dt)
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dt]
    wide.fill_(7.0)
    rc = mb._lib.lib().mortar_dequantize_fp8(want[0].data_ptr(), 3, 400, want[1].data_ptr(), 130, 400, block_rows,
                                             wide[:, per16:].data_ptr(), code, 400 + per16, torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(wide[:, per16:], back) and bool((wide[:, :per16] == 7.0).all())


@pytest.mark.parametrize("off,ld", [(4, 72), (0, 68), (8, 72), (4, 68)])
def test_layer_norm_fp32_rows_off_32_bytes(off, ld):
    """fp32 rows whose 8-column units start on 16 bytes only take the kernel for any alignment: the results are as close."""
    flat = torch.zeros(33 * 72 + 16, device=DEV)
    x = torch.as_strided(flat, (33, 64), (ld, 1), off)
    x.copy_(rand(33, 64, seed=1) + 0.5)
    w, b, dy = rand(64, seed=2), rand(64, seed=3), rand(33, 64, seed=4)
    y, stats = ops.layer_norm_forward(x, w, b, 1e-5, True)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, stats)
    ry, xh, rstd, mean, rdx, rdw, rdb = ln_ref(x, w, b, 1e-5, dy)
    # 64 terms in sums of depth <= 16, a few operations each: 64 f of the largest magnitudes that meet
    within(y, ry, 64 * F * (1 + ry.abs().max()), "y")
    within(dx, rdx, 64 * F * (1 + rdx.abs().max()) * (1 + xh.abs().max()) ** 2, "dx")
    within(dw, rdw.sum(0), 64 * F * (dy.double() * xh).abs().sum(0), "dw")
    within(db, rdb.sum(0), 64 * F * dy.double().abs().sum(0), "db")


@pytest.mark.parametrize("rows,out,cols", [(17, 128, 128), (32, 3333, 272), (33, 20000, 144), (64, 1000, 400), (65, 129, 2000),
                                           (100, 16, 16), (127, 20736, 96), (128, 515, 656), (18, 16, 16), (31, 20736, 96),
                                           (32, 20000, 656), (19, 129, 2000)])
def test_linear_fp8_few_rows(rows, out, cols):
    """17 to 32 rows, where the operands change places, and a few more: one tile and more than run at once, ragged widths."""
    test_linear_fp8(rows, out, cols, torch.float8_e5m2, torch.float8_e4m3fn)
    test_linear_fp8(rows, out, cols, torch.float8_e4m3fn, torch.float8_e5m2)


@pytest.mark.parametrize("rows,d_ff,cols", [(17, 128, 16), (31, 1280, 272), (40, 128 * 76, 144), (64, 384, 2000), (128, 640, 400),
                                            (32, 128 * 76, 144), (20, 384, 2000)])
def test_linear_fp8_few_rows_with_the_gate(rows, d_ff, cols):
    test_linear_fp8_with_the_gate(rows, d_ff, cols, torch.float8_e4m3fn)
    test_linear_fp8_with_the_gate(rows, d_ff, cols, torch.float8_e5m2)


def test_linear_fp8_few_rows_write_their_rows_only():
    """The C entry with rows of the output further apart than they are wide, and a wide reduction that the few rows'
    table has no room for."""
    for rows, out, cols in ((33, 300, 272), (100, 64, 128 * 170), (19, 300, 272), (30, 64, 128 * 1000)):
        x, xs, w, ws = fp8_operands(rows, out, cols, torch.float8_e4m3fn, torch.float8_e4m3fn)
        y = torch.full((rows + 3, out + 5), 7.0, device=DEV)
        rc = mb._lib.lib().mortar_linear_fp8(x.data_ptr(), 3, cols, xs.data_ptr(), xs.shape[1], rows, w.data_ptr(), 3, cols, ws.data_ptr(),
                                             ws.shape[1], out, cols, 0, y.data_ptr(), 0, out + 5, torch.cuda.current_stream().cuda_stream)
        ref, mag = fp8_linear_ref(x, xs, w, ws)
        assert rc == 0
        within(y[:rows, :out], ref, fp8_bound(ref, mag, cols, torch.float32))
        assert bool((y[rows:] == 7).all()) and bool((y[:, out:] == 7).all())
    errors_are_clear()


@pytest.mark.parametrize("rows,out,cols", [(17, 300, 400), (24, 515, 2000), (32, 3070, 144), (32, 4096, 2064), (31, 16, 16)])
def test_linear_fp8_few_rows_of_narrow_weights(rows, out, cols):
    """17 to 32 rows and few output columns: the reduction is shared instead."""
    test_linear_fp8(rows, out, cols, torch.float8_e4m3fn, torch.float8_e4m3fn)
    test_linear_fp8(rows, out, cols, torch.float8_e5m2, torch.float8_e5m2)
    if out == 4096:
        test_linear_fp8_with_the_gate(rows, out // 2, cols, torch.float8_e4m3fn)


@pytest.mark.parametrize("rows,out,cols", [(33, 2048, 5632), (64, 300, 128 * 40 + 16), (128, 515, 4096), (333, 768, 128 * 23), (600, 300, 3200)])
def test_linear_fp8_cut_reductions(rows, out, cols):
    """Few tiles and long reductions: the parts are joined in order, the same bits every time (the called test compares
    two calls), any output type, width and stride."""
    assert mb._lib.lib().mortar_linear_fp8_scratch_floats(rows, out, cols, 0) > 0
    test_linear_fp8(rows, out, cols, torch.float8_e4m3fn, torch.float8_e4m3fn)
    x, xs, w, ws = fp8_operands(rows, out, cols, torch.float8_e5m2, torch.float8_e4m3fn)
    whole, cut = (torch.full((rows + 2, out + 3), 7.0, device=DEV) for _ in range(2))
    lib, st = mb._lib.lib(), torch.cuda.current_stream().cuda_stream
    n = lib.mortar_linear_fp8_scratch_floats(rows, out, cols, 0)
    scratch = torch.empty(n, device=DEV)
    args = lambda y: (x.data_ptr(), 4, cols, xs.data_ptr(), xs.shape[1], rows, w.data_ptr(), 3, cols, ws.data_ptr(), ws.shape[1], out, cols, 0,
                      y.data_ptr(), 0, out + 3)
    assert lib.mortar_linear_fp8(*args(whole), st) == 0
    assert lib.mortar_linear_fp8_cut(*args(cut), scratch.data_ptr(), n, st) == 0
    assert lib.mortar_linear_fp8_cut(*args(cut), scratch.data_ptr(), n - 1, st) == -8
    ref, mag = fp8_linear_ref(x, xs, w, ws)
    for y in (whole, cut):
        within(y[:rows, :out], ref, fp8_bound(ref, mag, cols, torch.float32))
        assert bool((y[rows:] == 7).all()) and bool((y[:, out:] == 7).all())
    errors_are_clear()


# ---- many rows, tiles and units for each worker ------------------------------------------------

LN_MANY_ROWS = [(12007, 768), (6001, 1536), (5003, 2048), (1501, 4096), (1703, 5632), (1103, 8192), (14503, 136), (1003, 12000),
                (1002, 16384), (5003, 1001), (3001, 2047), (1005, 8191), (905, 16383), (20011, 7), (1502, 20011)]


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("rows,cols", LN_MANY_ROWS)
def test_layer_norm_many_rows_a_group(rows, cols, dt):
    """Each group of warps takes three to twenty rows, the last of them not in all groups: the row that is on its way, slots
    that are filled again, sums that take turns, and column sums that are carried from row to row, for every number of units
    a thread takes (8 to 32 columns), rows of whole vectors and others, and rows that are read again."""
    test_layer_norm_and_its_gradients(rows, cols, dt)
    x, dy = (rand(rows, cols, seed=1, scale=2.0) + 0.5).to(dt), rand(rows, cols, seed=4, dt=dt)
    w = 1 + rand(cols, seed=2, scale=0.2)
    _, stats = ops.layer_norm_forward(x, w, None, 1e-5, True)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, stats)
    # one gradient without the others has the same bits
    assert torch.equal(ops.layer_norm_backward(dy, x, w, stats, True, False, False)[0], dx)
    got = ops.layer_norm_backward(dy, x, w, stats, False, True, True)
    assert got[0] is None and torch.equal(got[1], dw) and torch.equal(got[2], db)


@pytest.mark.parametrize("dt", FLOATS)
def test_layer_norm_many_rows_of_a_wider_tensor(dt):
    """The same for rows that start anywhere and end inside a wider tensor, whose other values are NaN."""
    wide = torch.full((3001, 520), float("nan"), device=DEV, dtype=dt)
    x, dy, w = rand(3001, 512, seed=1, dt=dt), rand(3001, 512, seed=2, dt=dt), 1 + rand(512, seed=3, scale=0.2)
    y, stats = ops.layer_norm_forward(x, w, None, 1e-5, True)
    want = ops.layer_norm_backward(dy, x, w, stats)
    ry, xh, rstd, _, rdx, tw, tb = ln_ref(x, w, None, 1e-5, dy)
    by, bdx = ln_bounds(x, w, None, ry, xh, rstd, rdx, dy, dt)
    for off in (1, 3, 8):
        v = wide[:, off:off + 512]
        v.copy_(x)
        got, st = ops.layer_norm_forward(v, w, None, 1e-5, True)
        dx, dw, db = ops.layer_norm_backward(dy, v, w, st)
        within(got, ry, by, f"y at {off}")
        within(dx, rdx, bdx, f"dx at {off}")
        # two sums in another order: each off by its bound
        n = 3001 / 8 + 320
        assert bool(((dw - want[1]).double().abs() <= 2 * F * (n * tw.abs() + (512 / 16 + 48) * (tw.abs() + dy.double().abs() * rstd * x.double().abs().mean(-1, keepdim=True))).sum(0)).all())
        assert bool(((db - want[2]).double().abs() <= 2 * F * n * tb.abs().sum(0)).all())
        wide.fill_(float("nan"))


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("rows,cols,block_rows", [(6007, 2064, 1), (40009, 144, 1), (6007, 2064, 128)])
def test_quantize_fp8_many_units_a_warp(rows, cols, block_rows, dt, dtype):
    """More blocks than the grid's warps take at once, written and read back."""
    test_quantize_fp8_is_exact(rows, cols, block_rows, dt, dtype)


@pytest.mark.parametrize("rows,d,f", [(8200, 1040, 2576), (8200, 2064, 528)])
def test_mlp_dense_many_tiles_a_cluster(rows, d, f):
    """Four and more tiles a cluster in every launch: both accumulators in turn, more than once."""
    test_mlp_dense_cut_reductions(rows, d, f)


@pytest.mark.parametrize("rows,out,cols", [(5000, 6500, 144), (5000, 6656, 400), (20, 60000, 272), (32, 40960, 400), (5, 30000, 272), (12, 30976, 656)])
def test_linear_fp8_many_tiles_a_cluster(rows, out, cols):
    """The same for the 8-bit product: whole tiles alone (seven rounds), few rows on either kind of kernel."""
    test_linear_fp8(rows, out, cols, torch.float8_e4m3fn, torch.float8_e4m3fn)
    if out % 256 == 0:
        test_linear_fp8_with_the_gate(rows, out // 2, cols, torch.float8_e5m2)


# ---- derivatives that do not exist -------------------------------------------------------------

def test_no_derivative_vanishes():
    """Tangents and required gradients where an operator has no rule: refused, not dropped."""
    import torch.autograd.forward_ad as fwd
    x, w = rand(5, 64, seed=1), rand(64, 64, seed=2)
    xb, gu, dn = (rand(5, 64, seed=3, dt=torch.bfloat16), rand(64, 64, seed=4, dt=torch.bfloat16), rand(64, 32, seed=5, dt=torch.bfloat16))
    m = mb.Fp8Matrix.from_dense(w)
    q, s = ops.quantize_fp8(x)
    with fwd.dual_level(), torch.no_grad():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for f in (lambda: ops.layer_norm(dual), lambda: ops.quantize_fp8(dual), lambda: ops.linear_fp8(dual, m),
                  lambda: ops.mlp_dense(fwd.make_dual(xb, xb), gu, dn), lambda: ops.mlp_fp8(dual, m, m),
                  lambda: torch.ops.mortar_b200.layer_norm(dual, None, None, 1e-5),
                  lambda: torch.ops.mortar_b200.mlp_dense(fwd.make_dual(xb, xb), gu, dn)):
            with pytest.raises(ValueError):
                f()
        primal, _ = fwd.unpack_dual(dual)
        assert torch.equal(ops.layer_norm(primal), ops.layer_norm(x))
    leaf = x.clone().requires_grad_()
    for f in (lambda: ops.quantize_fp8(leaf), lambda: ops.dequantize_fp8(q, s.clone().requires_grad_()), lambda: ops.linear_fp8(leaf, m),
              lambda: ops.linear_fp8(q, mb.Fp8Matrix(m.data, m.scale.clone().requires_grad_()), x_scale=s)):
        with pytest.raises(ValueError, match="not differentiable"):
            f()
        with torch.no_grad():
            f()


def test_linear_fp8_takes_scales_of_any_stride():
    """One column of scales that is a transposed row, and scales that are the negative of what memory holds."""
    x, xs, w, ws = fp8_operands(40, 300, 64, torch.float8_e4m3fn, torch.float8_e4m3fn)
    want = ops.linear_fp8(x, mb.Fp8Matrix(w, ws), x_scale=xs)
    assert torch.equal(ops.linear_fp8(x, mb.Fp8Matrix(w, ws.reshape(1, 3).clone().t()), x_scale=xs), want)
    assert torch.equal(ops.linear_fp8(x, mb.Fp8Matrix(w, torch._neg_view(-ws)), x_scale=xs), want)
    assert torch.equal(torch.ops.mortar_b200.linear_fp8(x, xs, w, ws.reshape(1, 3).clone().t(), False, want.dtype), want)


# ---- the registered operators ------------------------------------------------------------------

def test_registered_block_without_gradients_is_the_served_one():
    """``want_saved=False``: the kernels and the bits of the call without gradients, at one token and at many."""
    dt = torch.bfloat16
    gu, dn = rand(512, 128, seed=1, scale=0.1, dt=dt), rand(128, 256, seed=2, scale=0.1, dt=dt)
    for rows in (1, 32, 33, 300):
        x = rand(rows, 128, seed=3, dt=dt)
        before = ops.kernel_counts().get("dense", 0)
        y, hidden, sums = torch.ops.mortar_b200.mlp_dense(x, gu, dn, False)
        between = ops.kernel_counts()["dense"]
        assert torch.equal(y, ops.mlp_dense(x, gu, dn)) and hidden.numel() == 0 and sums.numel() == 0
        assert between - before == ops.kernel_counts()["dense"] - between
    errors_are_clear()


@pytest.mark.parametrize("wanted", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 1, 1)])
def test_registered_rules_compute_the_wanted_gradients(wanted, monkeypatch):
    asked = []
    for name in ("mlp_dense_backward", "layer_norm_backward"):
        def recorded(*args, real=getattr(ops, name)):
            asked.append([bool(w) for w in args[-3:]])
            return real(*args)
        monkeypatch.setattr(ops, name, recorded)
    ns, dt = torch.ops.mortar_b200, torch.bfloat16
    for call, parts in ((ns.mlp_dense, (rand(40, 64, seed=1, dt=dt), rand(256, 64, seed=2, scale=0.1, dt=dt), rand(64, 128, seed=3, scale=0.1, dt=dt))),
                        (lambda *a: ns.layer_norm(*a, 1e-5), (rand(40, 64, seed=1, dt=dt), rand(64, seed=2), rand(64, seed=3, dt=dt)))):
        plain = ops.mlp_dense if call is ns.mlp_dense else ops.layer_norm
        leaves = [t.requires_grad_(bool(w)) for t, w in zip(parts, wanted)]
        chosen = [t for t in leaves if t.requires_grad]
        dy = rand(40, 64, seed=4, dt=dt)
        asked.clear()
        got = torch.autograd.grad(call(*leaves)[0], chosen, dy)
        assert asked == [[bool(w) for w in wanted]]
        want = torch.autograd.grad(plain(*leaves), chosen, dy)
        assert all(torch.equal(p, q) and p.dtype == q.dtype for p, q in zip(got, want))
    errors_are_clear()


def test_captured_registered_step_beside_an_eager_graph():
    """The registered operators refuse the captured training step that ``ops`` refuses, and take it once the graph that holds
    the leaves is gone."""
    ns, dt = torch.ops.mortar_b200, torch.bfloat16
    x, dy = rand(40, 64, seed=1, dt=dt), rand(40, 64, seed=2, dt=dt)
    leaves = [rand(64, seed=3).requires_grad_(), rand(64, seed=4).requires_grad_(),
              rand(256, 64, seed=5, scale=0.1, dt=dt).requires_grad_(), rand(64, 128, seed=6, scale=0.1, dt=dt).requires_grad_()]

    def step():
        n = ns.layer_norm(x, *leaves[:2], 1e-5)[0]
        return ns.mlp_dense(n, *leaves[2:])[0]

    held = step()
    want = [held.detach().clone(), *torch.autograd.grad(held, leaves, dy, retain_graph=True)]
    for call in (lambda: ns.layer_norm(x, *leaves[:2], 1e-5), lambda: ns.mlp_dense(x, *leaves[2:]), step):
        with pytest.raises(RuntimeError, match="default stream"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want[0])
    del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
        got = torch.autograd.grad(y, leaves, dy)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip((y.detach(), *got), want))
    errors_are_clear()


def test_compiled_site_is_the_eager_one():
    """The site compiled into one graph (captured ahead of time, run as it is): the bits of the eager calls, trained and
    served, and the same kernels for a served token."""
    torch.manual_seed(0)
    site = mb.SwiGLUDense(64, 128, norm=True, device=DEV, dtype=torch.bfloat16)
    params = list(site.parameters())
    compiled = torch.compile(site, backend="aot_eager", fullgraph=True)
    for rows in (40, 1):
        x, dy = rand(rows, 64, seed=rows, dt=torch.bfloat16).requires_grad_(), rand(rows, 64, seed=3, dt=torch.bfloat16)
        y, want = compiled(x), site(x)
        assert torch.equal(y, want)
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, (x, *params), dy), torch.autograd.grad(want, (x, *params), dy)))
        with torch.no_grad():
            first = ops.kernel_counts()["dense"]
            want = site(x)
            second = ops.kernel_counts()["dense"]
            assert torch.equal(compiled(x), want) and ops.kernel_counts()["dense"] - second == second - first
    served = site.to_fp8()
    x = rand(40, 64, seed=7, dt=torch.bfloat16)
    assert torch.equal(torch.compile(served, backend="aot_eager", fullgraph=True)(x), served(x))
    torch._dynamo.reset()
    errors_are_clear()


def test_linear_fp8_takes_scales_that_lie_far_apart():
    """Rows of scales whose positions pass 32 bits (a column of a very wide table) are copied, as other strides are."""
    for rows in (2, 40):
        x, xs, w, ws = fp8_operands(rows, 300, 272, torch.float8_e4m3fn, torch.float8_e4m3fn)
        m = mb.Fp8Matrix(w, ws)
        step = (1 << 32) // (rows - 1) + 8
        table = torch.empty((rows - 1) * step + 3, device=DEV)       # 17 GB, of which the rows of scales are written
        far = table.as_strided((rows, 3), (step, 1))
        far.copy_(xs)
        assert torch.equal(ops.linear_fp8(x, m, x_scale=far), ops.linear_fp8(x, m, x_scale=xs))
        del far, table
        torch.cuda.empty_cache()
    errors_are_clear()
