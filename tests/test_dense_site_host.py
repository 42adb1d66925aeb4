"""The dense MLP site without a GPU: what the entry points refuse, the shapes and types the
registered operators promise, and that CPU tensors are turned away."""
import ctypes as C

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mortar_b200 as mb

L = mb._lib.lib()
NULL, SHAPE, ALIGN, DTYPE, CAP = -1, -2, -6, -7, -8
F32, BF16, F16, E4M3, E5M2 = 0, 1, 2, 3, 4


def _buf(nbytes=4096):
    a = np.zeros(nbytes + 256, dtype=np.uint8)
    return a, C.c_void_p((a.ctypes.data + 255) & ~255)


def _off(p, n):
    return C.c_void_p(p.value + n)


def test_layer_norm_entry_points_validate():
    keep, p = _buf()
    f = L.mortar_layer_norm
    assert f(None, F32, 64, 4, 64, p, p, 1e-5, p, 64, p, None) == NULL
    assert f(p, F32, 64, 4, 64, p, p, 1e-5, None, 64, p, None) == NULL
    assert f(p, F32, 63, 4, 64, p, p, 1e-5, p, 64, p, None) == SHAPE
    assert f(p, F32, 64, 4, 64, p, p, 1e-5, p, 63, p, None) == SHAPE
    assert f(p, F32, 64, -1, 64, p, p, 1e-5, p, 64, p, None) == SHAPE
    assert f(p, F32, 64, 4, 0, p, p, 1e-5, p, 64, p, None) == SHAPE
    assert f(p, E4M3, 64, 4, 64, p, p, 1e-5, p, 64, p, None) == DTYPE
    assert f(_off(p, 2), F32, 64, 4, 64, p, p, 1e-5, p, 64, p, None) == ALIGN
    assert f(p, F32, (1 << 20) + 1, 4, (1 << 20) + 1, p, p, 1e-5, p, (1 << 20) + 1, p, None) == CAP
    assert f(p, F32, 64, 0, 64, p, p, 1e-5, p, 64, p, None) == 0
    b = L.mortar_layer_norm_backward
    assert b(None, 64, p, 64, F32, 4, 64, p, p, p, 64, p, p, p, 1 << 20, None) == NULL
    assert b(p, 64, p, 64, F32, 4, 64, p, None, p, 64, p, p, p, 1 << 20, None) == NULL
    assert b(p, 64, p, 64, F32, 4, 64, p, p, p, 60, p, p, p, 1 << 20, None) == SHAPE
    assert b(p, 64, p, 64, 9, 4, 64, p, p, p, 64, p, p, p, 1 << 20, None) == DTYPE
    assert b(p, 64, p, 64, F32, 4, 64, p, p, p, 64, p, p, None, 0, None) == CAP
    assert b(p, 64, p, 64, F32, 4, 64, p, p, p, 64, p, p, p, 1, None) == CAP
    assert L.mortar_layer_norm_scratch_floats(4, 0) == SHAPE
    assert L.mortar_layer_norm_scratch_floats(0, 64) >= 0


def test_mlp_dense_entry_points_validate():
    keep, p = _buf()
    f = L.mortar_mlp_dense
    ok = [p, 64, BF16, 4, p, 64, p, 128, 64, 128, p, p, p, 64, p, 1 << 20, None]

    def call(fn, base, **at):
        args = list(base)
        for i, v in at.items():
            args[int(i[1:])] = v
        return fn(*args)

    for i in (0, 4, 6, 10, 12):
        assert call(f, ok, **{f"a{i}": None}) == NULL
    assert call(f, ok, a3=-1) == SHAPE
    assert call(f, ok, a8=60) == SHAPE and call(f, ok, a9=120) == SHAPE
    assert call(f, ok, a1=32) == SHAPE and call(f, ok, a5=32) == SHAPE and call(f, ok, a7=64) == SHAPE
    assert call(f, ok, a13=32) == SHAPE
    assert call(f, ok, a2=F32) == DTYPE
    assert call(f, ok, a0=_off(p, 2)) == ALIGN and call(f, ok, a1=68) == ALIGN
    assert call(f, ok, a3=1 << 31) == CAP
    assert call(f, ok, a3=0) == 0
    need = L.mortar_mlp_dense_scratch_floats(200, 64, 4096, 0)                   # few tiles, a long reduction: it is cut
    assert need > 0 and L.mortar_mlp_dense_scratch_floats(1 << 16, 2048, 5632, 1) == 0
    long = dict(a3=200, a7=4096, a9=4096)
    assert call(f, ok, a14=None, **long) == CAP and call(f, ok, a15=need - 1, **long) == CAP
    assert L.mortar_mlp_dense_scratch_floats(4, 60, 64, 0) == SHAPE
    assert L.mortar_mlp_dense_backward_scratch_floats(4, 64, 60, 1, 1, 1) == SHAPE
    b = L.mortar_mlp_dense_backward
    okb = [p, 64, p, 64, BF16, 4, p, 64, p, 128, 64, 128, p, p, p, p, p, p, p, 1 << 20, None]
    for i in (0, 2, 6, 8, 12, 13, 14):
        assert call(b, okb, **{f"a{i}": None}) == NULL
    assert call(b, okb, a10=60) == SHAPE and call(b, okb, a1=32) == SHAPE
    assert call(b, okb, a4=F32) == DTYPE
    assert call(b, okb, a15=_off(p, 8)) == ALIGN


def test_fp8_entry_points_validate():
    keep, p = _buf()
    f = L.mortar_quantize_fp8
    assert f(None, BF16, 256, 8, 256, 1, p, E4M3, 256, p, None) == NULL
    assert f(p, BF16, 256, 8, 250, 1, p, E4M3, 256, p, None) == SHAPE
    assert f(p, BF16, 256, 8, 256, 64, p, E4M3, 256, p, None) == SHAPE
    assert f(p, BF16, 128, 8, 256, 1, p, E4M3, 256, p, None) == SHAPE
    assert f(p, E4M3, 256, 8, 256, 1, p, E4M3, 256, p, None) == DTYPE
    assert f(p, BF16, 256, 8, 256, 1, p, BF16, 256, p, None) == DTYPE
    assert f(_off(p, 2), BF16, 256, 8, 256, 1, p, E4M3, 256, p, None) == ALIGN
    assert f(p, BF16, 256, 8, 256, 1, p, E4M3, 264, p, None) == ALIGN
    assert f(p, BF16, 256, 0, 256, 1, p, E4M3, 256, p, None) == 0
    d = L.mortar_dequantize_fp8
    assert d(None, E4M3, 256, p, 8, 256, 1, p, BF16, 256, None) == NULL
    assert d(p, E4M3, 256, p, 8, 256, 2, p, BF16, 256, None) == SHAPE
    assert d(p, F32, 256, p, 8, 256, 1, p, BF16, 256, None) == DTYPE
    g = L.mortar_linear_fp8
    assert g(None, E4M3, 256, p, 2, 8, p, E4M3, 256, p, 2, 256, 256, 0, p, BF16, 256, None) == NULL
    assert g(p, E4M3, 256, None, 2, 8, p, E4M3, 256, p, 2, 256, 256, 0, p, BF16, 256, None) == NULL
    assert g(p, E4M3, 256, p, 1, 8, p, E4M3, 256, p, 2, 256, 256, 0, p, BF16, 256, None) == SHAPE    # scales of 1 block
    assert g(p, E4M3, 256, p, 2, 8, p, E4M3, 256, p, 2, 384, 256, mb._lib.FLAG_SWIGLU, p, BF16, 256, None) == SHAPE
    assert g(p, E4M3, 256, p, 2, 8, p, E4M3, 256, p, 2, 256, 250, 0, p, BF16, 256, None) == SHAPE
    assert g(p, E4M3, 256, p, 2, 8, p, E4M3, 256, p, 2, 256, 256, 0, p, BF16, 128, None) == SHAPE
    assert g(p, BF16, 256, p, 2, 8, p, E4M3, 256, p, 2, 256, 256, 0, p, BF16, 256, None) == DTYPE
    assert g(p, E4M3, 256, p, 2, 8, p, E4M3, 256, p, 2, 256, 256, 4, p, BF16, 256, None) == DTYPE     # unknown flag
    assert g(p, E4M3, 256, p, 2, 8, p, E4M3, 256, p, 2, 256, 256, 0, p, E4M3, 256, None) == DTYPE
    assert g(_off(p, 8), E4M3, 256, p, 2, 8, p, E4M3, 256, p, 2, 256, 256, 0, p, BF16, 256, None) == ALIGN
    assert g(p, E4M3, 264, p, 2, 8, p, E4M3, 256, p, 2, 256, 256, 0, p, BF16, 256, None) == ALIGN
    assert g(p, E4M3, 256, p, 2, 0, p, E4M3, 256, p, 2, 256, 256, 0, p, BF16, 256, None) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="CUDA-only"):
        mb.ops.layer_norm(x)
    with pytest.raises(NotImplementedError, match="CUDA-only"):
        mb.ops.mlp_dense(x, torch.zeros(64, 64, dtype=x.dtype), torch.zeros(64, 32, dtype=x.dtype))
    with pytest.raises(NotImplementedError, match="CUDA-only"):
        mb.ops.quantize_fp8(x)
    q = torch.zeros(4, 64, dtype=torch.float8_e4m3fn)
    with pytest.raises(NotImplementedError, match="CUDA-only"):
        mb.ops.dequantize_fp8(q, torch.ones(4, 1))
    with pytest.raises(NotImplementedError, match="CUDA-only"):
        mb.ops.linear_fp8(q, mb.Fp8Matrix(q, torch.ones(1, 1)), x_scale=torch.ones(4, 1))


def test_wrong_arguments_are_refused():
    """On fake CUDA tensors: every refusal comes before a pointer is taken."""
    with FakeTensorMode():
        def z(*shape, dt=torch.bfloat16, dev="cuda"):
            return torch.empty(*shape, device=dev, dtype=dt)
        bad = [
            lambda: mb.ops.layer_norm(z(4, 64, dt=torch.int32)),
            lambda: mb.ops.layer_norm(z(4, 0)),
            lambda: mb.ops.layer_norm(z(4, 64), weight=z(63)),
            lambda: mb.ops.layer_norm(z(4, 64), bias=z(64, dt=torch.int64)),
            lambda: mb.ops.layer_norm(z(4, 64), weight=z(64, dev="cpu")),
            lambda: mb.ops.layer_norm_backward(z(4, 32), z(4, 64), None, z(2, 4, dt=torch.float32)),
            lambda: mb.ops.layer_norm_backward(z(4, 64), z(4, 64), None, z(2, 5, dt=torch.float32)),
            lambda: mb.ops.mlp_dense(z(4, 64, dt=torch.float32), z(64, 64), z(64, 32)),
            lambda: mb.ops.mlp_dense(z(4, 64), z(64, 64), z(64, 48)),
            lambda: mb.ops.mlp_dense(z(4, 48), z(64, 64), z(64, 32)),
            lambda: mb.ops.mlp_dense(z(4, 40), z(64, 40), z(40, 32)),
            lambda: mb.ops.mlp_dense(z(4, 64), z(64, 64, dt=torch.float16), z(64, 32)),
            lambda: mb.ops.mlp_dense(z(4, 64), z(64, 64, dev="cpu"), z(64, 32)),
            lambda: mb.ops.quantize_fp8(z(4, 64, 2)),
            lambda: mb.ops.quantize_fp8(z(4, 60)),
            lambda: mb.ops.quantize_fp8(z(4, 64), block_rows=32),
            lambda: mb.ops.quantize_fp8(z(4, 64), dtype=torch.float16),
            lambda: mb.ops.quantize_fp8(z(4, 64, dt=torch.int8)),
            lambda: mb.ops.dequantize_fp8(z(4, 64), z(4, 1, dt=torch.float32)),
            lambda: mb.ops.dequantize_fp8(z(4, 64, dt=torch.float8_e4m3fn), z(3, 1, dt=torch.float32)),
            lambda: mb.ops.dequantize_fp8(z(4, 64, dt=torch.float8_e4m3fn), z(4, 1)),
            lambda: mb.Fp8Matrix(z(64, 64), z(1, 1, dt=torch.float32)),
            lambda: mb.Fp8Matrix(z(64, 60, dt=torch.float8_e4m3fn), z(1, 1, dt=torch.float32)),
            lambda: mb.Fp8Matrix(z(64, 64, dt=torch.float8_e4m3fn), z(2, 1, dt=torch.float32)),
            lambda: mb.Fp8Matrix(z(64, 64, dt=torch.float8_e4m3fn), z(1, 1, dt=torch.float32, dev="cpu")),
        ]
        for i, f in enumerate(bad):
            with pytest.raises(ValueError):
                f()
                pytest.fail(f"call {i} was not refused")
        w = mb.Fp8Matrix.__new__(mb.Fp8Matrix)                       # fake tensors have no address to check
        w.data, w.scale = z(384, 64, dt=torch.float8_e4m3fn), z(3, 1, dt=torch.float32)
        w.out_features, w.in_features = 384, 64
        q = z(4, 64, dt=torch.float8_e4m3fn)
        xs = z(4, 1, dt=torch.float32)
        for f in (lambda: mb.ops.linear_fp8(q, w),                                         # no scale
                  lambda: mb.ops.linear_fp8(z(4, 64), w, x_scale=xs),                       # a scale too many
                  lambda: mb.ops.linear_fp8(z(4, 128), w),
                  lambda: mb.ops.linear_fp8(q, w, x_scale=xs, swiglu=True),                 # 384 is no multiple of 256
                  lambda: mb.ops.linear_fp8(q, w, x_scale=z(4, 2, dt=torch.float32)),
                  lambda: mb.ops.linear_fp8(q, w, x_scale=xs, out_dtype=torch.int32),
                  lambda: mb.ops.linear_fp8(z(4, 64).requires_grad_(), w)):
            with pytest.raises(ValueError):
                f()


def test_registered_operators_trace():
    ns = torch.ops.mortar_b200
    with FakeTensorMode():
        x = torch.empty(6, 5, 64, device="cuda", dtype=torch.bfloat16)
        y, stats = ns.layer_norm(x, None, None, 1e-5)
        assert y.shape == x.shape and stats.shape == (2, 30) and stats.dtype == torch.float32
        y, hidden, sums = ns.mlp_dense(x, x.new_empty(64, 64), x.new_empty(64, 32))
        assert y.shape == x.shape and hidden.shape == (30, 32) and sums.shape == (30, 64)
        q, s = ns.quantize_fp8(x.reshape(30, 64), 128, True)
        assert q.dtype == torch.float8_e5m2 and s.shape == (1, 1)
        assert ns.dequantize_fp8(q, s, torch.float16).dtype == torch.float16
        y = ns.linear_fp8(q, s.new_empty(30, 1), q.new_empty(256, 64), s.new_empty(2, 1), True, torch.float32)
        assert y.shape == (30, 128) and y.dtype == torch.float32


def test_modules_hold_their_parameters():
    m = mb.SwiGLUDense(64, 128, norm=True)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "gate_up.weight": (256, 64), "down.weight": (64, 128), "norm.weight": (64,), "norm.bias": (64,)}
    with pytest.raises(ValueError):
        mb.SwiGLUDense(60, 128)
    q = lambda o, i: mb.Fp8Matrix(torch.zeros(o, i, dtype=torch.float8_e4m3fn), torch.ones(-(-o // 128), -(-i // 128)))
    s = mb.SwiGLUFp8(q(256, 64), q(64, 128))
    assert set(s.state_dict()) == {"gate_up_data", "gate_up_scale", "down_data", "down_scale"}
    with pytest.raises(ValueError):
        mb.SwiGLUFp8(q(192, 64), q(64, 96))                          # 96 hidden columns: no multiple of 128
    with pytest.raises(ValueError):
        mb.SwiGLUFp8(q(256, 64), q(128, 128))


def test_linear_fp8_parts_run_at_once_on_any_device():
    """The kernel that cuts a reduction gives a cluster of two SMs one part of one half tile at most, whatever the number of
    SMs, and the parts fit the scratch that was asked for."""
    n = L.mortar_linear_fp8_parts
    cut = 0
    for rows in (33, 64, 333, 512, 1000, 4000):
        for out in (64, 768, 2048, 2304, 4096):
            for k in (128, 2048, 5632, 16384):
                halves = 2 * -(-rows // 256) * -(-out // 256)
                assert n(rows, out, k, 1, 148) == 1 or out % 256
                for sms in (2, 16, 40, 70, 108, 132, 146, 148, 160):
                    parts = n(rows, out, k, 0, sms)
                    assert 1 <= parts <= -(-k // 128) and (parts == 1 or halves * parts <= sms // 2)
                    need = parts * rows * (-(-out // 32) * 32) if parts > 1 else 0
                    assert need <= L.mortar_linear_fp8_scratch_floats(rows, out, k, 0)
                    cut += parts > 1
                parts = n(rows, out, k, 0, 148)
                assert L.mortar_linear_fp8_scratch_floats(rows, out, k, 0) == (parts * rows * (-(-out // 32) * 32) if parts > 1 else 0)
    assert cut > 100
    assert n(64, 2048, 5632, 0, 148) == 4 and n(512, 2304, 5632, 0, 148) == 2 and n(512, 2304, 5632, 0, 132) == 1
    assert n(64, 2048, 5632, 0, 0) == SHAPE and n(-1, 64, 64, 0, 148) == SHAPE


def test_linear_fp8_scratch():
    n = L.mortar_linear_fp8_scratch_floats
    assert n(64, 2048, 5632, 0) > 0 and n(64, 2048, 5632, 1) == 0
    assert n(4, 2048, 5632, 0) == 0 and n(8192, 2048, 5632, 0) == 0 and n(64, 2048, 256, 0) == 0 and n(0, 2048, 5632, 0) == 0
    assert n(64, 2048, 5630, 0) == SHAPE and n(64, 0, 5632, 0) == SHAPE and n(-1, 64, 64, 0) == SHAPE and n(64, 64, 64, 2) == DTYPE
    keep, p = _buf()
    ok = [p, E4M3, 5632, p, 44, 64, p, E4M3, 5632, p, 44, 2048, 5632, 0, p, BF16, 2048]
    f = L.mortar_linear_fp8_cut
    assert f(*ok[:5], 0, *ok[6:], None, 0, None) == 0
    assert f(None, *ok[1:], None, 0, None) == NULL
    assert f(*ok, _off(p, 16), 1 << 30, None) == ALIGN


def fake_matrix(data, scale):
    """A matrix whose parts were put in place one by one (fake tensors have no address for the constructor)."""
    w = mb.Fp8Matrix.__new__(mb.Fp8Matrix)
    w.data, w.scale = data, scale
    w.out_features, w.in_features = data.shape
    return w


def test_parts_of_a_matrix_whose_rows_overlap_are_refused():
    """Replaced parts whose rows lie over one another (expanded, or a window that moves by less than a row): the kernels
    walk rows of the full width and would read past the end."""
    with FakeTensorMode():
        data, scale = (torch.empty(256, 256, device="cuda", dtype=torch.float8_e4m3fn),
                       torch.empty(2, 2, device="cuda", dtype=torch.float32))
        x = torch.empty(4, 256, device="cuda", dtype=torch.float8_e4m3fn)
        xs = torch.empty(4, 2, device="cuda", dtype=torch.float32)
        for d, s in ((data[:1].expand(256, 256), scale), (data.as_strided((256, 256), (16, 1)), scale),
                     (data, scale[:1].expand(2, 2)), (data, scale.as_strided((2, 2), (1, 1)))):
            with pytest.raises(ValueError, match="overlap"):
                mb.ops.linear_fp8(x, fake_matrix(d, s), x_scale=xs)


def test_matrix_lays_its_scales_out():
    """One column of scales in any stride (a transposed row), and views that stand for the negative of what memory holds."""
    data = torch.zeros(300, 64, dtype=torch.float8_e4m3fn)
    row = torch.tensor([[1.0, 2.0, 3.0]])
    m = mb.Fp8Matrix(data, row.t())
    assert m.scale.stride() == (1, 1) and torch.equal(m.scale, row.t())
    one = torch.as_strided(row, (1, 1), (7, 7))
    assert mb.Fp8Matrix(data[:100], one).scale.stride() == (1, 1)
    m = mb.Fp8Matrix(data, torch._neg_view(row.t().contiguous()))
    assert not m.scale.is_neg() and torch.equal(m.scale, -row.t())
    kept = torch.tensor([[1.0], [2.0], [3.0]])
    assert mb.Fp8Matrix(data, kept).scale is kept                        # nothing is copied without need
    with FakeTensorMode():
        x = torch.empty(4, 64, device="cuda", dtype=torch.float8_e4m3fn)
        xs = torch.empty(4, 1, device="cuda", dtype=torch.float32)
        d, s = torch.empty(300, 64, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(3, 1, device="cuda")
        with pytest.raises(ValueError, match="negative"):
            mb.ops.linear_fp8(x, fake_matrix(d, torch._neg_view(s)), x_scale=xs)


def test_negated_views_of_what_a_forward_call_kept_are_refused():
    with FakeTensorMode():
        def z(*shape, dt=torch.bfloat16):
            return torch.empty(*shape, device="cuda", dtype=dt)
        x, gu, dn, hidden, sums = z(4, 64), z(64, 64), z(64, 32), z(4, 32), z(4, 64, dt=torch.float32)
        neg = torch._neg_view
        for f in (lambda: mb.ops.layer_norm_backward(x, x, None, neg(z(2, 4, dt=torch.float32))),
                  lambda: mb.ops.mlp_dense_backward(x, x, gu, dn, neg(hidden), sums),
                  lambda: mb.ops.mlp_dense_backward(x, x, gu, dn, hidden, neg(sums))):
            with pytest.raises(ValueError, match="must be contiguous"):
                f()


def test_fp8_widths_end_at_2_to_the_30():
    """Wider rows would leave 32 bits where blocks and bytes of a row are counted."""
    keep, p = _buf()
    over = (1 << 30) + 16
    for wide in (over, (1 << 31) - 16):
        for block_rows in (1, 128):
            assert L.mortar_quantize_fp8(p, BF16, wide, 1, wide, block_rows, p, E4M3, wide, p, None) == CAP
            assert L.mortar_dequantize_fp8(p, E4M3, wide, p, 1, wide, block_rows, p, BF16, wide, None) == CAP
        for rows in (1, 20, 200):
            args = [p, E4M3, wide, p, wide // 128 + 1, rows, p, E4M3, wide, p, wide // 128 + 1, 64, wide, 0, p, BF16, 64]
            assert L.mortar_linear_fp8(*args, None) == CAP
            assert L.mortar_linear_fp8_cut(*args, p, 1 << 40, None) == CAP
            assert L.mortar_linear_fp8_scratch_floats(rows, 64, wide, 0) == CAP
    assert L.mortar_quantize_fp8(p, BF16, 1 << 30, 0, 1 << 30, 1, p, E4M3, 1 << 30, p, None) == 0
    assert L.mortar_linear_fp8_scratch_floats(4, 64, 1 << 30, 0) == 0
    with FakeTensorMode():
        x = torch.empty(1, over, device="cuda", dtype=torch.bfloat16)
        for f in (lambda: mb.ops.quantize_fp8(x), lambda: mb.ops.dequantize_fp8(x.to(torch.float8_e4m3fn), x.new_empty(1, (over + 127) // 128, dtype=torch.float32))):
            with pytest.raises(ValueError, match="cols"):
                f()


def test_tangents_are_refused():
    """Forward mode: no operator of the site has such a derivative, and none may drop a tangent in silence, without gradients
    (forward mode stays on under no_grad) or with them."""
    import torch.autograd.forward_ad as fwd
    with FakeTensorMode(), fwd.dual_level():
        def z(*shape, dt=torch.bfloat16, dual=False, grad=False):
            t = torch.empty(*shape, device="cuda", dtype=dt).requires_grad_(grad)
            return fwd.make_dual(t, torch.empty_like(t)) if dual else t
        f32 = dict(dt=torch.float32)
        stats, hidden, sums = z(2, 4, **f32), z(4, 32), z(4, 64, **f32)
        calls = [
            lambda **d: mb.ops.layer_norm(z(4, 64, **d)),
            lambda **d: mb.ops.layer_norm(z(4, 64), z(64, **d)),
            lambda **d: mb.ops.layer_norm(z(4, 64), None, z(64, **d)),
            lambda **d: mb.ops.layer_norm_forward(z(4, 64, **d), None, None, 1e-5, True),
            lambda **d: mb.ops.layer_norm_backward(z(4, 64, **d), z(4, 64), None, stats),
            lambda **d: mb.ops.layer_norm_backward(z(4, 64), z(4, 64), z(64, **d), stats),
            lambda **d: mb.ops.mlp_dense(z(4, 64, **d), z(64, 64), z(64, 32)),
            lambda **d: mb.ops.mlp_dense(z(4, 64), z(64, 64, **d), z(64, 32)),
            lambda **d: mb.ops.mlp_dense(z(4, 64), z(64, 64), z(64, 32, **d)),
            lambda **d: mb.ops.mlp_dense_forward(z(4, 64, **d), z(64, 64), z(64, 32), False),
            lambda **d: mb.ops.mlp_dense_backward(z(4, 64, **d), z(4, 64), z(64, 64), z(64, 32), hidden, sums),
            lambda **d: mb.ops.quantize_fp8(z(4, 64, **d)),
            lambda **d: mb.ops.dequantize_fp8(z(4, 64, dt=torch.float8_e4m3fn), z(4, 1, **f32, **d)),
            lambda **d: mb.ops.linear_fp8(z(4, 64, **d), fake_matrix(z(64, 64, dt=torch.float8_e4m3fn), z(1, 1, **f32))),
            lambda **d: mb.ops.linear_fp8(z(4, 64, dt=torch.float8_e4m3fn), fake_matrix(z(64, 64, dt=torch.float8_e4m3fn), z(1, 1, **f32)),
                                          x_scale=z(4, 1, **f32, **d)),
            lambda **d: mb.ops.linear_fp8(z(4, 64), fake_matrix(z(64, 64, dt=torch.float8_e4m3fn), z(1, 1, **f32, **d))),
            lambda **d: mb.ops.mlp_fp8(z(4, 64, **d), fake_matrix(z(256, 64, dt=torch.float8_e4m3fn), z(2, 1, **f32)),
                                       fake_matrix(z(64, 128, dt=torch.float8_e4m3fn), z(1, 1, **f32))),
        ]
        for i, call in enumerate(calls):
            for mode in (torch.no_grad, torch.enable_grad):
                with mode(), pytest.raises(ValueError, match="forward-mode"):
                    call(dual=True)
                    pytest.fail(f"call {i} was not refused")
        for call in (calls[0], calls[6]):
            with pytest.raises(ValueError, match="forward-mode"):
                call(dual=True, grad=True)


def test_8_bit_operators_refuse_what_requires_a_gradient():
    """One rule for all of them: none records a gradient, so none takes an input that asks for one while they are recorded.
    Under no_grad the call goes on (as far as fake tensors let it: there is no device to launch on)."""
    with FakeTensorMode():
        def z(*shape, dt=torch.float32, grad=False):
            return torch.empty(*shape, device="cuda", dtype=dt).requires_grad_(grad)
        q8 = torch.float8_e4m3fn
        calls = [
            lambda g: mb.ops.quantize_fp8(z(4, 64, grad=g)),
            lambda g: mb.ops.dequantize_fp8(z(4, 64, dt=q8), z(4, 1, grad=g)),
            lambda g: mb.ops.linear_fp8(z(4, 64, grad=g), fake_matrix(z(64, 64, dt=q8), z(1, 1))),
            lambda g: mb.ops.linear_fp8(z(4, 64, dt=q8), fake_matrix(z(64, 64, dt=q8), z(1, 1)), x_scale=z(4, 1, grad=g)),
            lambda g: mb.ops.linear_fp8(z(4, 64), fake_matrix(z(64, 64, dt=q8), z(1, 1, grad=g))),
        ]
        for i, call in enumerate(calls):
            with pytest.raises(ValueError, match="not differentiable"):
                call(True)
                pytest.fail(f"call {i} was not refused")
            if not torch.cuda.is_available():
                with torch.no_grad(), pytest.raises(RuntimeError) as e:
                    call(True)
                assert "not differentiable" not in str(e.value)


@pytest.mark.parametrize("cast", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.float(), lambda m: m.double(),
                                  lambda m: m.to(torch.bfloat16), lambda m: m.to("cpu", torch.float16)])
def test_a_cast_of_the_model_leaves_the_8_bit_form(cast):
    gen = torch.Generator().manual_seed(0)
    def matrix(o, i):
        return mb.Fp8Matrix(torch.randn(o, i, generator=gen).to(torch.float8_e4m3fn),
                            torch.rand(-(-o // 128), -(-i // 128), generator=gen) + 1.0 / 3)
    site = mb.SwiGLUFp8(matrix(256, 64), matrix(64, 128), (torch.ones(64), torch.zeros(64), 1e-5))
    before = {k: v.clone() for k, v in site.state_dict().items()}
    model = cast(torch.nn.Sequential(torch.nn.Linear(64, 64), site))
    for k, v in site.state_dict().items():
        if k.startswith("norm"):                                     # the norm follows the model
            assert v.dtype == model[0].weight.dtype
        else:
            assert v.dtype == before[k].dtype and torch.equal(v.view(torch.uint8), before[k].view(torch.uint8)), k
    mb.Fp8Matrix(site.gate_up_data, site.gate_up_scale)
    moved = site.to("meta")
    assert moved.down_data.is_meta and moved.down_data.dtype == torch.float8_e4m3fn


def test_registered_operators_make_what_is_wanted():
    """The registered block has a form that keeps nothing (served tokens write no sums and take the kernels for few rows), and
    both registered backward operators leave out what is not asked for."""
    ns = torch.ops.mortar_b200
    with FakeTensorMode():
        def z(*shape, dt=torch.bfloat16, grad=False):
            return torch.empty(*shape, device="cuda", dtype=dt).requires_grad_(grad)
        x, gu, dn, col = z(1, 64), z(256, 64), z(64, 128), z(64)
        y, hidden, sums = ns.mlp_dense(x, gu, dn, False)
        assert y.shape == (1, 64) and hidden.numel() == 0 and sums.numel() == 0
        assert hidden.dtype == torch.bfloat16 and sums.dtype == torch.float32
        with pytest.raises(ValueError, match="want_saved"):
            ns.mlp_dense(z(1, 64, grad=True), gu, dn, False)
        _, hidden, sums = ns.mlp_dense(x, gu, dn)
        stats = z(2, 1, dt=torch.float32)
        for want in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, True, True)):
            got = ns.mlp_dense_backward(x, x, gu, dn, hidden, sums, *want)
            assert [g.shape for g in got] == [t.shape if w else (0,) for t, w in zip((x, gu, dn), want)]
            got = ns.layer_norm_backward(x, x, col, stats, *want)
            assert [g.shape for g in got] == [t.shape if w else (0,) for t, w in zip((x, col, col), want)]


def test_the_site_compiles_into_one_graph():
    """torch.compile(fullgraph=True) of the modules and the operators traces to the registered operators: with the sums kept
    where a gradient is wanted, without them where none is."""
    graphs = []

    def backend(module, _):
        graphs.append([n for n in module.graph.nodes if str(n.target).startswith("mortar_b200.")])
        return module.forward

    def traced(f, *args):
        torch._dynamo.reset()
        graphs.clear()
        y = torch.compile(f, backend=backend, fullgraph=True)(*args)
        assert len(graphs) == 1
        return y, [str(n.target).split(".")[1] for n in graphs[0]]

    with FakeTensorMode():
        def z(*shape, dt=torch.bfloat16):
            return torch.empty(*shape, device="cuda", dtype=dt)
        def matrix(o, i):
            return fake_matrix(z(o, i, dt=torch.float8_e4m3fn), z(-(-o // 128), -(-i // 128), dt=torch.float32))
        site, x = mb.SwiGLUDense(64, 128, norm=True, device="cuda", dtype=torch.bfloat16), z(4, 64)
        y, names = traced(site, x)
        assert names == ["layer_norm", "mlp_dense"] and graphs[0][1].args[3] is True and y.requires_grad and y.shape == x.shape
        y, names = traced(torch.no_grad()(site.forward), x)
        assert names == ["layer_norm", "mlp_dense"] and graphs[0][1].args[3] is False and not y.requires_grad
        gate_up, down = matrix(256, 64), matrix(64, 128)
        served = mb.SwiGLUFp8(gate_up, down, (z(64), z(64), 1e-5))
        y, names = traced(served, x)
        assert names == ["layer_norm", "linear_fp8", "linear_fp8"] and y.shape == x.shape and y.dtype == x.dtype
        y, names = traced(lambda t: mb.ops.mlp_fp8(t, gate_up, down, out_dtype=torch.float32), x)
        assert names == ["linear_fp8", "linear_fp8"] and y.dtype == torch.float32
        def quantised(t):
            q, s = mb.ops.quantize_fp8(t, block_rows=1, dtype=torch.float8_e5m2)
            return mb.ops.linear_fp8(q, gate_up, x_scale=s, swiglu=True), mb.ops.dequantize_fp8(q, s, out_dtype=torch.float16)
        (y, back), names = traced(quantised, x)
        assert sorted(names) == ["dequantize_fp8", "linear_fp8", "quantize_fp8"]
        assert y.shape == (4, 128) and y.dtype == torch.bfloat16 and back.dtype == torch.float16
    torch._dynamo.reset()
