"""What the orthogonalised updates and the 4-bit weights refuse: host logic, on made-up addresses (nothing is
launched, no GPU is needed)."""
import ctypes

import numpy as np
import pytest

i64, f32, P = ctypes.c_int64, ctypes.c_float, ctypes.c_void_p
A, B, C, W = (P(n << 20) for n in (1, 2, 3, 4))
INVALID, LIMIT = 1, 5
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def L():
    import ctorch_b200 as cb
    return cb.load()


def ortho(L, g=A, ldg=8, out=B, ldo=8, rows=4, cols=8, steps=5, eps=1e-7, ws=W):
    return L.ctk_orthogonalize_f32(g, i64(ldg), out, i64(ldo), i64(rows), i64(cols), steps, f32(eps), ws, None)


def muon(L, p=A, ldp=8, g=B, ldg=8, m=C, ldm=8, rows=4, cols=8, steps=5, eps=1e-7, ws=W):
    return L.ctk_muon_update_f32(p, i64(ldp), g, i64(ldg), m, i64(ldm), i64(rows), i64(cols), f32(0.1), f32(0.9), 1, f32(0), f32(1), steps, f32(eps), ws, None)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(cols=-1), dict(steps=0), dict(steps=65), dict(eps=0.0), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF),
                                 dict(ldg=7), dict(g=None), dict(ws=P((4 << 20) + 16)), dict(g=P((1 << 20) + 2))])
def test_updates_refuse(L, bad):
    assert ortho(L, **bad) == INVALID
    assert muon(L, **bad) == INVALID
    assert L.ctk_last_error()


@pytest.mark.parametrize("bad", [dict(ldo=7), dict(out=None), dict(out=P((2 << 20) + 1))])
def test_orthogonalize_refuses(L, bad):
    assert ortho(L, **bad) == INVALID


@pytest.mark.parametrize("bad", [dict(ldp=7), dict(ldm=7), dict(p=None), dict(m=None), dict(p=B), dict(m=B), dict(p=C), dict(m=P((3 << 20) + 3)),
                                 # ranges that overlap without starting at the same address
                                 dict(p=P((2 << 20) + 32)), dict(m=P((1 << 20) + 64)), dict(g=P((3 << 20) - 16))])
def test_muon_update_refuses(L, bad):
    assert muon(L, **bad) == INVALID


def test_orthogonalize_refuses_overlaps(L):
    assert ortho(L, out=P((1 << 20) + 32)) == INVALID
    assert ortho(L, out=A, ldo=9) == INVALID               # in place needs the same pitch


def test_updates_size_limits(L):
    assert ortho(L, rows=1 << 16, cols=1 << 15, ldg=1 << 15, ldo=1 << 15) == LIMIT
    assert ortho(L, rows=1 << 40, cols=1 << 40, ldg=1 << 40, ldo=1 << 40) == LIMIT
    assert muon(L, rows=(1 << 30) + 1, cols=1, ldp=1, ldg=1, ldm=1) == LIMIT
    assert ortho(L, rows=0) == 0 and ortho(L, cols=0) == 0 and muon(L, rows=0) == 0
    assert L.ctk_orthogonalize_workspace_bytes(i64(0), i64(4)) == 0 and L.ctk_orthogonalize_workspace_bytes(i64(-1), i64(4)) == 0
    assert L.ctk_orthogonalize_workspace_bytes(i64(64), i64(64)) > 0


def quant(L, w=A, ldw=8, k=64, n=8, group=32, packed=B, scales=C, zeros=None):
    return L.ctk_w4_quantize_f32(w, i64(ldw), i64(k), i64(n), group, packed, scales, zeros, None)


def dequant(L, w=A, ldw=8, k=64, n=8, group=32, packed=B, scales=C, zeros=None):
    return L.ctk_w4_dequantize_f32(packed, scales, zeros, i64(k), i64(n), group, w, i64(ldw), None)


def product(L, x=A, ldx=64, k=64, n=8, m=2, group=32, packed=B, scales=C, y=W, ldy=8):
    return L.ctk_w4_matmul_f32(x, i64(ldx), packed, scales, None, None, 0, y, i64(ldy), i64(m), i64(k), i64(n), group, None)


@pytest.mark.parametrize("bad", [dict(k=-1), dict(n=-1), dict(group=0), dict(group=16), dict(group=48), dict(group=256), dict(ldw=7), dict(w=None), dict(packed=None),
                                 dict(scales=None), dict(packed=P((2 << 20) + 4)), dict(w=P((1 << 20) + 1)), dict(scales=P((3 << 20) + 2))])
def test_quantize_and_dequantize_refuse(L, bad):
    assert quant(L, **bad) == INVALID
    assert dequant(L, **bad) == INVALID


@pytest.mark.parametrize("bad", [dict(k=-1), dict(n=-1), dict(m=-1), dict(group=0), dict(group=96), dict(ldx=63), dict(ldy=7), dict(x=None), dict(packed=None),
                                 dict(scales=None), dict(y=None), dict(packed=P((2 << 20) + 8)), dict(x=P((1 << 20) + 2)), dict(y=P((4 << 20) + 3)),
                                 dict(y=P((1 << 20) + 256))])
def test_w4_product_refuses(L, bad):
    assert product(L, **bad) == INVALID


def test_w4_size_limits_and_empty(L):
    big = (1 << 30) + 1
    assert quant(L, n=big, ldw=big) == LIMIT and dequant(L, k=big) == LIMIT and product(L, k=big, ldx=big) == LIMIT and product(L, m=big) == LIMIT
    assert quant(L, n=0) == 0 and quant(L, k=0) == 0 and dequant(L, k=0) == 0 and product(L, m=0) == 0 and product(L, n=0) == 0
    assert L.ctk_w4_packed_bytes(i64(129), i64(10), 128) == 2 * 64 * 10
    assert L.ctk_w4_packed_bytes(i64(5), i64(3), 40) == 0 and L.ctk_w4_packed_bytes(i64(-5), i64(3), 32) == 0


def test_python_face_checks_shapes():
    import ctorch_b200 as cb

    def fake(shape, dtype=np.float32):
        return cb.DeviceArray(shape, dtype, _ptr=1 << 20)

    with pytest.raises(ValueError):
        cb.ops.orthogonalize(fake((8,)))
    with pytest.raises(ValueError):
        cb.ops.orthogonalize(fake((8, 4)), out=fake((4, 8)))
    with pytest.raises(ValueError):
        cb.ops.muon_update(fake((8, 4)), fake((8, 4)), fake((4, 8)), lr=0.1)
    with pytest.raises(ValueError):
        cb.ops.W4Weight(fake((8, 4), np.uint32), fake((8, 1)), None, 33, 8, 32)
    with pytest.raises(ValueError):
        cb.ops.W4Weight.empty(8, 8, group=20)
    w = cb.ops.W4Weight(fake((8, 4), np.uint32), fake((8, 1)), None, 32, 8, 32)
    with pytest.raises(ValueError):
        cb.ops.matmul_w4(fake((2, 31)), w)
    with pytest.raises(ValueError):
        cb.ops.matmul_w4(fake((2, 32)), w, bias=fake((7,)))
    with pytest.raises(ValueError):
        cb.ops.matmul_w4(fake((2, 32)), w, out=fake((2, 9)))
    with pytest.raises(ValueError):
        cb.ops.w4_quantize(fake((32, 8)), group=32, symmetric=False, out=w)
    with pytest.raises(ValueError):
        cb.ops.w4_dequantize(w, out=fake((8, 32)))


def test_front_end_refuses_host_tensors():
    from ctorch_b200 import frontend as F
    F.set_quiet(True)
    t = F.Tensor.from_numpy(np.ones((4, 8), np.float32), device=F.CPU)
    for call in (lambda: t.orthogonalize(), lambda: t.muon_update_(t, t.copy(), 0.1), lambda: F.W4Weight(t)):
        with pytest.raises(F.FrontendError):
            call()


def test_columns_of_one_buffer_must_not_cross(L):
    # 8 columns from column 0, 8 more from column 7 or (round the row's end) from column 13 of rows of 20
    assert ortho(L, ldg=20, ldo=20, out=P((1 << 20) + 4 * 7)) == INVALID
    assert ortho(L, ldg=20, ldo=20, out=P((1 << 20) + 4 * 13)) == INVALID
    assert ortho(L, ldg=20, ldo=21, out=P((1 << 20) + 4 * 10)) == INVALID  # different pitches: not side by side throughout
    assert product(L, ldx=80, ldy=80, y=P((1 << 20) + 4 * 60)) == INVALID
    assert product(L, ldx=80, ldy=80, y=P((1 << 20) + 4 * 75)) == INVALID


def test_python_face_checks_types_and_workspace():
    import ctorch_b200 as cb

    def fake(shape, dtype=np.float32):
        return cb.DeviceArray(shape, dtype, _ptr=1 << 20)

    g, d = fake((300, 200)), fake((300, 200), np.float64)
    small = fake((1024,), np.uint8)
    for call in (lambda: cb.ops.orthogonalize(d), lambda: cb.ops.orthogonalize(g, out=d), lambda: cb.ops.muon_update(g, d, g, lr=0.1),
                 lambda: cb.ops.muon_update(g, g, d, lr=0.1), lambda: cb.ops.orthogonalize(g, out=g, workspace=small),
                 lambda: cb.ops.muon_update(g, g, g, lr=0.1, workspace=small), lambda: cb.ops.w4_quantize(d, group=32),
                 lambda: cb.ops.W4Weight(fake((8, 4)), fake((8, 1)), None, 32, 8, 32),
                 lambda: cb.ops.W4Weight(fake((8, 4), np.uint32), fake((8, 1), np.float64), None, 32, 8, 32),
                 lambda: cb.ops.W4Weight(fake((8, 4), np.uint32), fake((8, 1)), fake((8, 1)), 32, 8, 32)):
        with pytest.raises(ValueError):
            call()
    w = cb.ops.W4Weight(fake((8, 4), np.uint32), fake((8, 1)), None, 32, 8, 32)
    for call in (lambda: cb.ops.matmul_w4(fake((2, 32), np.float64), w), lambda: cb.ops.matmul_w4(fake((2, 32)), w, bias=fake((8,), np.float64)),
                 lambda: cb.ops.matmul_w4(fake((2, 32)), w, out=fake((2, 8), np.float64)), lambda: cb.ops.w4_dequantize(w, out=fake((32, 8), np.float64))):
        with pytest.raises(ValueError):
            call()
