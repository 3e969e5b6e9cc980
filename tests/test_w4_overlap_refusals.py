"""Arrays of the 4-bit calls that share memory are refused: host logic, on made-up addresses (nothing is launched)."""
import ctypes

import pytest

i64, P = ctypes.c_int64, ctypes.c_void_p
M = 1 << 20
INVALID = 1


@pytest.fixture(scope="module")
def L():
    import ctorch_b200 as cb
    return cb.load()


# k 64, n 8, group 32: packed 8 x 8 words = 256 bytes, scales 8 x 2 floats = 64 bytes, zeros 16 bytes
def product(L, x=M, ldx=64, packed=2 * M, scales=3 * M, zeros=5 * M, bias=6 * M, y=4 * M, ldy=8, m=2):
    return L.ctk_w4_matmul_f32(P(x), i64(ldx), P(packed), P(scales), P(zeros), P(bias), 0, P(y), i64(ldy), i64(m), i64(64), i64(8), 32, None)


def quant(L, w=M, ldw=8, packed=2 * M, scales=3 * M, zeros=5 * M):
    return L.ctk_w4_quantize_f32(P(w), i64(ldw), i64(64), i64(8), 32, P(packed), P(scales), P(zeros), None)


def dequant(L, w=M, ldw=8, packed=2 * M, scales=3 * M, zeros=5 * M):
    return L.ctk_w4_dequantize_f32(P(packed), P(scales), P(zeros), i64(64), i64(8), 32, P(w), i64(ldw), None)


@pytest.mark.parametrize("bad", [dict(packed=4 * M), dict(packed=4 * M + 48), dict(packed=4 * M - 240), dict(scales=4 * M + 60), dict(scales=4 * M - 60), dict(zeros=4 * M + 63),
                                 dict(zeros=4 * M - 15), dict(bias=4 * M), dict(bias=4 * M + 32), dict(bias=4 * M - 28), dict(bias=4 * M + 4, m=1), dict(bias=4 * M - 4, m=1),
                                 # rows of y 80 bytes apart: from the gap behind the first into the second
                                 dict(ldy=20, bias=4 * M + 52), dict(ldy=20, zeros=4 * M + 70), dict(ldy=20, packed=4 * M + 32)])
def test_product(L, bad):
    assert product(L, **bad) == INVALID


@pytest.mark.parametrize("bad", [dict(packed=M), dict(packed=M + 2032), dict(scales=M + 1020), dict(scales=M - 60), dict(zeros=M + 2047), dict(zeros=M - 15), dict(ldw=20, zeros=M + 80 * 3 + 66)])
def test_quantize_and_dequantize(L, bad):
    assert quant(L, **bad) == INVALID
    assert dequant(L, **bad) == INVALID
