"""4-bit calls whose arrays lie in one buffer without overlapping, and one row added to what y holds."""
import ctypes

import numpy as np
import pytest

from test_gpu_w4 import random_weight

pytestmark = pytest.mark.gpu

i64 = ctypes.c_int64


@pytest.mark.parametrize("k,n", [(40, 30), (1000, 500)])
def test_one_row_added_to_y(cb, k, n):
    rng = np.random.default_rng(k)
    w4, _ = random_weight(cb, rng, k, n, 32, False)
    x, b = rng.standard_normal((1, k)).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    want = cb.ops.matmul_w4(cb.to_device(x), w4, bias=cb.to_device(b)).numpy()
    y = cb.to_device(b[None])
    cb.ops.matmul_w4(cb.to_device(x), w4, bias=y, out=y)
    assert np.array_equal(y.numpy(), want)


def test_bias_in_the_gap_between_the_rows_of_y(cb):
    rng = np.random.default_rng(3)
    m, k, n, ld = 4, 100, 20, 44
    w4, _ = random_weight(cb, rng, k, n, 32, True)
    x = rng.standard_normal((m, k)).astype(np.float32)
    host = rng.standard_normal((m, ld)).astype(np.float32)
    want = cb.ops.matmul_w4(cb.to_device(x), w4, bias=cb.to_device(host[1, 22:42])).numpy()
    dx, buf = cb.to_device(x), cb.to_device(host)
    cb.check(cb.lib.ctk_w4_matmul_f32(dx.p, i64(k), w4.packed.p, w4.scales.p, None, buf.view(ld + 22, (n,)).p, 0, buf.p, i64(ld), i64(m), i64(k), i64(n), 32, None))
    got = buf.numpy()
    assert np.array_equal(got[:, :n], want) and np.array_equal(got[:, n:], host[:, n:])
