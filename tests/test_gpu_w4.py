"""4-bit weights: quantising (exactly, by its definition), the values they stand for, and the product with a
few rows, against 64 bits.

Tolerance of the product.  Codes are exact, so every term x (code - zero) is; a sum of a group takes at most
`group` fp32 additions on any path, the scaled groups are added in at most `groups` more, and a further 40 cover the joining
of partial sums, the scale, the bias and x's own representation.  The tensor cores truncate (2^-23 a step), fp32
additions round (2^-24): |y - ref| <= (group + groups + 40) 2^-23 sum |x| |w| (+ the bias)."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

i64 = ctypes.c_int64
SHIFT = np.array([0, 16, 4, 20, 8, 24, 12, 28], np.uint32)


def quantize64(w, group, symmetric):
    """codes [n, groups, group], scales, zeros by the definition."""
    k, n = w.shape
    groups = -(-k // group)
    v = np.zeros((n, groups * group), np.float64)
    v[:, :k] = w.T
    v = v.reshape(n, groups, group)
    if symmetric:
        s = (np.abs(v).max(-1) / 7.0).astype(np.float32)
        zero = np.full(s.shape, 8.0)
    else:
        lo = np.minimum(v.min(-1), 0)
        s = ((np.maximum(v.max(-1), 0) - lo) / 15.0).astype(np.float32)
        zero = np.where(s > 0, np.rint(-lo / np.where(s > 0, s, 1).astype(np.float64)), 0)
    q = np.where(s[..., None] > 0, np.rint(v / np.where(s > 0, s, 1).astype(np.float64)[..., None]), 0)
    return np.clip(q + zero[..., None], 1 if symmetric else 0, 15).astype(np.uint32), s, None if symmetric else zero.astype(np.uint8)


def pack(codes):
    c = codes.reshape(codes.shape[0], -1, 8)
    return np.bitwise_or.reduce(c << SHIFT, axis=-1).astype(np.uint32)


def unpack(packed):
    return ((packed[:, :, None] >> SHIFT) & 15).reshape(packed.shape[0], -1)


def values64(packed, scales, zeros, k, group):
    q = unpack(packed).astype(np.float64).reshape(packed.shape[0], -1, group)
    z = 8.0 if zeros is None else zeros.astype(np.float64)[..., None]
    return ((q - z) * scales.astype(np.float64)[..., None]).reshape(packed.shape[0], -1)[:, :k].T


def random_weight(cb, rng, k, n, group, symmetric):
    groups = -(-k // group)
    packed = rng.integers(0, 2 ** 32, (n, groups * group // 8), dtype=np.uint64).astype(np.uint32)
    scales = rng.uniform(0.5, 1.5, (n, groups)).astype(np.float32)
    zeros = None if symmetric else rng.integers(0, 16, (n, groups)).astype(np.uint8)
    dev = cb.ops.W4Weight(cb.to_device(packed, np.uint32), cb.to_device(scales), None if symmetric else cb.to_device(zeros, np.uint8), k, n, group)
    return dev, values64(packed, scales, zeros, k, group)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("k,n", [(1, 1), (31, 5), (32, 32), (33, 7), (128, 100), (129, 33), (784, 128), (1001, 517), (300, 1), (4096, 64)])
def test_quantize_and_dequantize(cb, k, n, group, symmetric):
    rng = np.random.default_rng(k * 31 + n + group)
    w = rng.standard_normal((k, n)).astype(np.float32)
    w[:, n // 2] = np.rint(w[:, n // 2] * 8)           # many ties
    if k > 2 * group:
        w[group:2 * group, 0] = 0.0                    # a group of zeros
        w[:group, n - 1] = np.abs(w[:group, n - 1])    # one sign only
    codes, s, z = quantize64(w, group, symmetric)
    q = cb.ops.w4_quantize(cb.to_device(w), group=group, symmetric=symmetric)
    assert np.array_equal(q.scales.numpy(), s)
    if z is not None:
        assert np.array_equal(q.zeros.numpy(), z)
    assert np.array_equal(q.packed.numpy(), pack(codes))
    got = cb.ops.w4_dequantize(q).numpy()
    want = values64(q.packed.numpy(), s, z, k, group)
    assert np.array_equal(got, want.astype(np.float32))     # an integer times an fp32 scale, rounded once


def test_quantize_extreme_magnitudes(cb):
    rng = np.random.default_rng(4)
    for factor in (1e-45, 1e-42, 1e-38, 1e-30, 1e30, 1e38):
        w = (rng.uniform(-3, 3, (70, 9)) * factor).astype(np.float32)
        q = cb.ops.w4_quantize(cb.to_device(w), group=64)
        codes, s, _ = quantize64(w, 64, True)
        assert np.array_equal(q.scales.numpy(), s) and np.array_equal(q.packed.numpy(), pack(codes)), factor


@pytest.mark.parametrize("symmetric", [True, False])
def test_quantize_non_finite_poisons_its_group_only(cb, symmetric):
    w = np.random.default_rng(0).standard_normal((96, 6)).astype(np.float32)
    w[40, 2], w[3, 4] = np.nan, -np.inf
    q = cb.ops.w4_quantize(cb.to_device(w), group=32, symmetric=symmetric)
    bad = np.isnan(q.scales.numpy())
    assert bad.sum() == 2 and bad[2, 1] and bad[4, 0]
    v = cb.ops.w4_dequantize(q).numpy()
    assert np.isnan(v[32:64, 2]).all() and np.isnan(v[:32, 4]).all() and np.isnan(v).sum() == 64
    y = cb.ops.matmul_w4(cb.to_device(np.ones((1, 96), np.float32)), q).numpy()
    assert np.isnan(y[0, [2, 4]]).all() and np.isfinite(y[0, [0, 1, 3, 5]]).all()


SHAPES = [(1, 1, 1), (1, 32, 8), (1, 33, 17), (2, 128, 16), (3, 1001, 517), (1, 784, 128), (1, 128, 10), (4, 300, 65), (5, 4096, 48), (7, 513, 129),
          (8, 256, 256), (9, 640, 40), (16, 1000, 100), (17, 333, 64), (33, 512, 72), (64, 777, 130), (65, 260, 50), (130, 384, 200), (1, 20000, 9), (2, 5, 3000), (20, 2000, 300), (24, 1100, 129), (48, 4096, 64)]


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_matmul_w4(cb, m, k, n, group, symmetric):
    rng = np.random.default_rng(m * 1009 + k * 31 + n + group)
    w4, w = random_weight(cb, rng, k, n, group, symmetric)
    x = rng.standard_normal((m, k)).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32)
    dx, db = cb.to_device(x), cb.to_device(b)
    bound = (group + -(-k // group) + 40) * 2.0 ** -23 * (np.abs(x).astype(np.float64) @ np.abs(w) + np.abs(b)) + 1e-37
    want = x.astype(np.float64) @ w
    got = cb.ops.matmul_w4(dx, w4).numpy()
    assert (np.abs(got - want) <= bound).all()
    relu = cb.ops.matmul_w4(dx, w4, bias=db, relu=True).numpy()
    assert (np.abs(relu - np.maximum(want + b, 0)) <= bound).all()
    assert np.array_equal(cb.ops.matmul_w4(dx, w4).numpy(), got)           # the same bits again
    assert cb.ops.w4_status() == 0


@pytest.mark.parametrize("factor", [1e-30, 1e-6, 1e6, 1e30])
def test_matmul_w4_any_magnitude_of_x(cb, factor):
    rng = np.random.default_rng(8)
    w4, w = random_weight(cb, rng, 300, 40, 32, True)
    x = (rng.standard_normal((3, 300)) * factor).astype(np.float32)
    bound = (32 + 10 + 40) * 2.0 ** -23 * (np.abs(x).astype(np.float64) @ np.abs(w))
    assert (np.abs(cb.ops.matmul_w4(cb.to_device(x), w4).numpy() - x.astype(np.float64) @ w) <= bound).all()


def test_matmul_w4_non_finite_x_stays_in_its_row(cb):
    rng = np.random.default_rng(6)
    w4, w = random_weight(cb, rng, 200, 50, 64, False)
    x = rng.standard_normal((5, 200)).astype(np.float32)
    clean = cb.ops.matmul_w4(cb.to_device(x), w4).numpy()
    for bad in (np.nan, np.inf):
        h = x.copy()
        h[3, 77] = bad
        y = cb.ops.matmul_w4(cb.to_device(h), w4).numpy()
        assert np.array_equal(np.delete(y, 3, 0), np.delete(clean, 3, 0))
        assert not np.isfinite(y[3][w[77] != 0]).any()


def test_matmul_w4_rows_do_not_depend_on_the_batch(cb):
    """Row r of a batch of up to 8 rows has the bits it has alone."""
    rng = np.random.default_rng(12)
    w4, _ = random_weight(cb, rng, 700, 90, 128, True)
    x = rng.standard_normal((2, 700)).astype(np.float32)
    both = cb.ops.matmul_w4(cb.to_device(x), w4).numpy()
    for r in range(2):
        assert np.allclose(cb.ops.matmul_w4(cb.to_device(x[r:r + 1]), w4).numpy()[0], both[r], rtol=1e-5, atol=1e-5)


def test_matmul_w4_one_dimensional_x_and_pitches(cb):
    rng = np.random.default_rng(3)
    m, k, n, ldx, ldy = 3, 130, 45, 141, 50
    w4, w = random_weight(cb, rng, k, n, 64, False)
    host = rng.standard_normal(m * ldx + 1).astype(np.float32)
    x = host[1:].reshape(m, ldx)
    dx = cb.to_device(host)
    y = cb.to_device(np.full(m * ldy + 1, 9.0, np.float32))
    cb.check(cb.lib.ctk_w4_matmul_f32(dx.view(1, (m, ldx)).p, i64(ldx), w4.packed.p, w4.scales.p, w4.zeros.p, None, 0, y.view(1, (m, ldy)).p, i64(ldy), i64(m),
                                      i64(k), i64(n), 64, None))
    got = y.numpy()
    out = got[1:].reshape(m, ldy)
    bound = (64 + 3 + 40) * 2.0 ** -23 * (np.abs(x[:, :k]).astype(np.float64) @ np.abs(w))
    assert (np.abs(out[:, :n] - x[:, :k].astype(np.float64) @ w) <= bound).all()
    assert got[0] == 9.0 and (out[:, n:] == 9.0).all()
    one = cb.ops.matmul_w4(cb.to_device(x[1, :k]), w4)
    assert one.shape == (n,)
    assert (np.abs(one.numpy() - x[1, :k].astype(np.float64) @ w) <= bound[1]).all()


def test_matmul_w4_empty(cb):
    rng = np.random.default_rng(3)
    w4, _ = random_weight(cb, rng, 40, 6, 32, True)
    assert cb.ops.matmul_w4(cb.empty((0, 40)), w4).shape == (0, 6)
    none = cb.ops.W4Weight(cb.empty((6, 0), np.uint32), cb.empty((6, 0)), None, 0, 6, 32)      # no inputs: the bias
    b = rng.standard_normal(6).astype(np.float32)
    got = cb.ops.matmul_w4(cb.empty((2, 0)), none, bias=cb.to_device(b), relu=True).numpy()
    assert np.array_equal(got, np.tile(np.maximum(b, 0), (2, 1)))


@pytest.mark.parametrize("m", [1, 6, 40])
def test_matmul_w4_streams_and_replay(cb, m):
    rng = np.random.default_rng(14)
    w4, _ = random_weight(cb, rng, 900, 300, 128, False)
    xs = [rng.standard_normal((m, 900)).astype(np.float32) for _ in range(3)]
    want = [cb.ops.matmul_w4(cb.to_device(x), w4).numpy() for x in xs]
    s = cb.Stream()
    x, y = cb.to_device(xs[0]), cb.empty((m, 300))
    cb.synchronize()
    cb.check(cb.lib.ctk_stream_begin_capture(s.handle))
    cb.ops.matmul_w4(x, w4, out=y, stream=s)
    exe = ctypes.c_void_p()
    cb.check(cb.lib.ctk_stream_end_capture(s.handle, ctypes.byref(exe)))
    for h, ref in zip(xs, want):
        x.copy_from_host(h)
        cb.check(cb.lib.ctk_graph_launch(exe, s.handle, 0))
        assert np.array_equal(y.numpy(stream=s), ref)
    cb.check(cb.lib.ctk_graph_destroy(exe))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 3, 7, 12, 30])
def test_matmul_w4_whole_numbers_are_exact(cb, m, group):
    """Whole-number x, scales of 1: every sum stays below 2^24, so nothing may round."""
    rng = np.random.default_rng(m + group)
    k, n = 1000, 200
    w4, _ = random_weight(cb, rng, k, n, group, False)
    w4.scales.copy_from_host(np.ones((n, -(-k // group)), np.float32))
    w = values64(w4.packed.numpy(), w4.scales.numpy(), w4.zeros.numpy(), k, group)
    x = rng.integers(-999, 1000, (m, k)).astype(np.float32)
    assert (np.abs(x.astype(np.float64)) @ np.abs(w)).max() < 2 ** 24
    assert np.array_equal(cb.ops.matmul_w4(cb.to_device(x), w4).numpy(), x.astype(np.float64) @ w)


def test_matmul_w4_one_row_of_many_sizes(cb):
    """A row with elements of very different sizes: each block of 128 k is taken to 38 bits below its largest."""
    rng = np.random.default_rng(55)
    k, n = 512, 70
    w4, w = random_weight(cb, rng, k, n, 64, False)
    x = (rng.standard_normal((2, k)) * 10.0 ** rng.integers(-6, 6, (2, k))).astype(np.float32)
    largest = np.abs(x).reshape(2, -1, 128).max(-1).repeat(128, axis=1).astype(np.float64)
    bound = (64 + 8 + 40) * 2.0 ** -23 * (np.abs(x).astype(np.float64) @ np.abs(w)) + 2.0 ** -31 * (largest @ np.abs(w))
    assert (np.abs(cb.ops.matmul_w4(cb.to_device(x), w4).numpy() - x.astype(np.float64) @ w) <= bound).all()


def test_matmul_w4_more_rows_than_one_launch_takes(cb):
    rng = np.random.default_rng(91)
    w4, w = random_weight(cb, rng, 40, 8, 32, False)
    x = rng.standard_normal((140001, 40)).astype(np.float32)
    bound = (32 + 2 + 40) * 2.0 ** -23 * (np.abs(x).astype(np.float64) @ np.abs(w))
    assert (np.abs(cb.ops.matmul_w4(cb.to_device(x), w4).numpy() - x.astype(np.float64) @ w) <= bound).all()


@pytest.mark.parametrize("m", [1, 3, 12])
def test_matmul_w4_outliers_where_the_weight_is_zero(cb, m):
    """Single elements of x a million times the others: columns whose weight is zero there keep what the others give.  x enters
    within 2^-38 of the largest of its 128 neighbours, which adds that much per unit of weight to the tolerance."""
    rng = np.random.default_rng(40 + m)
    k, n, group = 640, 300, 64
    packed = pack(rng.integers(0, 16, (n, k)))
    codes = unpack(packed).reshape(n, k)
    codes[:, 5::128] = 8                                                # zero of the symmetric form
    packed = pack(codes)
    scales = rng.uniform(0.5, 1.5, (n, k // group)).astype(np.float32)
    w = values64(packed, scales, None, k, group)
    x = rng.standard_normal((m, k)).astype(np.float32)
    x[:, 5::128] *= 1e6
    w4 = cb.ops.W4Weight(cb.to_device(packed, np.uint32), cb.to_device(scales), None, k, n, group)
    y = cb.ops.matmul_w4(cb.to_device(x), w4).numpy()
    top = np.abs(x).reshape(m, -1, 128).max(axis=2).repeat(128, axis=1).astype(np.float64)
    bound = (group + k // group + 40) * 2.0 ** -23 * (np.abs(x).astype(np.float64) @ np.abs(w)) + 2.0 ** -38 * (top @ np.abs(w))
    assert (np.abs(y - x.astype(np.float64) @ w) <= bound).all()


def test_matmul_w4_input_and_result_in_one_buffer(cb):
    """x and y as columns of one buffer, side by side in its rows."""
    rng = np.random.default_rng(8)
    m, k, n, ld = 5, 96, 40, 140
    w4, w = random_weight(cb, rng, k, n, 32, True)
    host = rng.standard_normal((m, ld)).astype(np.float32)
    want = cb.ops.matmul_w4(cb.to_device(host[:, :k]), w4).numpy()
    for at_x, at_y in ((0, k), (n + 4, 0)):
        buf = cb.to_device(host)
        if at_x:
            host2 = host.copy()
            host2[:, at_x:at_x + k] = host[:, :k]
            buf = cb.to_device(host2)
        before = buf.numpy()
        cb.check(cb.lib.ctk_w4_matmul_f32(buf.view(at_x, (1,)).p, i64(ld), w4.packed.p, w4.scales.p, None, None, 0, buf.view(at_y, (1,)).p, i64(ld), i64(m), i64(k),
                                          i64(n), 32, None))
        after = buf.numpy()
        assert np.array_equal(after[:, at_y:at_y + n], want)
        keep = np.ones(ld, bool)
        keep[at_y:at_y + n] = False
        assert np.array_equal(after[:, keep], before[:, keep])


@pytest.mark.parametrize("group", [32, 128])
def test_scales_and_zeros_at_odd_addresses(cb, group):
    """Scales 4 bytes and zero points 1 byte past an aligned address: the same bits, nothing around them written."""
    rng = np.random.default_rng(group)
    k, n, m = 4 * group, 150, 3
    groups = k // group
    w = cb.to_device(rng.standard_normal((k, n)).astype(np.float32))
    want = cb.ops.w4_quantize(w, group=group, symmetric=False)
    scales = cb.to_device(np.full(n * groups + 2, -1.0, np.float32))
    zeros = cb.to_device(np.full(n * groups + 2, 77, np.uint8), np.uint8)
    odd = cb.ops.W4Weight(cb.empty((n, k // 8), np.uint32), scales.view(1, (n, groups)), zeros.view(1, (n, groups)), k, n, group)
    cb.ops.w4_quantize(w, group=group, symmetric=False, out=odd)
    assert np.array_equal(odd.packed.numpy(), want.packed.numpy())
    s, z = scales.numpy(), zeros.numpy()
    assert np.array_equal(s[1:-1].reshape(n, groups), want.scales.numpy()) and s[0] == -1.0 and s[-1] == -1.0
    assert np.array_equal(z[1:-1].reshape(n, groups), want.zeros.numpy()) and z[0] == 77 and z[-1] == 77
    x = cb.to_device(rng.standard_normal((m, k)).astype(np.float32))
    assert np.array_equal(cb.ops.w4_dequantize(odd).numpy(), cb.ops.w4_dequantize(want).numpy())
    assert np.array_equal(cb.ops.matmul_w4(x, odd).numpy(), cb.ops.matmul_w4(x, want).numpy())
