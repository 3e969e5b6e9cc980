"""4-bit weights at the ends of fp32's range: the product of very small and very large x and scales,
and of what is not finite, under relu too.

Tolerance of the product: that of the ordinary sizes, (group + groups + 40) 2^-23 sum |x| |w|, and near the smallest
numbers half a step of 2^-149 for each of the at most groups + 10 roundings of the result."""
import numpy as np
import pytest

from test_gpu_w4 import pack, values64

pytestmark = pytest.mark.gpu


def weight(cb, rng, k, n, group, symmetric, scale):
    groups = -(-k // group)
    packed = rng.integers(0, 2 ** 32, (n, groups * group // 8), dtype=np.uint64).astype(np.uint32)
    scales = (rng.uniform(0.5, 1.5, (n, groups)) * scale).astype(np.float32)
    zeros = None if symmetric else rng.integers(0, 16, (n, groups)).astype(np.uint8)
    dev = cb.ops.W4Weight(cb.to_device(packed, np.uint32), cb.to_device(scales), None if symmetric else cb.to_device(zeros, np.uint8), k, n, group)
    return dev, values64(packed, scales, zeros, k, group)


def bound_of(x, w, group):
    groups = -(-x.shape[1] // group)
    return (group + groups + 40) * 2.0 ** -23 * (np.abs(x).astype(np.float64) @ np.abs(w)) + (groups + 10) * 2.0 ** -150


@pytest.mark.parametrize("m,k,n,group", [(1, 300, 40, 32), (3, 4096, 130, 128), (12, 1000, 70, 64), (30, 2000, 200, 32)])
@pytest.mark.parametrize("factor,scale", [(1e-33, 1.0), (1e-34, 1e-3), (1e-36, 1.0), (1e-37, 1e-2), (1e-37, 1e6), (1e-38, 1.0), (1e-40, 1e4), (1e-43, 1e20), (1e-30, 1e-6),
                                          (1e-25, 1e-12), (1e20, 1e-38), (1e10, 1e-43), (1e30, 1.0), (1e34, 1e-3), (3e37, 1e-4), (3e37, 1e-38)])
def test_product_at_the_ends_of_the_range(cb, m, k, n, group, factor, scale):
    rng = np.random.default_rng(m + k)
    w4, w = weight(cb, rng, k, n, group, m % 2 == 1, scale)
    x = (rng.standard_normal((m, k)) * factor).astype(np.float32)
    assert np.isfinite(x).all()
    got = cb.ops.matmul_w4(cb.to_device(x), w4).numpy()
    assert (np.abs(got - x.astype(np.float64) @ w) <= bound_of(x, w, group)).all()


@pytest.mark.parametrize("m", [2, 5])
def test_product_of_blocks_from_the_smallest_to_the_largest(cb, m):
    """Neighbouring blocks of 128 k that hold numbers around 1e-40, 1e-30, .. 1e30, each with a scale that brings its products
    near 1: no block costs another its bits."""
    rng = np.random.default_rng(m)
    group, n = 64, 90
    exps = [-40, -37, -30, -20, -10, 0, 10, 20, 30, 36]
    k = 128 * len(exps)
    packed = pack(rng.integers(0, 16, (n, k)))
    mags = np.repeat(10.0 ** np.array(exps), 2)
    scales = (rng.uniform(0.5, 1.5, (n, k // group)) / np.maximum(mags, 1e-36)).astype(np.float32)
    w4 = cb.ops.W4Weight(cb.to_device(packed, np.uint32), cb.to_device(scales), None, k, n, group)
    w = values64(packed, scales, None, k, group)
    x = (rng.standard_normal((m, k)) * np.repeat(mags, group)).astype(np.float32)
    got = cb.ops.matmul_w4(cb.to_device(x), w4).numpy()
    assert (np.abs(got - x.astype(np.float64) @ w) <= bound_of(x, w, group)).all()


@pytest.mark.parametrize("m,k,n,group", [(1, 300, 40, 32), (3, 4096, 130, 128), (12, 1000, 70, 64)])
@pytest.mark.parametrize("factor,scale", [(1e-36, 1e-4), (1e-38, 1e-3), (1e-20, 1e-21), (1e-3, 1e-38), (1e-42, 1e-1)])
def test_products_below_the_smallest_normal_number(cb, m, k, n, group, factor, scale):
    """Where x's step times the scale is subnormal it is off by 2^-150.  The step is at least half of the largest |x| of 128, so the
    joined digits that it multiplies are below 2 * 15 * 128 < 2^12, and a group is off by 2^-138 at the most."""
    rng = np.random.default_rng(m + k)
    w4, w = weight(cb, rng, k, n, group, m % 2 == 1, scale)
    x = (rng.standard_normal((m, k)) * factor).astype(np.float32)
    got = cb.ops.matmul_w4(cb.to_device(x), w4).numpy()
    assert (np.abs(got - x.astype(np.float64) @ w) <= bound_of(x, w, group) + -(-k // group) * 2.0 ** -138).all()


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("m,k", [(1, 200), (5, 200), (5, 5000), (20, 900)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_non_finite_x_gives_nan_with_and_without_relu(cb, bad, m, k, relu):
    rng = np.random.default_rng(6)
    w4, _ = weight(cb, rng, k, 50, 64, False, 1.0)
    b = cb.to_device(rng.standard_normal(50).astype(np.float32))
    x = rng.standard_normal((m, k)).astype(np.float32)
    clean = cb.ops.matmul_w4(cb.to_device(x), w4, bias=b, relu=relu).numpy()
    x[m // 2, k // 3] = bad
    y = cb.ops.matmul_w4(cb.to_device(x), w4, bias=b, relu=relu).numpy()
    assert np.isnan(y[m // 2]).all()
    assert np.array_equal(np.delete(y, m // 2, 0), np.delete(clean, m // 2, 0)) and np.isfinite(clean).all()


def test_nan_scales_and_bias_show_under_relu(cb):
    rng = np.random.default_rng(7)
    w = rng.standard_normal((96, 6)).astype(np.float32)
    w[40, 2] = np.inf
    q = cb.ops.w4_quantize(cb.to_device(w), group=32)
    b = np.ones(6, np.float32)
    b[4] = np.nan
    y = cb.ops.matmul_w4(cb.to_device(np.ones((3, 96), np.float32)), q, bias=cb.to_device(b), relu=True).numpy()
    assert np.isnan(y[:, [2, 4]]).all() and np.isfinite(y[:, [0, 1, 3, 5]]).all() and (y[:, [0, 1, 3, 5]] >= 0).all()


def test_a_poisoned_hidden_layer_shows_in_the_prediction(cb):
    from ctorch_b200 import frontend as F
    rng = np.random.default_rng(9)
    dims = [40, 64, 10]
    params = rng.standard_normal(40 * 64 + 64 + 64 * 10 + 10).astype(np.float32)
    x = F.Tensor.from_numpy(rng.random((5, 40)).astype(np.float32))
    for bad in (np.nan, np.inf, -np.inf):
        poisoned = params.copy()
        poisoned[7 * 64 + 3] = bad
        tr = F.MlpTrainer(dims, poisoned, 0.1)
        tr.quantize_w4(group=32)
        assert np.isnan(tr.predict_w4(x).numpy()).all()
