"""Quantising groups whose scale is subnormal, by the definition."""
import numpy as np
import pytest

from test_gpu_w4 import pack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_subnormal_groups_with_zero_points(cb, group):
    """Where a scale is subnormal it cannot be a fifteenth of the range any more: the zero point is clamped to 15, the codes to
    0 .. 15."""
    rng = np.random.default_rng(group)
    tiny = 2.0 ** -149
    k, n = 3 * group - 5, 40
    w = np.zeros((k, n))
    for j in range(n):
        top = int(rng.integers(1, 400))
        w[:, j] = rng.integers(-top if j % 3 else 0, top if j % 4 else 1, k, endpoint=True) * tiny
    w[:, 0] = -22 * tiny
    w = w.astype(np.float32)
    q = cb.ops.w4_quantize(cb.to_device(w), group=group, symmetric=False)
    groups = -(-k // group)
    v = np.zeros((n, groups * group))
    v[:, :k] = w.astype(np.float64).T
    v = v.reshape(n, groups, group)
    lo = np.minimum(v.min(-1), 0)
    s = ((np.maximum(v.max(-1), 0) - lo) / 15.0).astype(np.float32)
    s64 = np.where(s > 0, s, 1).astype(np.float64)
    zero = np.where(s > 0, np.minimum(np.rint(-lo / s64), 15), 0)
    code = np.where(s[..., None] > 0, np.clip(np.rint(v / s64[..., None]) + zero[..., None], 0, 15), 0)
    assert zero.max() == 15 and (np.rint(-lo / s64) > 15).any()
    assert np.array_equal(q.scales.numpy(), s)
    assert np.array_equal(q.zeros.numpy(), zero.astype(np.uint8))
    assert np.array_equal(q.packed.numpy(), pack(code.astype(np.uint32)))
