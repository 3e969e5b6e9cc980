"""What the 4-bit forms and the orthogonalised matrix do not record on the tape they refuse: every tensor whose gradient the
current context would follow."""
import numpy as np
import pytest

from test_gpu_muon_and_w4_frontend import F  # noqa: F401

pytestmark = pytest.mark.gpu


def tracked(F, ctx, a):  # noqa: F811
    t = F.Tensor.from_numpy(a)
    ctx.make_leaf(t, True)
    t.requires_grad(True)
    return t


def test_tracked_tensors_are_refused(F):  # noqa: F811
    rng = np.random.default_rng(2)
    a, b, x = (rng.standard_normal(s).astype(np.float32) for s in ((6, 8), (8,), (3, 6)))
    q = F.W4Weight(F.Tensor.from_numpy(a), group=32)
    plain_x, plain_b = F.Tensor.from_numpy(x), F.Tensor.from_numpy(b)
    with F.AutoDiff() as ctx:
        w, bias, tx = tracked(F, ctx, a), tracked(F, ctx, b), tracked(F, ctx, x)
        for call in (lambda: F.W4Weight(w, group=32), lambda: F.W4Weight(tx.matmul(w), group=32), lambda: plain_x.linear_w4(q, bias), lambda: tx.linear_w4(q, plain_b),
                     lambda: tx.linear_w4(q), lambda: w.orthogonalize()):
            with pytest.raises(F.FrontendError):
                call()
        want = plain_x.linear_w4(q, plain_b).numpy()                 # nothing to follow: allowed
        assert np.array_equal(F.W4Weight(F.Tensor.from_numpy(a), group=32).dequantize().numpy(), q.dequantize().numpy())
    # no context: nothing would follow them
    assert np.array_equal(plain_x.linear_w4(F.W4Weight(w, group=32), bias).numpy(), want)
