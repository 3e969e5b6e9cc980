"""The CTA pairs' products with every operand orientation, and their last epilogue with the weights of an update in it: matrices
whose short side is above 2048, and wide products of medium ones; aligned and odd pitches.  The tolerance is that of the
small shapes (test_gpu_orthogonalize)."""
import ctypes

import numpy as np
import pytest

from test_gpu_orthogonalize import grad_like, ns64, ns_tol, rel

pytestmark = pytest.mark.gpu

i64, f32 = ctypes.c_int64, ctypes.c_float


@pytest.mark.parametrize("shape", [(2100, 2100), (2060, 2100), (2100, 2061), (2049, 4100)])
def test_orthogonalize_square_wide_and_tall(cb, shape):
    g = grad_like(np.random.default_rng(shape[0] + shape[1]), *shape)
    assert rel(cb.ops.orthogonalize(cb.to_device(g)).numpy(), ns64(g)) <= ns_tol(5)
    assert cb.ops.orthogonalize_status() == 0


def update_error(p_got, m_got, p, m, g, lr, mu, wd, scale, nesterov):
    """(error, bound) of the weights and (error, bound) of the momentum, as norms."""
    lr, mu, wd, scale = (float(np.float32(v)) for v in (lr, mu, wd, scale))
    m64 = mu * m.astype(np.float64) + g
    o = ns64(g + mu * m64 if nesterov else m64)
    want = (1 - lr * wd) * p.astype(np.float64) - lr * scale * o
    # lr scale NS(u) off by ns_tol; keep, step, their products and the sum each rounded once (2^-24 each)
    return (np.linalg.norm(p_got - want), lr * scale * np.linalg.norm(o) * (ns_tol(5) + 3 * 2.0 ** -24) + 3 * 2.0 ** -24 * np.linalg.norm(p),
            np.abs(m_got - m64).max(), 2.0 ** -23 * (np.abs(mu * m) + np.abs(g)).max())


@pytest.mark.parametrize("shape,nesterov", [((2100, 2060), True), ((2060, 2100), False), ((784, 4096), True), ((785, 4097), True), ((4096, 784), False), ((2049, 2049), True)])
def test_muon_update_through_the_pairs(cb, shape, nesterov):
    rng = np.random.default_rng(3 * shape[0] + shape[1])
    p, m, g = rng.standard_normal(shape).astype(np.float32), grad_like(rng, *shape), grad_like(rng, *shape)
    dp, dm, dg = cb.to_device(p), cb.to_device(m), cb.to_device(g)
    cb.ops.muon_update(dp, dg, dm, lr=0.5, momentum=0.9, nesterov=nesterov, weight_decay=0.1, scale=1.5)
    e, b, em, bm = update_error(dp.numpy(), dm.numpy(), p, m, g, 0.5, 0.9, 0.1, 1.5, nesterov)
    assert e <= b and em <= bm
    assert np.array_equal(dg.numpy(), g)
    assert cb.ops.orthogonalize_status() == 0


@pytest.mark.parametrize("rows,cols,ldp,ldg,ldm,at", [(784, 4096, 4100, 4096, 4104, 0), (784, 4096, 4099, 4097, 4101, 1), (2100, 2052, 2053, 2052, 2056, 3)])
def test_muon_update_through_the_pairs_with_pitches(cb, rows, cols, ldp, ldg, ldm, at):
    """Rows longer than the matrix, odd ones and odd addresses among them: what lies between the rows stays."""
    rng = np.random.default_rng(rows + at)

    def padded(ld, a):
        flat = rng.standard_normal(rows * ld + at).astype(np.float32)
        flat[at:].reshape(rows, ld)[:, :cols] = a
        return flat

    p, m, g = rng.standard_normal((rows, cols)).astype(np.float32), grad_like(rng, rows, cols), grad_like(rng, rows, cols)
    hp, hm, hg = padded(ldp, p), padded(ldm, m), padded(ldg, g)
    dp, dm, dg = cb.to_device(hp), cb.to_device(hm), cb.to_device(hg)
    cb.check(cb.lib.ctk_muon_update_f32(dp.view(at, (1,)).p, i64(ldp), dg.view(at, (1,)).p, i64(ldg), dm.view(at, (1,)).p, i64(ldm), i64(rows), i64(cols), f32(0.5), f32(0.9), 1,
                                        f32(0.1), f32(1.5), 5, f32(1e-7), None, None))
    fp, fm = dp.numpy(), dm.numpy()
    got_p, got_m = (f[at:].reshape(rows, ld) for f, ld in ((fp, ldp), (fm, ldm)))
    e, b, em, bm = update_error(got_p[:, :cols], got_m[:, :cols], p, m, g, 0.5, 0.9, 0.1, 1.5, True)
    assert e <= b and em <= bm
    hp[at:].reshape(rows, ldp)[:, :cols] = got_p[:, :cols]
    hm[at:].reshape(rows, ldm)[:, :cols] = got_m[:, :cols]
    assert np.array_equal(fp, hp) and np.array_equal(fm, hm) and np.array_equal(dg.numpy(), hg)
