"""Orthogonalised updates against their formulas in 64 bits.

Tolerances.  One Newton-Schulz step multiplies an error of X by at most a = 3.4445 (the slope of the step's
polynomial at 0 is its largest), so an error of relative size e made in step k of 5 arrives as at most
a^(5-k) e: over all steps and the rounding of the start, sum a^j (j = 0..5) = 682 e.  The kernels carry X in
22 bits or more and their products in fp32: e = 2^-23.  Errors are measured as |O - ref|_F / |ref|_F, so
NS_TOL = 682 * 2^-23 = 8.2e-5 for 5 steps."""
import ctypes
import math

import numpy as np
import pytest

from conftest import assert_close

pytestmark = pytest.mark.gpu

A_, B_, C_ = 3.4445, -4.7750, 2.0315
i64, f32 = ctypes.c_int64, ctypes.c_float


def ns_tol(steps):
    return sum(A_ ** j for j in range(steps + 1)) * 2.0 ** -23


def ns64(g, steps=5, eps=1e-7):
    x = np.asarray(g, np.float64)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (np.linalg.norm(x) + eps)
    for _ in range(steps):
        s = x @ x.T
        x = A_ * x + (B_ * s + C_ * (s @ s)) @ x
    return x.T if tall else x


def rel(got, ref):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    return np.linalg.norm(got - ref) / max(np.linalg.norm(ref), 1e-300)


def grad_like(rng, rows, cols, kind="noise"):
    g = rng.standard_normal((rows, cols))
    if kind == "decay":            # singular values over three decades
        u, s, v = np.linalg.svd(g, full_matrices=False)
        g = (u * np.exp(-7.0 * np.arange(len(s)) / max(len(s), 1))) @ v
    if kind == "spike":            # one direction a hundred times stronger than the rest
        g = g + 100.0 * np.sqrt(max(rows, cols)) / np.sqrt(rows * cols) * np.outer(rng.standard_normal(rows), rng.standard_normal(cols))
    return g.astype(np.float32)


SHAPES = [(1, 1), (1, 7), (7, 1), (8, 8), (10, 128), (128, 10), (127, 129), (129, 127), (128, 128), (64, 1500), (1500, 64), (256, 256), (257, 255),
          (300, 100), (333, 1001), (784, 128), (640, 640), (1000, 520), (513, 2049), (2049, 513), (1300, 1290)]


@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize_shapes(cb, shape):
    g = grad_like(np.random.default_rng(shape[0] * 7919 + shape[1]), *shape)
    o = cb.ops.orthogonalize(cb.to_device(g)).numpy()
    assert o.shape == shape
    assert rel(o, ns64(g)) <= ns_tol(5)
    assert cb.ops.orthogonalize_status() == 0


@pytest.mark.parametrize("steps", [1, 2, 3, 8])
@pytest.mark.parametrize("shape", [(40, 300), (300, 280)])
def test_orthogonalize_step_counts(cb, shape, steps):
    g = grad_like(np.random.default_rng(steps), *shape)
    assert rel(cb.ops.orthogonalize(cb.to_device(g), steps=steps).numpy(), ns64(g, steps)) <= ns_tol(steps)


@pytest.mark.parametrize("kind", ["decay", "spike"])
@pytest.mark.parametrize("shape", [(96, 200), (520, 512)])
def test_orthogonalize_spectra(cb, shape, kind):
    g = grad_like(np.random.default_rng(3), *shape, kind=kind)
    assert rel(cb.ops.orthogonalize(cb.to_device(g)).numpy(), ns64(g)) <= ns_tol(5)


@pytest.mark.parametrize("factor", [1e-30, 1e-20, 1e-12, 1e-8, 1e-6, 1e6, 1e30, 1e36])
@pytest.mark.parametrize("shape", [(33, 70), (270, 260)])
def test_orthogonalize_any_magnitude(cb, shape, factor):
    """eps is part of the formula: far below it the result shrinks with the input and keeps its relative accuracy."""
    g = (grad_like(np.random.default_rng(11), *shape).astype(np.float64) * factor).astype(np.float32)
    assert rel(cb.ops.orthogonalize(cb.to_device(g)).numpy(), ns64(g)) <= ns_tol(5)


@pytest.mark.parametrize("shape", [(5, 9), (200, 140), (300, 400)])
def test_orthogonalize_zero_and_non_finite(cb, shape):
    g = np.zeros(shape, np.float32)
    assert not cb.ops.orthogonalize(cb.to_device(g)).numpy().any()
    for bad in (np.nan, np.inf, -np.inf):
        h = grad_like(np.random.default_rng(1), *shape)
        h[shape[0] // 2, shape[1] // 3] = bad
        assert np.isnan(cb.ops.orthogonalize(cb.to_device(h)).numpy()).all()


def test_orthogonalize_one_strong_element(cb):
    g = np.full((300, 310), 1e-6, np.float32)
    g[17, 200] = 1.0
    assert rel(cb.ops.orthogonalize(cb.to_device(g)).numpy(), ns64(g)) <= ns_tol(5)


def test_orthogonalize_pitches_in_place_and_unaligned(cb):
    rng = np.random.default_rng(5)
    rows, cols, ldg, ldo = 150, 201, 208, 203
    g = grad_like(rng, rows, cols)
    host = np.full((rows, ldg), 7.0, np.float32)
    host[:, :cols] = g
    src = cb.to_device(host)
    dst = cb.to_device(np.full(rows * ldo + 1, -3.0, np.float32))
    cb.check(cb.lib.ctk_orthogonalize_f32(src.p, i64(ldg), dst.view(1, (rows, ldo)).p, i64(ldo), i64(rows), i64(cols), 5, f32(1e-7), None, None))
    flat = dst.numpy()
    out = flat[1:].reshape(rows, ldo)
    assert rel(out[:, :cols], ns64(g)) <= ns_tol(5)
    assert flat[0] == -3.0 and (out[:, cols:] == -3.0).all()          # what lies between the rows stays
    assert (src.numpy() == host).all()
    # in place
    d = cb.to_device(g)
    cb.ops.orthogonalize(d, out=d)
    assert np.array_equal(d.numpy(), out[:, :cols])


@pytest.mark.parametrize("shape", [(48, 200), (900, 300), (1100, 1100)])
def test_orthogonalize_same_bits_own_workspace_and_stream(cb, shape):
    g = cb.to_device(grad_like(np.random.default_rng(9), *shape))
    first = cb.ops.orthogonalize(g).numpy()
    ws = cb.ops.orthogonalize_workspace(shape)
    ws.fill_bytes(0xFF)                                                 # whatever it held before
    s = cb.Stream()
    out = cb.empty(shape)
    cb.synchronize()
    cb.ops.orthogonalize(g, out=out, workspace=ws, stream=s)
    assert np.array_equal(out.numpy(stream=s), first)
    cb.ops.orthogonalize(g, out=out, workspace=ws, stream=s)
    assert np.array_equal(out.numpy(stream=s), first)


def test_orthogonalize_two_streams_at_once(cb):
    rng = np.random.default_rng(21)
    shapes = [(500, 700), (90, 1200)]
    gs = [cb.to_device(grad_like(rng, *s)) for s in shapes]
    alone = [cb.ops.orthogonalize(g).numpy() for g in gs]
    streams = [cb.Stream(), cb.Stream()]
    outs = [cb.empty(s) for s in shapes]
    cb.synchronize()
    for _ in range(4):
        for g, o, st in zip(gs, outs, streams):
            cb.ops.orthogonalize(g, out=o, stream=st)
    for o, st, want in zip(outs, streams, alone):
        assert np.array_equal(o.numpy(stream=st), want)


@pytest.mark.parametrize("shape", [(60, 110), (600, 400)])
@pytest.mark.parametrize("own_workspace", [False, True])
def test_muon_update_captured_and_replayed(cb, shape, own_workspace):
    rng = np.random.default_rng(33)
    p0, m0 = (rng.standard_normal(shape).astype(np.float32) for _ in range(2))
    gs = [grad_like(rng, *shape) for _ in range(3)]
    ws = cb.ops.orthogonalize_workspace(shape) if own_workspace else None

    def fresh():
        return cb.to_device(p0), cb.to_device(m0), cb.to_device(gs[0])

    p, m, g = fresh()
    for h in gs:
        g.copy_from_host(h)
        cb.ops.muon_update(p, g, m, lr=0.02, weight_decay=0.1)
    want = p.numpy(), m.numpy()

    p, m, g = fresh()
    s = cb.Stream()
    cb.synchronize()
    cb.check(cb.lib.ctk_stream_begin_capture(s.handle))
    cb.ops.muon_update(p, g, m, lr=0.02, weight_decay=0.1, workspace=ws, stream=s)
    exe = ctypes.c_void_p()
    cb.check(cb.lib.ctk_stream_end_capture(s.handle, ctypes.byref(exe)))
    cb.ops.orthogonalize(cb.to_device(gs[1]))                            # an eager call in between
    for h in gs:
        g.copy_from_host(h)
        cb.check(cb.lib.ctk_graph_launch(exe, s.handle, 0))
        s.sync()
    assert np.array_equal(p.numpy(), want[0]) and np.array_equal(m.numpy(), want[1])
    cb.check(cb.lib.ctk_graph_destroy(exe))


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shape", [(3, 2), (10, 128), (128, 10), (333, 1001), (784, 130), (700, 700)])
def test_muon_update(cb, shape, nesterov):
    rng = np.random.default_rng(shape[0] + shape[1])
    p, m, g = rng.standard_normal(shape).astype(np.float32), grad_like(rng, *shape), grad_like(rng, *shape)
    lr, mu, wd, scale = 0.02, 0.95, 0.1, 1.7
    dp, dm = cb.to_device(p), cb.to_device(m)
    cb.ops.muon_update(dp, cb.to_device(g), dm, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd, scale=scale)
    lr, mu, wd, scale = (float(np.float32(v)) for v in (lr, mu, wd, scale))
    m64 = mu * m.astype(np.float64) + g
    # fl(mu m + g): one rounding of at most 2^-24 of the sum (and of the product, where it is not fused)
    assert (np.abs(dm.numpy() - m64) <= 2.0 ** -23 * (np.abs(mu * m) + np.abs(g)) + 1e-38).all()
    u = g + mu * m64 if nesterov else m64
    o = ns64(u)
    want = (1 - lr * wd) * p.astype(np.float64) - lr * scale * o
    err = np.linalg.norm(dp.numpy() - want)
    # lr scale NS(u) off by ns_tol; keep, step, their products and the sum each rounded once (2^-24 each)
    assert err <= lr * scale * np.linalg.norm(o) * (ns_tol(5) + 3 * 2.0 ** -24) + 3 * 2.0 ** -24 * np.linalg.norm(p)


def test_muon_update_default_scale_and_pitches(cb):
    rng = np.random.default_rng(77)
    rows, cols, ldp, ldg, ldm = 70, 180, 183, 180, 200
    p, m, g = (rng.standard_normal((rows, ld)).astype(np.float32) for ld in (ldp, ldm, ldg))
    dp, dm, dg = cb.to_device(p), cb.to_device(m), cb.to_device(g)
    scale = math.sqrt(cols / rows)
    cb.check(cb.lib.ctk_muon_update_f32(dp.p, i64(ldp), dg.p, i64(ldg), dm.p, i64(ldm), i64(rows), i64(cols), f32(0.1), f32(0.9), 1, f32(0.0), f32(scale), 5,
                                        f32(1e-7), None, None))
    a, b = cb.to_device(p[:, :cols]), cb.to_device(m[:, :cols])
    cb.ops.muon_update(a, cb.to_device(g[:, :cols]), b, lr=0.1, momentum=0.9)          # scale None: sqrt(cols / rows)
    got_p, got_m = dp.numpy(), dm.numpy()
    assert np.array_equal(got_p[:, :cols], a.numpy()) and np.array_equal(got_m[:, :cols], b.numpy())
    assert np.array_equal(got_p[:, cols:], p[:, cols:]) and np.array_equal(got_m[:, cols:], m[:, cols:])


def test_empty_matrices(cb):
    for shape in ((0, 5), (5, 0)):
        assert cb.ops.orthogonalize(cb.empty(shape)).shape == shape


def test_large_matrix_rows_against_float64(cb):
    """2100 x 2060: every tile row of the large kernels, edges included."""
    g = grad_like(np.random.default_rng(2), 2100, 2060)
    assert rel(cb.ops.orthogonalize(cb.to_device(g)).numpy(), ns64(g)) <= ns_tol(5)


@pytest.mark.parametrize("shape", [(1, 2048), (2048, 1), (128, 2048), (2048, 128), (127, 2047), (65, 1025), (1030, 17), (16, 16), (17, 129), (128, 129), (129, 128),
                                   (2, 3), (100, 640), (500, 33), (128, 2049), (2049, 128)])
def test_sizes_around_the_one_launch_limit(cb, shape):
    rng = np.random.default_rng(shape[0] + 3 * shape[1])
    g, p, m = grad_like(rng, *shape), rng.standard_normal(shape).astype(np.float32), grad_like(rng, *shape)
    assert rel(cb.ops.orthogonalize(cb.to_device(g)).numpy(), ns64(g)) <= ns_tol(5)
    dp, dm = cb.to_device(p), cb.to_device(m)
    cb.ops.muon_update(dp, cb.to_device(g), dm, lr=0.5, momentum=0.5, scale=1.0)
    m64 = 0.5 * m.astype(np.float64) + g
    o = ns64(g + 0.5 * m64)
    assert np.linalg.norm(dp.numpy() - (p - 0.5 * o)) <= 0.5 * np.linalg.norm(o) * (ns_tol(5) + 3 * 2.0 ** -24) + 3 * 2.0 ** -24 * np.linalg.norm(p)
    assert (np.abs(dm.numpy() - m64) <= 2.0 ** -23 * (np.abs(0.5 * m) + np.abs(g)) + 1e-38).all()
    assert cb.ops.orthogonalize_status() == 0


@pytest.mark.parametrize("shape", [(3, 20000), (128, 9000), (30011, 100), (130, 16000), (16001, 200), (300, 12345)])
def test_long_thin_matrices(cb, shape):
    g = grad_like(np.random.default_rng(shape[0]), *shape)
    d = cb.to_device(g)
    o = cb.ops.orthogonalize(d).numpy()
    assert rel(o, ns64(g)) <= ns_tol(5)
    assert np.array_equal(cb.ops.orthogonalize(d).numpy(), o)
    assert cb.ops.orthogonalize_status() == 0


@pytest.mark.parametrize("shape", [(70, 90), (300, 210)])
def test_orthogonalize_columns_of_one_buffer(cb, shape):
    """g and out side by side in the rows of one buffer, in both orders."""
    rows, cols = shape
    rng = np.random.default_rng(rows)
    ld = 2 * cols + 3
    g = grad_like(rng, rows, cols)
    want = cb.ops.orthogonalize(cb.to_device(g)).numpy()
    for at_g, at_out in ((0, cols + 3), (cols, 0)):
        host = rng.standard_normal((rows, ld)).astype(np.float32)
        host[:, at_g:at_g + cols] = g
        buf = cb.to_device(host)
        cb.check(cb.lib.ctk_orthogonalize_f32(buf.view(at_g, (1,)).p, i64(ld), buf.view(at_out, (1,)).p, i64(ld), i64(rows), i64(cols), 5, f32(1e-7), None, None))
        got = buf.numpy()
        # (which loads are taken four at a time depends on the alignment, not what they add up to)
        assert rel(got[:, at_out:at_out + cols], want) <= ns_tol(5)
        host[:, at_out:at_out + cols] = got[:, at_out:at_out + cols]
        assert np.array_equal(got, host)


def test_orthogonalize_from_several_threads(cb):
    """Calls from four threads at once, each on a stream of its own, give what they give alone."""
    import threading
    rng = np.random.default_rng(77)
    shapes = [(64, 300), (400, 250), (129, 40), (300, 2000)]
    gs = [cb.to_device(grad_like(rng, *s)) for s in shapes]
    outs = [cb.empty(s) for s in shapes]
    errors = []
    cb.synchronize()

    def work(i):
        try:
            st = cb.Stream()
            for _ in range(5):
                cb.ops.orthogonalize(gs[i], out=outs[i], stream=st)
            st.sync()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(shapes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for g, o in zip(gs, outs):
        assert np.array_equal(o.numpy(), cb.ops.orthogonalize(g).numpy())
