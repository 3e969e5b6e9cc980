"""Orthogonalised steps and 4-bit weights through the front end: tensors, the MLP trainer's eager and graph steps, and the
two together as they are used -- train with orthogonalised steps, quantise, predict."""
import math

import numpy as np
import pytest

from test_gpu_orthogonalize import grad_like, ns64, ns_tol
from test_gpu_w4 import pack, quantize64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def F(cb):
    from ctorch_b200 import frontend
    frontend.set_quiet(True)
    return frontend


def make_params(rng, dims):
    parts = []
    for i, o in zip(dims[:-1], dims[1:]):
        parts += [(rng.standard_normal((i, o)) * math.sqrt(2.0 / i)).astype(np.float32).ravel(), (0.1 * rng.standard_normal(o)).astype(np.float32)]
    return np.concatenate(parts)


def unpack(dims, flat):
    out, at = [], 0
    for i, o in zip(dims[:-1], dims[1:]):
        out.append((flat[at:at + i * o].reshape(i, o), flat[at + i * o:at + i * o + o]))
        at += i * o + o
    return out


def batch(rng, n, width, classes):
    return rng.random((n, width)).astype(np.float32), rng.integers(0, classes, n).astype(np.float32)


def test_tensor_forms_equal_the_c_entry_points(cb, F):
    rng = np.random.default_rng(1)
    g, p, m = grad_like(rng, 200, 300), rng.standard_normal((200, 300)).astype(np.float32), rng.standard_normal((200, 300)).astype(np.float32)
    tg, tp, tm = (F.Tensor.from_numpy(a) for a in (g, p, m))
    assert np.array_equal(tg.orthogonalize().numpy(), cb.ops.orthogonalize(cb.to_device(g)).numpy())
    keep = tp.copy()                                          # shares the buffer until the update writes
    tp.muon_update_(tg, tm, lr=0.1, mu=0.9, weight_decay=0.2)
    dp, dm = cb.to_device(p), cb.to_device(m)
    cb.ops.muon_update(dp, cb.to_device(g), dm, lr=0.1, momentum=0.9, weight_decay=0.2)
    assert np.array_equal(tp.numpy(), dp.numpy()) and np.array_equal(tm.numpy(), dm.numpy())
    assert np.array_equal(keep.numpy(), p)

    for symmetric in (True, False):
        q = F.W4Weight(tg, group=64, symmetric=symmetric)
        assert q.info() == dict(shape=(200, 300), group=64, symmetric=symmetric)
        ref = cb.ops.w4_quantize(cb.to_device(g), group=64, symmetric=symmetric)
        assert np.array_equal(q.dequantize().numpy(), cb.ops.w4_dequantize(ref).numpy())
        x, b = rng.standard_normal((3, 200)).astype(np.float32), rng.standard_normal(300).astype(np.float32)
        y = F.Tensor.from_numpy(x).linear_w4(q, F.Tensor.from_numpy(b), relu=True)
        assert np.array_equal(y.numpy(), cb.ops.matmul_w4(cb.to_device(x), ref, bias=cb.to_device(b), relu=True).numpy())
        one = F.Tensor.from_numpy(x[0]).linear_w4(q)
        assert one.shape == (300,) and np.array_equal(one.numpy(), cb.ops.matmul_w4(cb.to_device(x[0]), ref).numpy())


def test_tensor_forms_refuse(F):
    rng = np.random.default_rng(2)
    a = F.Tensor.from_numpy(rng.standard_normal((6, 8)).astype(np.float32))
    b = F.Tensor.from_numpy(rng.standard_normal((8, 6)).astype(np.float32))
    v = F.Tensor.from_numpy(rng.standard_normal(8).astype(np.float32))
    q = F.W4Weight(a, group=32)
    for call in (lambda: v.orthogonalize(), lambda: a.t().orthogonalize(), lambda: a.orthogonalize(steps=0), lambda: a.orthogonalize(eps=0.0),
                 lambda: a.muon_update_(b, a.copy(), 0.1), lambda: a.muon_update_(a.copy(), b, 0.1), lambda: F.W4Weight(a, group=48), lambda: F.W4Weight(v),
                 lambda: F.W4Weight(a.t()), lambda: v.linear_w4(q), lambda: b.linear_w4(q, b.narrow_rows(0, 1)), lambda: b.linear_w4(q, a), lambda: b.t().linear_w4(F.W4Weight(b))):
        with pytest.raises(F.FrontendError):
            call()
    with F.AutoDiff() as ctx:
        t = F.Tensor.from_numpy(rng.standard_normal((8, 6)).astype(np.float32))
        ctx.make_leaf(t, True)
        t.requires_grad(True)
        with pytest.raises(F.FrontendError):
            t.orthogonalize()
        with pytest.raises(F.FrontendError):
            t.linear_w4(q)


@pytest.mark.parametrize("hidden_only", [False, True])
@pytest.mark.parametrize("corrected", [False, True])
def test_trainer_steps_follow_the_formula(F, hidden_only, corrected):
    rng = np.random.default_rng(3)
    dims, lr, mlr, mu, wd = [40, 96, 130, 10], 0.001, 0.03, 0.9, 0.1
    flat = make_params(rng, dims)
    tr = F.MlpTrainer(dims, flat, lr)
    tr.set_corrected(corrected, corrected)
    tr.set_muon(lr=mlr, momentum=mu, weight_decay=wd, hidden_only=hidden_only)
    want = [(w.astype(np.float64), b.astype(np.float64)) for w, b in unpack(dims, flat)]
    mom = [np.zeros(w.shape) for w, _ in want]
    for step in range(3):
        before = unpack(dims, tr.params())
        x, lab = batch(rng, 32, dims[0], dims[-1])
        tr.step_host(x, lab)
        grads, after = unpack(dims, tr.grads()), unpack(dims, tr.params())
        for l, ((gw, gb), (w0, b0), (w1, b1)) in enumerate(zip(grads, before, after)):
            assert np.allclose(b1, b0 - np.float32(lr) * gb, rtol=1e-6, atol=1e-7)
            if hidden_only and l in (0, len(dims) - 2):
                assert np.allclose(w1, w0 - np.float32(lr) * gw, rtol=1e-6, atol=1e-7)
                continue
            mom[l] = mu * mom[l] + gw.astype(np.float64)
            o = ns64(gw + mu * mom[l])
            scale = math.sqrt(max(1.0, gw.shape[1] / gw.shape[0]))
            ref = (1 - mlr * wd) * w0 - mlr * scale * o
            # the step off by ns_tol (the momentum, kept in fp32, adds its own 2^-24 a step), the weights by a rounding
            assert np.linalg.norm(w1 - ref) <= mlr * scale * np.linalg.norm(o) * (2 * ns_tol(5)) + 4 * 2.0 ** -24 * np.linalg.norm(w0)


def test_trainer_graph_steps_equal_eager_steps(F):
    rng = np.random.default_rng(4)
    dims = [784, 128, 300, 10]
    flat = make_params(rng, dims)
    data = [batch(rng, 64, dims[0], dims[-1]) for _ in range(6)]

    def run(graph):
        tr = F.MlpTrainer(dims, flat, 1e-4)
        tr.set_muon(lr=0.01)
        losses = [(tr.step_graph_host if graph else tr.step_host)(x, lab) for x, lab in data]
        return tr, losses

    eager, le = run(False)
    graph, lg = run(True)
    assert le == lg
    assert np.array_equal(eager.params(), graph.params()) and np.array_equal(eager.muon_state(), graph.muon_state())


def test_trainer_state_resumes_and_muon_switches_off(F):
    rng = np.random.default_rng(5)
    dims = [30, 64, 10]
    flat = make_params(rng, dims)
    data = [batch(rng, 16, dims[0], dims[-1]) for _ in range(4)]
    a = F.MlpTrainer(dims, flat, 1e-3)
    a.set_corrected(True, True)             # (fresh weights: the tape holds nothing a new trainer does not have)
    a.set_muon(lr=0.02)
    for x, lab in data[:2]:
        a.step_host(x, lab)
    b = F.MlpTrainer(dims, a.params(), 1e-3)
    b.set_corrected(True, True)
    b.set_muon(lr=0.02)
    b.load_muon_state(a.muon_state())
    for x, lab in data[2:]:
        assert a.step_host(x, lab) == b.step_host(x, lab)
    assert np.array_equal(a.params(), b.params())
    # off: plain SGD again
    a.set_muon(on=False)
    with pytest.raises(F.FrontendError):
        a.muon_state()
    p0 = a.params()
    a.step_host(*data[0])
    assert np.allclose(a.params(), p0 - np.float32(1e-3) * a.grads(), rtol=1e-6, atol=1e-7)


def test_trainer_refusals(F):
    tr = F.MlpTrainer([8, 16, 4], np.zeros(8 * 16 + 16 + 16 * 4 + 4, np.float32), 0.1)
    for bad in (dict(steps=0), dict(steps=65), dict(eps=0.0), dict(eps=float("nan")), dict(momentum=1.0), dict(momentum=-0.1)):
        with pytest.raises(F.FrontendError):
            tr.set_muon(**bad)
    with pytest.raises(F.FrontendError):
        tr.predict_w4(F.Tensor.from_numpy(np.zeros((2, 8), np.float32)))
    with pytest.raises(F.FrontendError):
        tr.quantize_w4(group=24)
    with pytest.raises(ValueError):
        tr.load_muon_state(np.zeros(3, np.float32))
    tr.set_dp_mode("sharded")
    with pytest.raises(F.FrontendError):
        tr.set_muon()
    tr.set_dp_mode("arena")
    tr.set_muon()
    with pytest.raises(F.FrontendError):
        tr.set_dp_mode("sharded")


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("use_graph", [False, True])
def test_train_quantise_predict(F, symmetric, use_graph):
    """The run they are made for.  The prediction is held to the dequantised weights in 64 bits."""
    rng = np.random.default_rng(6)
    dims, group = [784, 128, 10], 64
    tr = F.MlpTrainer(dims, make_params(rng, dims), 1e-4)
    tr.set_muon(lr=0.01, weight_decay=0.01)
    for _ in range(5):
        x, lab = batch(rng, 64, dims[0], dims[-1])
        (tr.step_graph_host if use_graph else tr.step_host)(x, lab)
    snapshot = unpack(dims, tr.params())
    tr.quantize_w4(group=group, symmetric=symmetric)
    x, lab = batch(rng, 5, dims[0], dims[-1])
    tx = F.Tensor.from_numpy(x)
    probs = tr.predict_w4(tx).numpy()

    h = x.astype(np.float64)
    for l, (w, b) in enumerate(snapshot):
        codes, s, z = quantize64(w, group, symmetric)
        zero = 8.0 if symmetric else z.astype(np.float64)[..., None]
        w4 = ((codes - zero) * s.astype(np.float64)[..., None]).reshape(w.shape[1], -1)[:, :w.shape[0]].T
        h = h @ w4 + b
        h = np.maximum(h, 0) if l + 2 < len(dims) else h
    e = np.exp(h - h.max(1, keepdims=True))
    want = e / e.sum(1, keepdims=True)
    # logits to 2^-23 (group + groups + 40) of sums of a few tens, softmax's own 1e-5
    assert np.allclose(probs, want, rtol=2e-3, atol=1e-6)
    labels = F.Tensor.from_numpy(lab)
    assert tr.accuracy_w4(tx, labels) == pytest.approx(float((probs.argmax(1) == lab).mean()), abs=1e-6)
    # a snapshot: further steps, graph ones too, leave it as it is
    for _ in range(3):
        (tr.step_graph_host if use_graph else tr.step_host)(*batch(rng, 64, dims[0], dims[-1]))
    assert np.array_equal(tr.predict_w4(tx).numpy(), probs)
    one = tr.predict_w4(F.Tensor.from_numpy(x[0])).numpy()
    assert one.shape == (10,) and np.allclose(one, probs[0], rtol=1e-4, atol=1e-6)
