"""Orthogonalised steps in the data-parallel trainer: with one rank the run of a trainer without a communicator, bit for bit, in each
data-parallel mode that takes them; with two, the formula on the exchanged gradients and the same weights everywhere."""
import ctypes
import math
import os
import socket
import subprocess
import sys

import numpy as np
import pytest

import dp_muon_worker as W
from test_gpu_muon_and_w4_frontend import unpack
from test_gpu_orthogonalize import ns64, ns_tol

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def launch(world, out, mode, fresh, hidden_only, muon=True):
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = str(s.getsockname()[1])
    s.close()
    procs = []
    for r in range(world):
        env = dict(os.environ, RANK=str(r), WORLD_SIZE=str(world), LOCAL_RANK=str(r), MASTER_ADDR="127.0.0.1", MASTER_PORT=port, NCCL_NVLS_ENABLE="0")
        procs.append(subprocess.Popen([sys.executable, os.path.join(ROOT, "tests", "dp_muon_worker.py"), out, mode, *("01"[v] for v in (fresh, hidden_only, muon))], env=env,
                                      stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True))
    logs = []
    for p in procs:
        try:
            logs.append(p.communicate(timeout=300)[0])
        except subprocess.TimeoutExpired:
            p.kill()
            logs.append(p.communicate()[0])
    assert all(p.returncode == 0 for p in procs), "\n".join(logs)
    return np.load(out)


def follows_the_formula(r, hidden_only):
    """Each step's weights and momenta from the step before it and this step's gradients."""
    lr, mu, wd = (float(np.float32(W.MUON[k])) for k in ("lr", "momentum", "weight_decay"))
    before, mom = unpack(W.DIMS, W.params0()), [np.zeros((i, o)) for i, o in zip(W.DIMS[:-1], W.DIMS[1:])]
    for s in range(W.STEPS):
        grads, after, at = unpack(W.DIMS, r["grads"][s]), unpack(W.DIMS, r["params"][s]), 0
        for l, ((gw, gb), (w0, b0), (w1, b1)) in enumerate(zip(grads, before, after)):
            got_m = r["momenta"][s][at:at + gw.size].reshape(gw.shape)
            at += gw.size
            assert np.allclose(b1, b0 - np.float32(W.LR) * gb, rtol=1e-6, atol=1e-7)
            if hidden_only and l in (0, len(W.DIMS) - 2):
                assert np.allclose(w1, w0 - np.float32(W.LR) * gw, rtol=1e-6, atol=1e-7)
                continue
            m = mu * mom[l] + gw
            assert (np.abs(got_m - m) <= 2.0 ** -23 * (np.abs(mu * mom[l]) + np.abs(gw)) + 1e-38).all()
            o = ns64(gw + mu * m)
            scale = math.sqrt(max(1.0, gw.shape[1] / gw.shape[0]))
            # the step off by ns_tol (the momentum, kept in fp32, adds its own 2^-24), the weights by roundings
            assert np.linalg.norm(w1 - ((1 - lr * wd) * w0.astype(np.float64) - lr * scale * o)) <= lr * scale * np.linalg.norm(o) * (2 * ns_tol(5)) + 4 * 2.0 ** -24 * np.linalg.norm(w0)
            mom[l] = got_m.astype(np.float64)
        before = after
    assert int(r["status"]) == 0 and float(r["spread"]) == 0.0


@pytest.mark.parametrize("hidden_only", [False, True])
@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("mode", ["inplace", "arena", "serial"])
def test_one_rank(tmp_path, cb, mode, fresh, hidden_only):
    r = launch(1, str(tmp_path / "one.npz"), mode, fresh, hidden_only)
    for what in ("losses", "grads", "params", "momenta"):
        assert np.array_equal(r[what], r["alone_" + what]), what
    follows_the_formula(r, hidden_only)


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("mode", ["inplace", "arena", "serial", "sharded"])
def test_one_rank_of_sgd(tmp_path, cb, mode, fresh):
    """The current weights in backward (fresh) also where updates come out of the communicator's buffer."""
    r = launch(1, str(tmp_path / "sgd.npz"), mode, fresh, False, muon=False)
    for what in ("losses", "grads", "params"):
        assert np.array_equal(r[what], r["alone_" + what]), what


@pytest.mark.parametrize("mode", ["inplace", "arena", "serial"])
def test_two_ranks(tmp_path, cb, mode):
    n = ctypes.c_int()
    cb.check(cb.lib.ctk_device_count(ctypes.byref(n)))
    if n.value < 2:
        pytest.skip("needs 2 GPUs")
    follows_the_formula(launch(2, str(tmp_path / "two.npz"), mode, True, False), False)
