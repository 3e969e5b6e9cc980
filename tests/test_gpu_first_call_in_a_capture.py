"""The orthogonalised updates and the 4-bit weights inside a stream capture as the first call of their kernels in the process:
each case runs in a process of its own, records, replays, and compares with the same call made eagerly afterwards."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

WORKER = r"""
import ctypes, sys
import numpy as np
import ctorch_b200 as cb
kind, a, b, c = sys.argv[1], int(sys.argv[2]), int(sys.argv[3]), int(sys.argv[4])
cb.check(cb.lib.ctk_set_device(0))
rng = np.random.default_rng(1)
def arr(*shape):
    return rng.standard_normal(shape).astype(np.float32)
s = cb.Stream()
if kind == "orthogonalize":
    g, out = cb.to_device(arr(a, b)), cb.empty((a, b))
    call = lambda stream=None: cb.ops.orthogonalize(g, out=out, stream=stream)
    result = lambda: [out.numpy()]
    restore = lambda: None
elif kind == "muon":
    hp, hm = arr(a, b), arr(a, b)
    p, m, g = cb.to_device(hp), cb.to_device(hm), cb.to_device(arr(a, b))
    call = lambda stream=None: cb.ops.muon_update(p, g, m, lr=0.1, stream=stream)
    result = lambda: [p.numpy(), m.numpy()]
    def restore():
        p.copy_from_host(hp); m.copy_from_host(hm)
elif kind == "quantize":
    w, q, v = cb.to_device(arr(a, b)), cb.ops.W4Weight.empty(a, b, c, False), cb.empty((a, b))
    def call(stream=None):
        cb.ops.w4_quantize(w, group=c, symmetric=False, out=q, stream=stream)
        cb.ops.w4_dequantize(q, out=v, stream=stream)
    result = lambda: [q.packed.numpy(), q.scales.numpy(), q.zeros.numpy(), v.numpy()]
    restore = lambda: None
else:
    k, n, m = a, b, c
    packed = rng.integers(0, 2 ** 32, (n, -(-k // 64) * 8), dtype=np.uint64).astype(np.uint32)
    q = cb.ops.W4Weight(cb.to_device(packed, np.uint32), cb.to_device(rng.uniform(0.5, 1.5, (n, -(-k // 64))).astype(np.float32)), None, k, n, 64)
    x, y = cb.to_device(arr(m, k)), cb.empty((m, n))
    call = lambda stream=None: cb.ops.matmul_w4(x, q, out=y, stream=stream)
    result = lambda: [y.numpy()]
    restore = lambda: None
cb.synchronize()
cb.check(cb.lib.ctk_stream_begin_capture(s.handle))
call(s)
exe = ctypes.c_void_p()
cb.check(cb.lib.ctk_stream_end_capture(s.handle, ctypes.byref(exe)))
replays = []
for _ in range(2):
    restore()
    cb.synchronize()
    cb.check(cb.lib.ctk_graph_launch(exe, s.handle, 0))
    s.sync()
    replays.append(result())
cb.check(cb.lib.ctk_graph_destroy(exe))
restore()
call()
want = result()
for got in replays:
    assert all(np.array_equal(x, y) for x, y in zip(got, want)), kind
assert cb.ops.orthogonalize_status() == 0 and cb.ops.w4_status() == 0
print("as eager")
"""


@pytest.mark.parametrize("case", [("orthogonalize", 100, 300, 0), ("orthogonalize", 300, 500, 0), ("orthogonalize", 2100, 2060, 0), ("orthogonalize", 128, 9000, 0), ("muon", 10, 128, 0),
                                  ("muon", 784, 4096, 0), ("quantize", 700, 130, 32), ("quantize", 700, 130, 128), ("matmul", 300, 60, 2), ("matmul", 5000, 200, 3),
                                  ("matmul", 5000, 200, 40)])
def test_first_call_recorded(cb, case):
    env = dict(os.environ, PYTHONPATH=ROOT + os.pathsep + os.environ.get("PYTHONPATH", ""))
    r = subprocess.run([sys.executable, "-c", WORKER, *map(str, case)], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as eager" in r.stdout, r.stdout + r.stderr
