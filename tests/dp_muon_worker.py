"""Worker of the data-parallel tests of the update rules (one process per rank; started by the tests, not collected).  Trains the
MLP on this rank's shard with the communicator attached; rank 0 writes, step by step, the exchanged gradients, the weights and
the momenta, and how far any rank's weights and momenta are from its own."""
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

DIMS, BATCH, STEPS, LR = [96, 160, 140, 10], 32, 4, 0.001
MUON = dict(lr=0.03, momentum=0.9, weight_decay=0.1)


def params0():
    rng = np.random.default_rng(78)
    parts = []
    for i, o in zip(DIMS[:-1], DIMS[1:]):
        parts += [(rng.standard_normal((i, o)) * np.sqrt(2.0 / i)).astype(np.float32).ravel(), (0.1 * rng.standard_normal(o)).astype(np.float32)]
    return np.concatenate(parts)


def data(rank):
    rng = np.random.default_rng(100 + rank)
    return rng.random((STEPS, BATCH, DIMS[0])).astype(np.float32), rng.integers(0, DIMS[-1], (STEPS, BATCH)).astype(np.float32)


def train(F, comm, mode, fresh, rank, hidden_only, muon):
    """(losses, grads, params, momenta) after every step; muon False: SGD, without the momenta."""
    tr = F.MlpTrainer(DIMS, params0(), LR)
    tr.set_corrected(fresh, fresh)
    if comm is not None:
        tr.set_dp_mode(mode)
    if muon:
        tr.set_muon(hidden_only=hidden_only, **MUON)
    if comm is not None:
        tr.set_comm(comm)
    x, lab = data(rank)
    out = [[], [], [], []]
    for s in range(STEPS):
        for o, v in zip(out, (tr.step_host(x[s], lab[s]), tr.grads(), tr.params(), tr.muon_state() if muon else np.zeros(0, np.float32))):
            o.append(v)
    if comm is not None:
        tr.set_comm(None)
    return [np.stack(o) for o in out]


def main():
    out, mode, fresh, hidden_only, muon = sys.argv[1], sys.argv[2], sys.argv[3] == "1", sys.argv[4] == "1", sys.argv[5] == "1"
    from ctorch_b200 import dp
    cp = dp.ControlPlane()
    import ctorch_b200 as cb
    from ctorch_b200 import frontend as F
    cb.check(cb.lib.ctk_set_device(cp.local_rank))
    F.set_quiet(True)
    comm, _ = dp.make_comm(cb, cp)
    losses, grads, params, momenta = train(F, comm, mode, fresh, cp.rank, hidden_only, muon)
    spread = 0.0
    for mine in (params, momenta):
        first = cp.broadcast_bytes(mine.ravel().view(np.uint8).copy(), 0).view(np.float32).reshape(mine.shape)
        spread = max(spread, cp.max_over_ranks(float(np.abs(mine - first).max(initial=0.0))))
    alone = train(F, None, mode, fresh, cp.rank, hidden_only, muon)
    if cp.rank == 0:
        np.savez(out, losses=losses, grads=grads, params=params, momenta=momenta, spread=spread, status=cb.ops.orthogonalize_status(),
                 **{f"alone_{n}": v for n, v in zip(("losses", "grads", "params", "momenta"), alone)})
    cb.synchronize()
    cb.lib.ctk_comm_destroy(comm)
    cp.close()


if __name__ == "__main__":
    main()
