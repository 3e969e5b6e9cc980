"""The trainer's update rule changed between graph steps: before, while and after the step is recorded, the run gives what the
same run of eager steps gives.  A recorded step may not allocate: each case has layer sizes of its own and runs its graph steps
first, so that nothing has left a buffer of the right size behind."""
import numpy as np
import pytest

from test_gpu_muon_and_w4_frontend import F, batch, make_params  # noqa: F401

pytestmark = pytest.mark.gpu


def run(F, dims, data, graph, change, at, undo_at):
    tr = F.MlpTrainer(dims, make_params(np.random.default_rng(1), dims), 1e-4)
    losses = []
    for i, (x, lab) in enumerate(data):
        if i == at:
            change(tr, True)
        if i == undo_at:
            change(tr, False)
        losses.append((tr.step_graph_host if graph else tr.step_host)(x, lab))
    return losses, tr.params()


@pytest.mark.parametrize("undo_after", [1, 2, 3, None])
@pytest.mark.parametrize("at", [1, 2, 3, 4])
def test_set_muon_after_any_number_of_graph_steps(F, at, undo_after):  # noqa: F811
    case = 4 * at + (undo_after or 0)
    dims = [200 + 8 * case, 300 + 16 * case, 10]
    rng = np.random.default_rng(case)
    data = [batch(rng, 32, dims[0], dims[-1]) for _ in range(at + 8)]

    def change(tr, on):
        tr.set_muon(lr=0.01, on=on)

    undo_at = None if undo_after is None else at + undo_after
    graph, eager = run(F, dims, data, True, change, at, undo_at), run(F, dims, data, False, change, at, undo_at)
    assert eager[0] == graph[0]
    assert np.array_equal(eager[1], graph[1])


@pytest.mark.parametrize("at", [1, 2, 3, 4])
def test_set_corrected_after_any_number_of_graph_steps(F, at):  # noqa: F811
    """The other switch that changes what a step allocates."""
    dims = [204 + 8 * at, 308 + 16 * at, 10]
    rng = np.random.default_rng(30 + at)
    data = [batch(rng, 32, dims[0], dims[-1]) for _ in range(at + 5)]

    def change(tr, on):
        tr.set_corrected(on, on)

    graph, eager = run(F, dims, data, True, change, at, None), run(F, dims, data, False, change, at, None)
    assert eager[0] == graph[0]
    assert np.array_equal(eager[1], graph[1])
