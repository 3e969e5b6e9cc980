"""Arguments of the trainer's orthogonalised steps that the step itself would refuse, in the middle of its updates."""
import numpy as np
import pytest

from test_gpu_muon_and_w4_frontend import F, batch, make_params  # noqa: F401

pytestmark = pytest.mark.gpu


def test_an_infinite_eps_is_refused_before_any_step(F):  # noqa: F811
    dims = [12, 16, 10]
    rng = np.random.default_rng(0)
    tr = F.MlpTrainer(dims, make_params(rng, dims), 0.01)
    tr.set_muon(lr=0.01)
    with pytest.raises(F.FrontendError):
        tr.set_muon(lr=0.02, eps=float("inf"))
    before = tr.params()
    tr.step_host(*batch(rng, 8, 12, 10))                     # the rule that was set before still holds
    assert np.isfinite(tr.params()).all() and not np.array_equal(tr.params(), before)
