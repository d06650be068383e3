"""Drawing classes and learning from draws at numbers where float arithmetic ends or draws leave their range; definitions and bounds are those of
tests/draws_ref.py, or stand beside the test."""
import numpy as np
import pytest

from test_gpu_draws import _check_sample, _dev, _masked
from test_gpu_scores import _make, _tensor, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('layout', ['row', 'class'])
@pytest.mark.parametrize('k', [2, 8, 9, 32])
def test_limits_of_rows_that_a_warp_has(ops, layout, k):
    """Up to 32 classes a warp works on 32 rows alone; all its lanes read a table that the others fill."""
    torch, scores = ops
    r = np.random.default_rng(k)
    t = _tensor(torch, _masked(r, _make(r, 20000, k)), 'f32', layout)
    u = r.random((20000, 2))
    for limits in (dict(top_p=0.9), dict(min_p=0.05, top_k=3), dict(top_k=1)):
        _check_sample(ops, t, u, limits, (layout, k, str(limits)))
        first = scores.sample(t, _dev(torch, u), **limits)
        for _ in range(20):
            assert all(torch.equal(a, b) for a, b in zip(first, scores.sample(t, _dev(torch, u), **limits)))
