"""The operators on scores where rows, lists and arguments are at their edges; definitions and bounds are those of tests/scores_ref.py."""
import numpy as np
import pytest

import scores_ref as ref
from test_gpu_scores import _close, _given, _tensor, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('kind', ['f16', 'bf16', 'f32'])
@pytest.mark.parametrize('order', ['up', 'steps', 'ends', 'block'])
def test_top_of_long_rising_rows(ops, order, kind):
    """Rows whose scores rise along the row, most of them in runs of equal ones: every step of a block finds more candidates than its list
    has room for, the last ones above all that were kept."""
    torch, scores = ops
    k = 50021
    z = np.arange(k) / 64
    if order == 'steps':      # one score per 8192 classes
        z = np.floor(np.arange(k) / 8192)
    elif order == 'ends':     # the last scores of every 8192 stand out, each time further
        z = np.where(np.arange(k) % 8192 >= 8192 - 2048, 16 * (np.arange(k) // 8192) + np.arange(k) % 64 / 8, -1.0)
    elif order == 'block':
        z = np.where((np.arange(k) // 1500) % 3 == 1, np.arange(k) / 32, 0.0)
    one = _tensor(torch, z[None], kind, 'row')
    for m in (65, 100, 128):
        values, ids, lse, off = ref.top(_given(one), m)
        for n in (1, 300):   # a cluster for the row, a block for each
            got = [x.cpu().numpy() for x in scores.top(one.repeat(n, 1), m)]
            assert (got[1] == ids).all() and (got[0] == values).all(), (m, n)
            _close(got[2], lse.repeat(n), off[0], (order, m, n))
