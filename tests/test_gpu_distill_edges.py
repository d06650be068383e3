"""Training from a teacher at its edges: gradients that grow small, many classes, best classes under rules entry by entry, ranks."""
import numpy as np
import pytest

import scores_ref as ref

pytestmark = pytest.mark.gpu


def _separable(classes, per_class):
    """`per_class` rows of every class, each with the one feature that names it."""
    from thundergbm_b200.synth import CsrData
    y = np.arange(classes * per_class) % classes
    n = y.size
    return CsrData(n, classes, np.arange(n + 1, dtype=np.int32), y.astype(np.int32), np.ones(n, np.float32), y.astype(np.float32)), y


def _check_roots(trees, want, n, bits):
    """Roots hold the sums of what the definition says: a value may be off by its own bound and by one step of the grid, 2^-bits of the
    next power of two above the largest value (which a kernel's may exceed by its bound), the sum by half a step of a float."""
    for name, at in (('sum_g', 'g'), ('sum_h', 'h')):
        v, off = want[at], want[at + '_off']
        step = 2.0 ** (np.floor(np.log2((np.abs(v) + off).max())) + 1 - bits)
        for c in range(v.shape[1]):
            got = float(trees[c][0][name])
            assert abs(got - v[:, c].sum()) <= off[:, c].sum() + n * step + 2.0 ** -24 * abs(got), (name, c, got, v[:, c].sum())


# classes of a lane per row, of a tile, of a block per row
@pytest.mark.parametrize('classes,per_class,lam', [(40, 10, 0.25), (600, 2, 0.1), (1100, 2, 0.09)])
@pytest.mark.parametrize('top', [1, 3])
def test_the_grid_of_a_round_is_as_fine_as_its_gradients(gpu, classes, per_class, lam, top):
    """Rows without a teacher whose labels are all but certain after a round: the gradients of their labels are as small as those of the
    other classes together, and the grid of the next round is that of small numbers."""
    from thundergbm_b200.booster import Booster
    d, y = _separable(classes, per_class)
    n, alpha = y.size, 0.25
    ids, logits = np.full((n, top), -1, np.int32), np.zeros((n, top), np.float32)
    b = Booster(d, objective='multi:softprob', num_class=classes, depth=2, n_trees=2, learning_rate=1.0, max_num_bin=255, hist_mode='exact',
                lambda_=lam, min_child_weight=0.0)
    b.set_teacher(ids, logits, None, 2.0, alpha)
    b.boost(1)
    s = b.ypred().T.copy()
    b.boost(1)
    want = ref.distill(s, ids, logits, None, y.astype(np.int32), None, 2.0, alpha)
    largest = float(np.abs(want['g']).max())
    assert largest < 2.0 ** -6
    _check_roots(b.trees()[1], want, n, 18)
    b.close()
