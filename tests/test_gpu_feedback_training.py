"""Training from drawn classes and the gains that followed, and drawing from a model, through the public entry points: the gradients that
trees were grown on are those of the definition (tests/draws_ref.py), round after round, and the pieces run together."""
import numpy as np
import pytest

import draws_ref as ref
from test_gpu_distill_training import _data

pytestmark = pytest.mark.gpu


def _logged(r, n, classes, m):
    drawn = r.integers(0, classes, (n, m)).astype(np.int32)
    drawn[r.random((n, m)) < 0.1] = -1
    drawn[0] = -1
    gains = r.standard_normal((n, m)).astype(np.float32)
    old = np.full((n, m), -np.log(classes), np.float32) + 0.3 * r.standard_normal((n, m)).astype(np.float32)
    return drawn, gains, old


@pytest.mark.parametrize('n,classes,m,T,clip,entropy,with_old,with_weights', [(3000, 3, 1, 1.0, None, 0.0, False, False), (2500, 7, 2, 0.8, (0.2, 0.4), 0.05, True, True),
                                                                              (1500, 40, 5, 1.5, (0.3, 0.3), 0.0, True, False), (9000, 5, 1, 1.0, None, 0.1, True, False)])
@pytest.mark.parametrize('mode', ['exact', 'fp32'])
def test_nodes_hold_the_gradients_of_the_definition(gpu, n, classes, m, T, clip, entropy, with_old, with_weights, mode):
    """The root of every tree of a round holds the sum of the gradients at the scores of the round before.  A value is rounded to a grid
    of 2^-18 (exact) or finer of a power of two above the round's largest, which is at most twice that; the sum is then a float.  A draw
    whose ratio lies within 2^-18 of a bound (its log is off by less) may count with or without its gradient."""
    from thundergbm_b200.booster import Booster
    d, x, y, _ = _data(n, 6, classes, n + classes)
    r = np.random.default_rng(n)
    drawn, gains, old = _logged(r, n, classes, m)
    more = dict(old=old if with_old else None, weights=r.random(n).astype(np.float32) if with_weights else None, temperature=T, clip=clip, entropy=entropy)
    rounds = 4
    for stop in range(1, rounds + 1):   # (from the second round on a boosting round is a graph that is replayed)
        b = Booster(d, objective='multi:softprob', num_class=classes, depth=4, n_trees=rounds, learning_rate=0.5, max_num_bin=64, hist_mode=mode)
        b.set_feedback(drawn if m > 1 else drawn[:, 0], gains if m > 1 else gains[:, 0],
                       **{**more, 'old': None if not with_old else old if m > 1 else old[:, 0]})
        s = np.zeros((classes, n), np.float32)
        if stop > 1:
            b.boost(stop - 1)
            s = b.ypred()
        loss = b.feedback_loss()
        b.boost(1)
        trees = b.trees()[stop - 1]
        want = ref.feedback(s.T, drawn, gains, **more)
        either = np.where(want['gap'] < 2.0 ** -18, np.abs(gains), 0).sum() * 2 / T
        for c in range(classes):
            for name, g, off in (('sum_g', want['g'][:, c], want['g_off'][:, c]), ('sum_h', want['h'][:, c], want['h_off'][:, c])):
                scale = 2 * max(np.abs(want['g']).max(), want['h'].max()) * 2.0 ** -17 * n
                got = float(trees[c][0][name])
                assert abs(got - g.sum()) <= off.sum() + scale + 2.0 ** -22 * abs(g).sum() + 2 * either, (stop, c, name)
        assert abs(loss - want['loss'].mean()) <= want['loss_off'].mean() + 2.0 ** -40 * abs(want['loss']).sum()
        b.close()


def test_a_gain_of_one_without_a_ratio_is_a_label(gpu):
    """Every row's label drawn, with a gain of 1: the gradients of the softmax objective, and its first trees' splits."""
    from thundergbm_b200.booster import Booster
    d, x, y, _ = _data(4000, 5, 4, 3)
    par = dict(objective='multi:softmax', num_class=4, depth=3, n_trees=1, learning_rate=0.3, max_num_bin=32, hist_mode='exact')
    a, b = Booster(d, **par), Booster(d, **par)
    a.set_feedback(y.astype(np.int32), np.ones(4000, np.float32))
    a.boost(1)
    b.boost(1)
    ta, tb = a.trees()[0], b.trees()[0]
    valid = tb['is_valid'].astype(bool)
    assert np.array_equal(ta['is_valid'], tb['is_valid'])
    assert np.array_equal(ta['split_feature_id'][valid], tb['split_feature_id'][valid]) and np.array_equal(ta['split_bid'][valid], tb['split_bid'][valid])
    # a probability of 1/4 is off by 2^-22 + 4 steps at most, then by one step of the grid
    assert np.abs(ta['sum_g'] - tb['sum_g'])[valid].max() <= 4000 * (2.0 ** -17 + 2.0 ** -22)


@pytest.mark.parametrize('classes', [6, 45, 300])
def test_rows_do_not_depend_on_their_neighbours(gpu, classes):
    import torch
    from thundergbm_b200 import scores
    r = np.random.default_rng(classes)
    n = 3003
    z = torch.from_numpy((r.standard_normal((classes, n)) * 2).astype(np.float32)).cuda().t()
    drawn, gains, old = (torch.from_numpy(v).cuda() for v in _logged(r, n, classes, 3))
    whole = scores.feedback(z, drawn, gains, old=old, clip=0.2, entropy=0.1, gives='pairs')
    for lo, hi in ((0, 1), (1, 40), (40, 1000), (1000, n)):
        part = scores.feedback(z[lo:hi].t().contiguous().t(), drawn[lo:hi], gains[lo:hi], old=old[lo:hi], clip=0.2, entropy=0.1, gives='pairs')
        assert all(torch.equal(a, b[lo:hi]) for a, b in zip(part, whole))


@pytest.mark.parametrize('sparse', [False, True])
@pytest.mark.parametrize('n,classes', [(1, 5), (900, 5), (700, 40)])
def test_predict_sample(gpu, sparse, n, classes):
    import scipy.sparse as sp
    from thundergbm_b200.thundergbm import TGBMClassifier
    d, x, y, _ = _data(1200, 6, classes, classes)
    m = TGBMClassifier(depth=4, n_trees=5, learning_rate=0.4, objective='multi:softprob', verbose=0)
    m.fit(x, y)
    rows = sp.csr_matrix(x[:n]) if sparse else x[:n]
    all_ids, all_values, _ = m.predict_top(rows, classes)
    s = np.zeros((n, classes), np.float32)
    np.put_along_axis(s, all_ids, all_values, 1)
    r = np.random.default_rng(n)
    for u, limits in ((r.random(n), {}), (r.random((n, 3)), dict(temperature=0.7, top_k=3)), (r.random((n, 2)), dict(top_p=0.8, min_p=0.05)), (r.random(n), dict(temperature=0.0))):
        ids, logs, every = m.predict_sample(rows, u, **limits)
        want = ref.sample(s, u, **limits)
        assert np.array_equal(ids, want[0])
        assert (np.abs(logs - want[1]) <= want[3]).all() and (np.abs(every - want[2]) <= want[4]).all()
    allowed = r.random((n, classes)) < 0.6
    allowed[:, 0] |= ~allowed.any(1)
    ids, logs, every = m.predict_sample(rows, r.random((n, 8)), allowed=allowed, bias=np.linspace(-1, 1, classes))
    assert np.take_along_axis(allowed, ids, 1).all() and (logs <= 0).all() and np.array_equal(logs, every)


def test_a_bandit_from_end_to_end(gpu):
    """A model draws classes, they earn gains, another model learns from them (and an fp32 and a sparse one run as well)."""
    import scipy.sparse as sp
    from thundergbm_b200.thundergbm import TGBMClassifier
    d, x, y, _ = _data(2000, 6, 5, 9)
    first = TGBMClassifier(depth=3, n_trees=3, objective='multi:softprob', verbose=0).fit(x, y)
    r = np.random.default_rng(0)
    drawn, logs, _ = first.predict_sample(x, r.random((2000, 4)), temperature=1.5)
    assert drawn.shape == (2000, 4) and (drawn >= 0).all() and (logs <= 0).all()
    gains = np.where(drawn == y[:, None].astype(int), 1.0, -0.25)
    for rows in (x, sp.csr_matrix(x)):
        second = TGBMClassifier(depth=3, n_trees=6, objective='multi:softprob', verbose=0)
        second.fit(rows, y, feedback=dict(classes=drawn, gains=gains, old=logs, clip=0.5, entropy=0.01))
        p = second.predict(rows)
        assert np.isfinite(p).all() and p.shape == (2000, 5)


def test_refusals(gpu):
    from thundergbm_b200.booster import Booster
    from thundergbm_b200.thundergbm import TGBMClassifier, TGBMRegressor
    d, x, y, logits = _data(200, 4, 3, 1)
    par = dict(num_class=3, depth=2, n_trees=2)
    c, g = np.zeros(200, np.int32), np.zeros(200, np.float32)
    b = Booster(d, objective='multi:softmax', **par)
    for bad in (dict(classes=c[:5]), dict(gains=g[:, None]), dict(old=g[:3]), dict(weights=g[:3]), dict(classes=np.zeros((200, 2), np.int32))):
        with pytest.raises(ValueError):
            b.set_feedback(**{**dict(classes=c, gains=g), **bad})
    for bad in (dict(temperature=0.0), dict(clip=-0.1), dict(clip=(1.5, 0.0)), dict(entropy=-1.0), dict(classes=np.zeros((200, 129), np.int32), gains=np.zeros((200, 129)))):
        with pytest.raises(RuntimeError):
            b.set_feedback(**{**dict(classes=c, gains=g), **bad})
    with pytest.raises(RuntimeError):
        b.feedback_loss()
    b.set_teacher(np.zeros((200, 1), np.int32), np.zeros((200, 1), np.float32))
    with pytest.raises(RuntimeError):
        b.set_feedback(c, g)
    b = Booster(d, objective='multi:softmax', **par)
    b.set_feedback(c, g)
    with pytest.raises(RuntimeError):
        b.set_teacher(np.zeros((200, 1), np.int32), np.zeros((200, 1), np.float32))
    b.boost(1)
    with pytest.raises(RuntimeError):
        b.set_feedback(c, g)
    with pytest.raises(RuntimeError):
        Booster(d, objective='reg:linear', depth=2, n_trees=2).set_feedback(c, g)
    for model, more in ((TGBMRegressor(verbose=0), {}), (TGBMClassifier(verbose=0, n_gpus=2), {}), (TGBMClassifier(verbose=0), dict(teacher=dict(ids=c, logits=g)))):
        with pytest.raises(ValueError):
            model.fit(x, y, feedback=dict(classes=c, gains=g), **more)
    m = TGBMClassifier(depth=2, n_trees=2, verbose=0).fit(x, y)
    for bad in (dict(uniform=g[:3]), dict(uniform=np.zeros((200, 129))), dict(uniform=np.zeros((200, 0)))):
        with pytest.raises(ValueError):
            m.predict_sample(x, **bad)
    for bad in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=2.0), dict(min_p=-0.5)):
        with pytest.raises(RuntimeError):
            m.predict_sample(x, g, **bad)
