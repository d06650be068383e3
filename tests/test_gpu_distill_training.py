"""Training from a teacher's largest scores and the best classes of a row under rules, through the public entry points: the gradients that
trees were grown on are those of the definition (tests/scores_ref.py), round after round, and the pieces run together."""
import numpy as np
import pytest

import scores_ref as ref

pytestmark = pytest.mark.gpu


def _data(n, f, classes, seed):
    from thundergbm_b200.synth import dense_to_csr
    r = np.random.default_rng(seed)
    x = r.integers(1, 40, (n, f)).astype(np.float32)
    y = (r.random((n, classes)) + 0.1 * x[:, :1] * np.arange(classes) / classes).argmax(1).astype(np.float32)
    y[:classes] = np.arange(classes)
    logits = r.standard_normal((n, classes)) * 2 + (x[:, 1:2] / 20 - 1) * np.linspace(-1, 1, classes)
    return dense_to_csr(x, y), x, y, logits


def _keep(logits, k, T):
    ids = np.argsort(-logits, axis=1, kind='stable')[:, :k].astype(np.int32)
    m = logits.max(1, keepdims=True)
    lse = (m[:, 0] / T + np.log(np.exp((logits - m) / T).sum(1))).astype(np.float32)
    return ids, np.take_along_axis(logits, ids, 1).astype(np.float32), lse


@pytest.mark.parametrize('n,classes,k,T,alpha,with_lse', [(3000, 3, 2, 1.0, 1.0, True), (2500, 7, 3, 2.0, 0.6, False), (1500, 40, 8, 1.5, 0.8, True),
                                                          (700, 40, 40, 1.0, 0.5, False), (9000, 5, 3, 2.0, 0.7, True)])
@pytest.mark.parametrize('mode', ['exact', 'fp32'])
def test_nodes_hold_the_gradients_of_the_definition(gpu, n, classes, k, T, alpha, with_lse, mode):
    """The root of every tree of a round holds the sum of the gradients at the scores of the round before.  A value is rounded to a grid
    of 2^-18 (exact) or finer of a power of two above the round's largest, which is at most 2 alpha T + 2; the sum is then a float."""
    from thundergbm_b200.booster import Booster
    d, x, y, logits = _data(n, 6, classes, n + classes)
    ids, kept, lse = _keep(logits, k, T)
    lse = lse if with_lse else None
    rounds = 4
    for stop in range(1, rounds + 1):   # (from the second round on a boosting round is a graph that is replayed)
        b = Booster(d, objective='multi:softprob', num_class=classes, depth=4, n_trees=rounds, learning_rate=0.5, max_num_bin=64, hist_mode=mode)
        b.set_teacher(ids, kept, lse, T, alpha)
        s = np.zeros((classes, n), np.float32)
        if stop > 1:
            b.boost(stop - 1)
            s = b.ypred()
        loss = b.teacher_loss()
        b.boost(1)
        trees = b.trees()[stop - 1]
        want = ref.distill(s.T, ids, kept, lse, y.astype(np.int32), None, T, alpha)
        scale = (T + 1) * 2.0 * 2.0 ** -17 * n
        for c in range(classes):
            for name, g, off in (('sum_g', want['g'][:, c], want['g_off'][:, c]), ('sum_h', want['h'][:, c], want['h_off'][:, c])):
                got = float(trees[c][0][name])
                assert abs(got - g.sum()) <= off.sum() + scale + 2.0 ** -22 * abs(g).sum(), (stop, c, name)
        assert abs(loss - want['loss'].mean()) <= want['loss_off'].mean() + 2.0 ** -40 * abs(want['loss']).sum()
        b.close()


def test_a_certain_teacher_is_a_label(gpu):
    """alpha = 1 and a teacher that gives all mass to the label: the gradients of the softmax objective, and its first trees' splits."""
    from thundergbm_b200.booster import Booster
    d, x, y, _ = _data(4000, 5, 4, 3)
    par = dict(objective='multi:softmax', num_class=4, depth=3, n_trees=1, learning_rate=0.3, max_num_bin=32, hist_mode='exact')
    a, b = Booster(d, **par), Booster(d, **par)
    a.set_teacher(y.astype(np.int32)[:, None], np.zeros((4000, 1), np.float32))
    a.boost(1)
    b.boost(1)
    ta, tb = a.trees()[0], b.trees()[0]
    valid = tb['is_valid'].astype(bool)
    assert np.array_equal(ta['is_valid'], tb['is_valid'])
    assert np.array_equal(ta['split_feature_id'][valid], tb['split_feature_id'][valid]) and np.array_equal(ta['split_bid'][valid], tb['split_bid'][valid])
    # a probability of 1/4 is off by 2^-22 + 4 steps at most, then by one step of the grid
    assert np.abs(ta['sum_g'] - tb['sum_g'])[valid].max() <= 4000 * (2.0 ** -17 + 2.0 ** -22)


@pytest.mark.parametrize('classes', [6, 45])
def test_rows_do_not_depend_on_their_neighbours(gpu, classes):
    """A row's gradients are the same bits whatever rows it is computed with: trainings on parts of the rows add up to one on all of them."""
    import torch
    from thundergbm_b200 import scores
    r = np.random.default_rng(classes)
    z = torch.from_numpy((r.standard_normal((classes, 5003)) * 2).astype(np.float32)).cuda().t()
    v, i, lse = scores.top(torch.from_numpy((r.standard_normal((5003, classes)) * 2).astype(np.float32)).cuda(), min(classes, 9))
    whole = scores.distill(z, i, v, lse=lse, gives='pairs')
    for lo, hi in ((0, 1), (1, 40), (40, 1000), (1000, 5003)):
        part = scores.distill(z[lo:hi].t().contiguous().t(), i[lo:hi], v[lo:hi], lse=lse[lo:hi].contiguous(), gives='pairs')
        assert torch.equal(part[0], whole[0][lo:hi]) and torch.equal(part[1], whole[1][lo:hi])


@pytest.mark.parametrize('sparse', [False, True])
@pytest.mark.parametrize('n,classes', [(1, 5), (900, 5), (700, 40)])
def test_predict_top(gpu, sparse, n, classes):
    import scipy.sparse as sp
    from thundergbm_b200.booster import predict_raw
    from thundergbm_b200.thundergbm import TGBMClassifier
    d, x, y, _ = _data(1200, 6, classes, classes)
    m = TGBMClassifier(depth=4, n_trees=5, learning_rate=0.4, objective='multi:softprob', verbose=0)
    m.fit(x, y)
    rows = x[:n]
    prob = m.predict(rows).reshape(classes, n).T.astype(np.float64)   # (the front end reshapes a buffer by class)
    given = sp.csr_matrix(rows) if sparse else rows
    ids, values, lse = m.predict_top(given, 4, temperature=1.0)
    p = np.exp(values.astype(np.float64) - lse[:, None])
    # probabilities: two ways of computing them, each off by the steps of a few operations on numbers below 2^5
    assert np.abs(p - np.take_along_axis(prob, ids, 1)).max() <= 2.0 ** -18
    assert np.array_equal(ids[:, 0], prob.argmax(1)) or np.abs(prob.max(1) - np.take_along_axis(prob, ids[:, :1], 1)[:, 0]).max() <= 2.0 ** -18
    # under rules: the definition on the scores that come back without any
    all_ids, all_values, _ = m.predict_top(given, classes)
    s = np.zeros((n, classes), np.float32)
    np.put_along_axis(s, all_ids, all_values, 1)
    r = np.random.default_rng(n)
    bias = r.standard_normal(classes).astype(np.float32)
    allowed = r.random((3, classes)) < 0.7
    row = r.integers(-1, 3, n)
    past = [r.integers(0, classes, r.integers(0, 6)).tolist() for _ in range(n)]
    ptr = np.concatenate([[0], np.cumsum([len(h) for h in past])])
    flat = np.array([c for h in past for c in h], np.int32)
    par = dict(repetition=1.2, frequency=0.1, presence=0.3)
    ids, values, lse = m.predict_top(given, 3, bias=bias, allowed=allowed, allowed_row=row, history=past, temperature=1.5, **par)
    want, off = ref.adjust(s, bias, allowed, row, (ptr, flat), **par)
    for i in range(n):
        order = np.sort(want[i])[::-1][:3]
        assert np.allclose(values[i][order > -np.inf], order[order > -np.inf], rtol=0, atol=off[i].max() + 2.0 ** -22 * np.abs(s[i]).max() + 1e-7)
        assert (ids[i][order == -np.inf] == -1).all() and allowed[row[i]][ids[i][ids[i] >= 0]].all() if row[i] >= 0 else True
    if n > 1:
        raw_ids, raw_values, _ = m.predict_top(rows[: n // 2], 4)
        again, values2, _ = m.predict_top(rows, 4)
        assert np.array_equal(raw_ids, again[: n // 2]) and np.array_equal(raw_values, values2[: n // 2])


def test_teacher_and_student_together(gpu, tmp_path):
    """A large model's best classes train a small one: fit, predict_top under rules, fit from it, save and load."""
    from thundergbm_b200.thundergbm import TGBMClassifier
    d, x, y, _ = _data(3000, 8, 12, 5)
    big = TGBMClassifier(depth=6, n_trees=12, learning_rate=0.3, objective='multi:softprob', verbose=0)
    big.fit(x, y)
    ids, logits, lse = big.predict_top(x, 5, bias=np.linspace(-0.5, 0.5, 12), temperature=2.0)
    small = TGBMClassifier(depth=3, n_trees=4, learning_rate=0.3, objective='multi:softprob', verbose=0)
    small.fit(x, y + 100, teacher=dict(ids=ids, logits=logits, lse=lse, temperature=2.0, alpha=0.7))
    assert small.group_label == [100.0 + c for c in range(12)] and small.tree_per_iter == 12
    p = small.predict(x)
    assert p.shape == (3000, 12) and np.isfinite(p).all()
    small.save_model(tmp_path / 'small')
    other = TGBMClassifier(objective='multi:softprob', verbose=0)
    other.load_model(tmp_path / 'small')
    assert all(np.array_equal(a, b) for a, b in zip(other.predict_top(x, 3), small.predict_top(x, 3)))
    for method in ('exact', 'hist'):
        m = TGBMClassifier(depth=3, n_trees=2, objective='multi:softmax', verbose=0, tree_method=method, bagging=1)
        m.fit(x, y, teacher=dict(ids=ids, logits=logits))
        assert set(m.predict(x)) <= set(range(12))


def test_no_teacher_leaves_training_as_it_was(gpu):
    """A booster that was refused a teacher grows the trees of one that never heard of it."""
    from thundergbm_b200.booster import Booster
    d, x, y, logits = _data(2000, 5, 4, 8)
    par = dict(objective='multi:softmax', num_class=4, depth=4, n_trees=3, hist_mode='exact')
    a, b = Booster(d, **par), Booster(d, **par)
    with pytest.raises(RuntimeError):
        a.set_teacher(np.zeros((2000, 1), np.int32), np.zeros((2000, 1), np.float32), temperature=-1.0)
    a.boost(3)
    b.boost(3)
    assert a.trees().tobytes() == b.trees().tobytes()


def test_refusals(gpu):
    from thundergbm_b200.booster import Booster
    from thundergbm_b200.thundergbm import TGBMClassifier, TGBMRegressor
    d, x, y, logits = _data(500, 5, 4, 9)
    ids, kept, lse = _keep(logits, 3, 1.0)
    b = Booster(d, objective='multi:softmax', num_class=4, depth=3, n_trees=3)
    with pytest.raises(RuntimeError, match='no teacher'):
        b.teacher_loss()
    for bad in (dict(alpha=1.5), dict(alpha=float('nan')), dict(temperature=0.0), dict(temperature=float('inf'))):
        with pytest.raises(RuntimeError):
            b.set_teacher(ids, kept, lse, **bad)
    for bad in ((ids[:10], kept[:10]), (ids, kept[:, :2]), (ids[:, 0], kept[:, 0]), (ids, kept, lse[:5])):
        with pytest.raises(ValueError):
            b.set_teacher(*bad)
    with pytest.raises(RuntimeError, match='128'):
        b.set_teacher(np.zeros((500, 129), np.int32), np.zeros((500, 129), np.float32))
    b.boost(1)
    with pytest.raises(RuntimeError, match='first round'):
        b.set_teacher(ids, kept)
    with pytest.raises(RuntimeError, match='multi'):
        Booster(d, objective='reg:linear', depth=3, n_trees=1).set_teacher(ids, kept)
    teacher = dict(ids=ids, logits=kept)
    for model, t in ((TGBMRegressor(verbose=0), teacher), (TGBMClassifier(n_gpus=2, verbose=0), teacher), (TGBMClassifier(verbose=0), dict(ids=ids[:3], logits=kept[:3])),
                     (TGBMClassifier(verbose=0, tree_method='none'), teacher)):
        with pytest.raises(ValueError):
            model.fit(x, y, teacher=t)
    m = TGBMClassifier(depth=3, n_trees=2, verbose=0)
    with pytest.raises(ValueError, match='train'):
        m.predict_top(x)
    m.fit(x, y)
    for bad in (dict(k=0), dict(k=200), dict(bias=np.zeros(3)), dict(allowed=np.ones((500, 3))), dict(allowed=np.ones((2, 4))), dict(allowed_row=np.zeros(500)),
                dict(history=[[0]])):
        with pytest.raises(ValueError):
            m.predict_top(x, **bad)
    for bad in (dict(temperature=0.0), dict(history=[[0]] * 500, repetition=0.0), dict(history=[[0]] * 500, presence=float('nan'))):
        with pytest.raises(RuntimeError):
            m.predict_top(x, **bad)
    one = TGBMClassifier(depth=3, n_trees=2, verbose=0, objective='binary:logistic')
    one.fit(x, (y > 1).astype(np.float32))
    with pytest.raises(RuntimeError, match='several classes'):
        one.predict_top(x)
