"""Drawing classes and learning from draws at numbers where float arithmetic ends or draws leave their range; definitions and bounds are those of
tests/draws_ref.py, or stand beside the test."""
import numpy as np
import pytest

import draws_ref as ref
from scores_ref import HALF, U
from test_gpu_draws import _check_sample, _dev, _masked
from test_gpu_scores import _close, _given, _make, _tensor, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def _check_far(ops, t, kind, classes, gains, gives, **more):
    torch, scores = ops
    want = ref.feedback(_given(t), classes, gains, **more)
    loss, logs, grad = scores.feedback(t, _dev(torch, classes), _dev(torch, gains), gives=gives, **more)
    _close(loss.cpu().numpy(), want['loss'], want['loss_off'], 'loss')
    _close(logs.cpu().numpy(), want['logs'], want['logs_off'], 'logs')
    if gives == 'gradient':
        _close(_given(grad), want['g'], want['g_off'] + (HALF[kind] * np.abs(want['g']) * (1 + 2.0 ** -8) if kind != 'f32' else 0), 'gradient')
    else:
        _close(grad.cpu().numpy()[..., 0], want['g'], want['g_off'], 'g')
        _close(grad.cpu().numpy()[..., 1], want['h'], want['h_off'], 'h')


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


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('layout,n,k', [('class', 40, 5), ('class', 40, 200), ('class', 40, 600), ('class', 3, 1500), ('row', 1100, 300), ('row', 6, 300), ('row', 3, 3000),
                                        ('row', 3, 20000), ('row+', 3, 20001), ('row', 3, 131072), ('any', 3, 300)])
def test_numbers_that_are_not_below_one(ops, layout, n, k, kind):
    """They are taken as the largest number below 1.  The likely classes have 1 each and the others e^-60, so that all sums of doubles are whole numbers
    and nothing behind the last likely class counts."""
    torch, scores = ops
    likely = min(96, k // 2)
    z = np.full((n, k), -60.0)
    z[:, :likely] = 0
    z[1, :] = -60
    z[1, k - likely:] = 0
    t = _tensor(torch, z, kind, layout)
    u = np.tile([1.0, 1 - 2.0 ** -53, 7.0, np.inf], (n, 1))
    for limits in ({}, dict(top_k=k - 1), dict(top_p=0.9999999), dict(min_p=1e-30), dict(top_k=likely), dict(top_k=np.resize([0, likely], n).astype(np.int32))):
        given = {name: _dev(torch, v) if isinstance(v, np.ndarray) else v for name, v in limits.items()}
        for at in (u, u[:, :1], u.astype(np.float32)):
            ids, logs, every = scores.sample(t, _dev(torch, at), **given)
            want = np.full(at.shape, likely - 1)
            want[1] = k - 1
            assert np.array_equal(ids.cpu().numpy(), want), limits
            for got in (logs, every):
                _close(got.cpu().numpy(), np.full(at.shape, -np.log(likely)), 2.0 ** -22, limits)


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('k', [40000, 40001])
def test_feedback_where_a_block_has_only_masked_classes(ops, k, kind):
    """Thousands of neighbouring classes at the type's lowest number: their part of the entropy's sum is 0, not 0 times infinity."""
    torch, scores = ops
    r = np.random.default_rng(k)
    z = np.full((3, k), float(torch.finfo(torch.float32 if kind == 'f32' else torch.bfloat16).min))
    z[0, :3000], z[1, 30000:31000], z[2, ::4000] = r.standard_normal(3000), r.standard_normal(1000), 1.0
    t = _tensor(torch, z, kind, 'row')
    classes, gains = np.array([[0, 10], [30001, 30002], [4000, 8000]], np.int32), np.ones((3, 2), np.float32)
    for gives in ('gradient', 'pairs'):
        _check_far(ops, t, kind, classes, gains, gives, entropy=0.05)


@pytest.mark.parametrize('gives', ['gradient', 'pairs'])
@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('layout,n,k', [('class', 5, 5), ('class', 5, 200), ('row', 5, 5), ('row', 5, 200), ('row', 5, 2000), ('row', 5, 9000), ('row+', 5, 9000), ('any', 5, 40)])
def test_feedback_of_classes_masked_by_the_lowest_number(ops, layout, n, k, kind, gives):
    """A share of 0 times what a class so far away would earn for the row's entropy is 0."""
    torch, scores = ops
    r = np.random.default_rng(k)
    z = r.standard_normal((n, k))
    low = float(torch.finfo(torch.float32 if kind == 'f32' else torch.bfloat16).min)
    z[:, 1::2] = low
    z[3, 2] = -np.inf
    t = _tensor(torch, z, kind, layout)
    classes, gains = np.array([[0, 2, -1]] * n, np.int32), r.standard_normal((n, 3)).astype(np.float32)
    _check_far(ops, t, kind, classes, gains, gives, temperature=0.2, entropy=0.05)


@pytest.mark.parametrize('layout,n,k', [('class', 5, 5), ('class', 5, 200), ('row', 5, 5), ('row', 5, 200), ('row', 5, 9000), ('row+', 5, 9000), ('any', 5, 40)])
def test_feedback_at_small_temperatures(ops, layout, n, k):
    """entropy / T^2 times a distance that stands for infinity must not be infinite."""
    torch, _ = ops
    r = np.random.default_rng(k)
    z = _masked(r, r.standard_normal((n, k))) * 2.0 ** -17
    t = _tensor(torch, z, 'f32', layout)
    classes, gains = np.array([[0, 2, 1]] * n, np.int32), r.standard_normal((n, 3)).astype(np.float32)
    for gives in ('gradient', 'pairs'):
        _check_far(ops, t, 'f32', classes, gains, gives, temperature=2.0 ** -17, entropy=0.5)


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('layout,n,k', [('class', 40, 6), ('class', 40, 200), ('class', 9, 700), ('row', 9, 6), ('row', 9, 200), ('row', 9, 3000), ('row', 9, 3001), ('any', 9, 40), ('class', 9, 1500)])
def test_norm_leaves_masked_classes_masked(ops, layout, n, k, kind):
    """Also where the variance of the others is more than a float holds (their deviation counts as infinite, so they are 0), or their sum is."""
    torch, scores = ops
    z = np.random.default_rng(k).standard_normal((n, k))
    low = float(torch.finfo(torch.float32 if kind == 'f32' else torch.bfloat16).min)
    z[:, 3] = -np.inf
    z[0, 0], z[0, 1] = 1e20, -1e20
    z[1, 0] = low
    z[2, 0] = z[2, 1] = low
    t = _tensor(torch, z, kind, layout)
    gone = _given(t) == -np.inf
    for gain in (None, torch.ones(k, device='cuda')):
        y, mean, rstd = scores.norm(t, gain)
        y = _given(y)
        assert (y[gone] == -np.inf).all()
        assert (rstd[:2] == 0).all() and (y[:2][~gone[:2]] == 0).all() and np.isfinite(y[3:][~gone[3:]]).all()


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('layout,n,k', [('class', 70, 6), ('class', 70, 30), ('class', 70, 250), ('class', 70, 700), ('row', 70, 30), ('row', 1100, 250), ('row', 30, 250), ('row', 5, 9001),
                                        ('row', 5, 70000), ('any', 9, 40)])
def test_logs_among_all_classes(ops, layout, n, k, kind):
    """Their mass is a sum of doubles under all limits: the logs are rounded once, no class is likelier among all than among those that are
    left, and what a row gets does not depend on the limits of its neighbours."""
    torch, scores = ops
    r = np.random.default_rng(k)
    z = _masked(r, _make(r, n, k))
    z[3] = -30
    z[3, k // 2] = 0      # nearly all of the mass
    z[4] = np.where(np.arange(k) % 2, 0.0, -1.0)
    t = _tensor(torch, z, kind, layout)
    u = r.random((n, 3))
    rows = dict(temperature=r.choice([0.5, 1.0, 2.0], n).astype(np.float32), top_k=r.choice([0, 1, 2, 20, 2 * k], n).astype(np.int32),
                top_p=r.choice([1.0, 0.4, 0.9], n).astype(np.float32), min_p=r.choice([0.0, 0.01, 1.0], n).astype(np.float32))
    for limits in ({}, dict(top_k=max(1, k // 3)), dict(min_p=0.001), dict(top_p=0.8), dict(top_k=5, top_p=0.9, min_p=1e-4, temperature=0.7), rows):
        given = {name: _dev(torch, v) if isinstance(v, np.ndarray) else v for name, v in limits.items()}
        ids, logs, every = scores.sample(t, _dev(torch, u), **given)
        want = ref.sample(_given(t), u, **limits)
        assert np.array_equal(ids.cpu().numpy(), want[0])
        exact = want[2]
        _close(every.cpu().numpy(), exact, 2.0 ** -32 + U * (1 + 2.0 ** -18) * np.abs(np.where(np.isfinite(exact), exact, 0)), limits)
        assert bool(((every <= logs) | every.isnan()).all())
        for i in (0, 3, 31, 32, n - 1):
            if i >= n or layout == 'row' and n > 1000:   # (one row alone is another kernel's)
                continue
            one = slice(i, i + 1)
            alone = scores.sample(t[one], _dev(torch, u)[one], **{name: v[one] if isinstance(v, torch.Tensor) else v for name, v in given.items()})
            assert all(torch.equal(a.nan_to_num(nan=9.0), b[one].nan_to_num(nan=9.0)) for a, b in zip(alone, (ids, logs, every))), (i, limits)


@pytest.mark.parametrize('layout,n,k', [('class', 40, 5), ('class', 40, 200), ('class', 9, 700), ('row', 9, 5), ('row', 1100, 200), ('row', 9, 200), ('row', 5, 9001), ('row', 5, 70000),
                                        ('any', 9, 40), ('class', 9, 1500)])
def test_sample_at_the_largest_and_smallest_temperatures(ops, layout, n, k):
    """Differences of scores above 3.4e38 and below 2^-126 at temperatures to match: e^-6 is e^-6."""
    torch, _ = ops
    r = np.random.default_rng(k)
    unit = r.uniform(-1, 1, (n, k))
    unit[0] = np.where(np.arange(k) % 3, 1, -1)
    unit[1, 0], unit[1, 1] = 1, -1
    u = r.random((n, 3))
    for size, temperatures in ((3.3e38, (1e38, 3e37)), (3e-40, (1e-40, 3e-41))):
        t = _tensor(torch, unit * size, 'f32', layout)
        for limits in ({}, dict(top_k=max(1, k // 2)), dict(top_p=0.9), dict(top_p=0.2), dict(min_p=0.01), dict(min_p=0.01, top_p=0.7, top_k=k - 1)):
            for T in temperatures:
                _check_sample(ops, t, u, dict(limits, temperature=T), (layout, k, T, str(limits)))


@pytest.mark.parametrize('layout,n,k', [('class', 5, 5), ('class', 5, 200), ('row', 5, 5), ('row', 5, 200), ('row', 5, 3000), ('any', 5, 40)])
def test_feedback_of_gains_and_logs_that_are_none(ops, layout, n, k):
    """A NaN among what a draw that counts came with is told by the row's loss and gradient, and by no other row's."""
    torch, scores = ops
    nan = float('nan')
    z = _tensor(torch, np.random.default_rng(k).standard_normal((n, k)), 'f32', layout)
    c = torch.tensor([[0, 1], [0, 1], [2, -1], [2, 3], [4, 4]], dtype=torch.int32, device='cuda')
    gains = torch.tensor([[nan, 1.0], [1, 1], [1, nan], [1, 1], [1, 1]], device='cuda')
    old = torch.tensor([[-1.0, -1], [-1, nan], [-1, nan], [-1, -1], [-1, nan]], device='cuda')
    weights = torch.tensor([1.0, 1, 1, 1, 0], device='cuda')
    for gives in ('gradient', 'pairs'):
        loss, logs, grad = scores.feedback(z, c, gains, old=old, weights=weights, clip=0.2, gives=gives)
        g = grad if gives == 'gradient' else grad[..., 0]
        assert loss[:2].isnan().all() and g[:2].isnan().all()
        assert loss[2:].isfinite().all() and g[2:].isfinite().all() and loss[4] == 0 and not g[4].any()
        assert logs[:2].isfinite().all()


def test_counts_that_32_bits_do_not_hold_are_refused(ops):
    """2^32 + 3 is not 3, and -2^32 does not mean all."""
    torch, scores = ops
    from thundergbm_b200.thundergbm import TGBMClassifier
    z, u = torch.zeros(4, 9, device='cuda'), torch.rand(4, device='cuda')
    x = np.random.default_rng(1).random((60, 3)).astype(np.float32)
    model = TGBMClassifier(depth=2, n_trees=2, verbose=0).fit(x, np.arange(60) % 3)
    for top_k in (2 ** 31, 2 ** 32 + 3, -2 ** 32, -2 ** 40, 2.5, float('inf'), float('nan')):
        with pytest.raises(ValueError, match='whole number'):
            scores.sample(z, u, top_k=top_k)
        with pytest.raises(ValueError, match='whole number'):
            model.predict_sample(x, np.zeros(60), top_k=top_k)
    model.predict_sample(x, np.zeros(60), top_k=np.int64(2))
