"""Drawing classes from scores and learning from draws (sample, feedback, norm, norm_backward of thundergbm_b200/scores.py) against
their definitions in 64 bits: layouts, types, sizes where kernels change over, masks that leave nothing, ties, infinities; bounds are
those of tests/draws_ref.py, which count the roundings."""
import numpy as np
import pytest

import draws_ref as ref
from scores_ref import HALF, TINY
from test_gpu_scores import SIZES, TYPES, _close, _given, _make, _tensor, _type, ops  # noqa: F401

pytestmark = pytest.mark.gpu
LAYOUTS = ['row', 'class', 'row+', 'class+', 'any']


def _dev(torch, x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()


def _masked(r, z, share=0.15):
    """masked classes; where there are rows enough one without a class, one with a single one, one of equal scores"""
    n, k = z.shape
    z = z.copy()
    z[r.random((n, k)) < share] = -np.inf
    if n > 2:
        z[n // 2] = -np.inf
        z[n - 1] = -np.inf
        z[n - 1, k // 2] = 0.75
        z[0] = 1.5
    return z


def _check_sample(ops, t, u, limits, what):
    torch, scores = ops
    given = {name: _dev(torch, v) if isinstance(v, np.ndarray) else v for name, v in limits.items()}
    before = t.clone()
    got = scores.sample(t, _dev(torch, u), **given)
    assert torch.equal(t.nan_to_num(nan=9.0), before.nan_to_num(nan=9.0))
    assert got[0].dtype == torch.int32 and got[1].dtype == got[2].dtype == torch.float32 and all(x.shape == u.shape for x in got)
    ids, logs, every, off, all_off = ref.sample(_given(t), u, **limits)
    assert np.array_equal(got[0].cpu().numpy(), ids), what
    _close(got[1].cpu().numpy(), logs, off, what + ('logs',))
    _close(got[2].cpu().numpy(), every, all_off, what + ('all logs',))
    return ids


@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('n,k', SIZES)
def test_sample(ops, n, k, layout):
    torch, _ = ops
    r = np.random.default_rng(n * 1000 + k + 5)
    for kind, m, ties, limits in (('f32', 1, False, {}), ('bf16', 3, False, dict(temperature=0.7)), ('f16', 1, True, dict(top_k=max(1, k // 3), temperature=1.3)),
                                  ('f32', 1, True, dict(top_p=0.8)), ('bf16', 33, False, dict(min_p=0.03, top_p=0.9)), ('f32', 2, True, dict(top_k=7, top_p=0.6, min_p=0.01)),
                                  ('f16', 128, False, dict(top_p=0.95, temperature=2.0)),
                                  ('f32', 5, False, dict(temperature=r.choice([0.0, 0.5, 1.0, 3.0], n).astype(np.float32),
                                                         top_k=r.choice([0, 1, 2, 20, 2 * k], n).astype(np.int32),
                                                         top_p=r.choice([1.0, 0.0, 0.4, 0.9], n).astype(np.float32),
                                                         min_p=r.choice([0.0, 0.1, 1.0], n).astype(np.float32)))):
        t = _tensor(torch, _masked(r, _make(r, n, k, ties)), kind, layout)
        u = r.random((n, m)) if m > 1 else r.random(n)
        _check_sample(ops, t, u if kind != 'f16' else u.astype(np.float32), limits, (kind, m, ties))


@pytest.mark.parametrize('layout,n,k', [('class', 9, 6), ('class', 9, 100), ('class', 9, 2000), ('row', 9, 6), ('row', 9, 300), ('row', 9, 9001), ('any', 9, 50)])
def test_sample_borders_that_are_exact(ops, layout, n, k):
    """Equal scores have equal masses, and their sums are exact: borders between classes, at and between them."""
    torch, scores = ops
    z = np.full((n, k), -3.25)
    t = _tensor(torch, z, 'bf16', layout)
    m = min(k, 64)
    at = np.linspace(0, k - 1, m).astype(int)
    u = np.tile(at / k, (n, 1))
    u = np.where(np.floor(u * k) < at, np.nextafter(u, 1), u)   # (at / k * k may round below at)
    got = scores.sample(t, _dev(torch, u))[0].cpu().numpy()
    assert np.array_equal(got, np.tile(at, (n, 1)))
    # what no number in [0, 1) is: the nearest one that is
    u = np.tile(np.array([0.0, -1.0, np.nan, 1.0, 7.0, np.inf, 1 - 2.0 ** -53]), (n, 1))
    got = scores.sample(t, _dev(torch, u))[0].cpu().numpy()
    assert np.array_equal(got, np.tile([0, 0, 0, k - 1, k - 1, k - 1, k - 1], (n, 1)))
    # of equal ones the lower classes are left, as many as it takes
    half = scores.sample(t, _dev(torch, u), top_p=0.5)[0].cpu().numpy()
    assert half.max() == (k + 1) // 2 - 1 and half.min() == 0
    few = scores.sample(t, _dev(torch, u), top_k=3)
    assert few[0].max() == min(3, k) - 1
    _close(few[1].cpu().numpy(), np.full((n, 7), -np.log(min(3, k))), 2.0 ** -24, 'logs')


@pytest.mark.parametrize('kind', TYPES)
@pytest.mark.parametrize('layout,n,k', [('class', 12, 5), ('class', 12, 100), ('class', 12, 3000 // 2), ('row', 12, 5), ('row', 12, 300), ('row', 12, 9001), ('any', 12, 40)])
def test_sample_of_unusual_numbers(ops, kind, layout, n, k):
    torch, _ = ops
    r = np.random.default_rng(k)
    low, high = float(torch.finfo(_type(torch, kind)).min), float(torch.finfo(_type(torch, kind)).max)
    z = _make(r, n, k)
    z[0] = low                               # masked by the type's lowest value, all of it
    z[1] = low
    z[1, k - 2] = 1.0
    z[2] = np.where(np.arange(k) % 2, 0.0, -0.0)
    z[3, 1] = np.nan
    z[4] = np.nan
    z[5, :] = -np.inf
    z[5, k - 1] = low
    z[6, k // 2] = np.inf
    z[7] = -np.inf
    z[8, 0], z[8, 1] = high, low
    z[9] = np.where(np.arange(k) == k - 1, -high, low)
    t = _tensor(torch, z, kind, layout)
    u = r.random((n, 3))
    for limits in ({}, dict(top_k=2), dict(top_p=0.7), dict(min_p=0.5), dict(temperature=0), dict(temperature=1e-30), dict(temperature=1e30), dict(temperature=1e-45, top_p=0.5), dict(temperature=1e-45, top_k=3), dict(temperature=2e-40, min_p=0.5),
                   dict(temperature=np.array([np.nan, -1, np.inf, 0, 1e-45, 1, 1, 1, 1, 1, 0, -0.0], np.float32)),
                   dict(top_p=np.array([np.nan, -1, 2, 0] * 3, np.float32), min_p=np.array([-1, 5, np.nan] * 4, np.float32),
                        top_k=np.array([-1, 1 << 30, 1, 0] * 3, np.int32))):
        want = {name: np.where(np.isnan(v), none, v) if isinstance(v, np.ndarray) else v
                for (name, v), none in zip(limits.items(), (1.0, 0.0, 0) if 'top_p' in limits else (np.nan,) * 3)}
        given = {name: _dev(torch, v) if isinstance(v, np.ndarray) else v for name, v in limits.items()}
        got = ops[1].sample(t, _dev(torch, u), **given)
        ids, logs, every, off, all_off = ref.sample(_given(t), u, **want)
        assert np.array_equal(got[0].cpu().numpy(), ids), limits
        _close(got[1].cpu().numpy(), logs, off, limits)
        _close(got[2].cpu().numpy(), every, all_off, limits)


def test_sample_draws_what_it_says(ops):
    """Shares of many draws against the probabilities that are given with them."""
    torch, scores = ops
    r = np.random.default_rng(3)
    z = np.tile(_make(r, 1, 37), (20000, 1))
    for layout in ('row', 'class'):
        t = _tensor(torch, z, 'f32', layout)
        ids, logs, _ = scores.sample(t, _dev(torch, r.random(20000)), top_p=0.9)
        share = torch.bincount(ids.long(), minlength=37).cpu().numpy() / 20000
        p = np.zeros(37)
        p[ids.cpu().numpy()] = np.exp(logs.cpu().numpy())
        assert abs(p.sum() - 1) < 1e-5 and (np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / 20000) + 1e-9).all()   # (five deviations)


# ------------------------------------------------------------------ feedback
def _draws(r, z, m, T, clip, **more):
    """logged draws; none where its ratio lies so near a bound that rounding decides on which side"""
    n, k = z.shape
    classes = r.integers(0, k, (n, m)).astype(np.int32)
    classes[r.random((n, m)) < 0.1] = -1
    classes[r.random((n, m)) < 0.05] = k + 2
    if m > 2:
        classes[::2, 1] = classes[::2, 0]      # the same class twice
    gains = r.standard_normal((n, m)).astype(np.float32)
    lp = ref.feedback(z, classes, gains, temperature=T)['logs']
    lp = np.where(np.isfinite(lp), lp, 0)
    old = (lp + 0.4 * r.standard_normal((n, m))).astype(np.float32)
    reference = (lp + 0.5 * r.standard_normal((n, m))).astype(np.float32)
    near = ref.feedback(z, classes, gains, old, temperature=T, clip=clip)['gap'] < 1e-3
    gains[near] = 0
    return classes, gains, old, reference


def _check_feedback(ops, t, kind, classes, gains, what, **more):
    torch, scores = ops
    want = ref.feedback(_given(t), classes, gains, **more)
    args = {name: _dev(torch, v) if isinstance(v, np.ndarray) else v for name, v in more.items()}
    c, g = _dev(torch, classes), _dev(torch, gains)
    for gives in ('loss', 'gradient', 'pairs'):
        loss, logs, grad = scores.feedback(t, c, g, gives=gives, **args)
        assert loss.shape == (t.size(0),) and logs.shape == c.shape and logs.dtype == loss.dtype == torch.float32
        _close(loss.cpu().numpy(), want['loss'], want['loss_off'], what + ('loss',))
        _close(logs.cpu().numpy(), want['logs'], want['logs_off'], what + ('logs',))
        if gives == 'loss':
            assert grad is None
        elif gives == 'gradient':
            assert grad.dtype == t.dtype and grad.shape == t.shape
            off = want['g_off'] + (HALF[kind] * np.abs(want['g']) * (1 + 2.0 ** -8) + TINY[kind] if kind != 'f32' else 0)
            _close(_given(grad), want['g'], off, what + ('gradient',))
        else:
            assert grad.dtype == torch.float32 and tuple(grad.shape) == (*t.shape, 2)
            p = grad.cpu().numpy()
            _close(p[..., 0], want['g'], want['g_off'], what + ('pairs g',))
            _close(p[..., 1], want['h'], want['h_off'], what + ('pairs h',))
    return want


@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('n,k', SIZES)
def test_feedback(ops, n, k, layout):
    torch, _ = ops
    r = np.random.default_rng(n * 1000 + k + 6)
    for kind, m, T, clip, kl, b, with_old, with_weights in (('f32', 1, 1.0, None, 0.0, 0.0, False, False), ('f32', 4, 0.7, (0.2, 0.3), 0.1, 0.05, True, True),
                                                            ('bf16', 1, 1.0, (0.2, 0.2), 0.05, 0.0, True, False), ('f16', 33, 2.0, (1.0, 0.5), 0.0, 0.3, True, True),
                                                            ('f32', 128, 1.0, (0.1, float('inf')), 0.2, 0.01, True, False)):
        z = _masked(r, _make(r, n, k))
        t = _tensor(torch, z, kind, layout)
        classes, gains, old, reference = _draws(r, _given(t), m, T, clip)
        weights = r.random(n).astype(np.float32) if with_weights else None
        if with_weights:
            weights[0] = 0
        _check_feedback(ops, t, kind, classes, gains, (kind, m, T), old=old if with_old else None, reference=reference if kl else None, weights=weights,
                        temperature=T, clip=clip, kl=kl, entropy=b)


@pytest.mark.parametrize('layout,n,k', [('class', 6, 5), ('class', 6, 200), ('row', 6, 5), ('row', 6, 200), ('row', 4, 2000), ('any', 4, 30)])
def test_feedback_against_differences(ops, layout, n, k):
    """The gradient against differences of the loss, which the same function gives: central ones, a step of 2^-7 on scores that are
    multiples of it; the third derivative of the loss is below 4 here, so the difference is off by step^2 / 6 * 4 and by the loss's own error
    over the step."""
    torch, scores = ops
    r = np.random.default_rng(k)
    z = np.round(r.standard_normal((n, k)) * 64) / 64
    classes = r.integers(0, k, (n, 2)).astype(np.int32)
    gains = r.uniform(-0.5, 0.5, (n, 2)).astype(np.float32)
    lp = ref.feedback(z, classes, gains)['logs']
    old, reference = (lp - 0.1).astype(np.float32), (lp + 0.2).astype(np.float32)
    args = dict(old=old, reference=reference, kl=0.3, entropy=0.1, clip=(0.5, 0.5))
    want = ref.feedback(z, classes, gains, **args)
    dev = {name: _dev(torch, v) if isinstance(v, np.ndarray) else v for name, v in args.items()}
    call = lambda x, gives: scores.feedback(_tensor(torch, x, 'f32', layout), _dev(torch, classes), _dev(torch, gains), gives=gives, **dev)   # noqa: E731
    grad = call(z, 'gradient')[2].cpu().numpy()
    step = 2.0 ** -7
    for i in sorted({0, 1, k - 1, *map(int, classes[:, 0])})[:6]:
        up, down = z.copy(), z.copy()
        up[:, i] += step
        down[:, i] -= step
        slope = (call(up, 'loss')[0].double() - call(down, 'loss')[0].double()).cpu().numpy() / (2 * step)
        assert (np.abs(slope - grad[:, i]) <= 4 * step ** 2 / 6 + want['loss_off'].max() / step * 1.5 + want['g_off'][:, i]).all()


@pytest.mark.parametrize('layout,n,k', [('class', 7, 5), ('class', 7, 90), ('row', 7, 5), ('row', 7, 400), ('row', 7, 9001), ('any', 7, 50), ('class', 7, 2000)])
def test_feedback_of_unusual_numbers(ops, layout, n, k):
    """Masked classes drawn, rows of weight 0 or without a draw, ratios without bounds times nothing: no gradient, no loss."""
    torch, scores = ops
    r = np.random.default_rng(k)
    z = _make(r, n, k)
    z[0] = -np.inf
    z[1, 2] = -np.inf
    z[2] = np.nan            # of weight 0
    z[3, 1] = np.inf         # without a draw
    z[5] = float(np.finfo(np.float32).min)
    classes = np.array([[1, 2], [2, 2], [0, 1], [-1, k], [3, 3], [0, 4], [1, -5]], np.int32)
    gains = np.array([[1, 1], [1, -1], [1, 1], [1, 1], [0, 0], [1, 0.5], [2, 7]], np.float32)
    old = np.full((n, 2), -1.0, np.float32)
    old[4] = -1e30           # an infinite ratio, and no gain
    weights = np.array([1, 1, 0, 1, 1, 1, 1], np.float32)
    t = _tensor(torch, z, 'f32', layout)
    loss, logs, pairs = scores.feedback(t, _dev(torch, classes), _dev(torch, gains), old=_dev(torch, old), weights=_dev(torch, weights), clip=0.2, gives='pairs')
    loss, logs, pairs = (x.cpu().numpy() for x in (loss, logs, pairs))
    assert (loss[:5] == 0).all() and np.isfinite(loss).all()
    assert (logs[0] == -np.inf).all() and (logs[1] == -np.inf).all() and (logs[3] == -np.inf).all() and logs[6, 1] == -np.inf
    assert (pairs[:5, :, 0] == 0).all() and (pairs[:5, :, 1] == np.float32(1e-16)).all()
    rows = [4, 5, 6]
    want = ref.feedback(z[rows], classes[rows], gains[rows], old=old[rows], clip=(0.2, 0.2))
    _close(loss[rows], want['loss'], want['loss_off'], 'loss')
    _close(pairs[rows, :, 0], want['g'], want['g_off'], 'g')


# ------------------------------------------------------------------ norm
@pytest.mark.parametrize('layout', LAYOUTS)
@pytest.mark.parametrize('n,k', SIZES)
def test_norm_and_back(ops, n, k, layout):
    torch, scores = ops
    r = np.random.default_rng(n * 1000 + k + 7)
    for kind, weights, share in (('f32', True, 0.0), ('f32', False, 0.3), ('bf16', True, 0.2), ('f16', True, 0.0), ('bf16', False, 0.0)):
        z = _make(r, n, k) + 3
        z = _masked(r, z, share) if share else z
        t = _tensor(torch, z, kind, layout)
        gain = (1 + 0.3 * r.standard_normal(k)).astype(np.float32) if weights else None
        bias = r.standard_normal(k).astype(np.float32) if weights else None
        eps = 1e-5 if kind != 'f16' else 0.01
        want = ref.norm(_given(t), gain, bias, eps)
        before = t.clone()
        y, mean, rstd = scores.norm(t, _dev(torch, gain), _dev(torch, bias), eps=eps)
        assert torch.equal(t, before) and y.dtype == t.dtype and mean.dtype == rstd.dtype == torch.float32
        _close(mean.cpu().numpy(), want['mean'], want['mean_off'], (kind, 'mean'))
        _close(rstd.cpu().numpy(), want['rstd'], want['rstd_off'], (kind, 'rstd'))
        half = lambda v: HALF[kind] * np.abs(np.where(np.isfinite(v), v, 0)) * (1 + 2.0 ** -8) + TINY[kind] if kind != 'f32' else 0   # noqa: E731
        _close(_given(y), want['y'], want['y_off'] + half(want['y']), (kind, 'y'))
        # and back
        g = r.standard_normal((n, k))
        g[r.random((n, k)) < 0.01] = 30
        there = _given(t) != -np.inf
        g = np.where(there, g, np.nan)    # what stands beside a masked class is not looked at
        gt = _tensor(torch, g, kind, 'class' if layout == 'row+' else layout)
        back = ref.norm_backward(_given(gt), _given(t), mean.cpu().numpy(), rstd.cpu().numpy(), gain)
        out, to_gain, to_bias = scores.norm_backward(gt, t, mean, rstd, _dev(torch, gain))
        assert out.dtype == t.dtype and torch.equal(t, before)
        _close(_given(out), back['g'], back['g_off'] + half(back['g']), (kind, 'g'))
        _close(to_gain.cpu().numpy(), back['to_gain'], back['to_gain_off'], (kind, 'to_gain'))
        _close(to_bias.cpu().numpy(), back['to_bias'], back['to_bias_off'], (kind, 'to_bias'))
        only, a, b = scores.norm_backward(gt, t, mean, rstd, _dev(torch, gain), weights=False)
        assert a is None and b is None
        _close(_given(only), back['g'], back['g_off'] + half(back['g']), (kind, 'g alone'))
        again = scores.norm_backward(gt, t, mean, rstd, _dev(torch, gain))
        assert all(torch.equal(a, b) for a, b in zip((out, to_gain, to_bias), again))   # sums in one order
        # in place, and into another layout
        other = _tensor(torch, np.zeros((n, k)), kind, 'class+' if layout == 'row' else 'row+')
        assert scores.norm(t, _dev(torch, gain), _dev(torch, bias), eps=eps, out=other)[0] is other
        _close(_given(other), want['y'], want['y_off'] + half(want['y']), (kind, 'other'))
        scores.norm(t, _dev(torch, gain), _dev(torch, bias), eps=eps, out=t)
        assert torch.equal(t, y)


@pytest.mark.parametrize('layout', ['row', 'class'])
@pytest.mark.parametrize('n,k', [(5000, 9), (3001, 250), (700, 1000), (257, 5000)])
def test_norm_backward_of_many_rows(ops, n, k, layout):
    torch, scores = ops
    r = np.random.default_rng(k)
    for kind in ('f32', 'bf16'):
        t = _tensor(torch, _masked(r, _make(r, n, k)), kind, layout)
        gt = _tensor(torch, r.standard_normal((n, k)), kind, layout)
        gain = r.standard_normal(k).astype(np.float32)
        _, mean, rstd = scores.norm(t)
        back = ref.norm_backward(_given(gt), _given(t), mean.cpu().numpy(), rstd.cpu().numpy(), gain)
        out, to_gain, to_bias = scores.norm_backward(gt, t, mean, rstd, _dev(torch, gain))
        half = HALF[kind] * np.abs(back['g']) * (1 + 2.0 ** -8) if kind != 'f32' else 0
        _close(_given(out), back['g'], back['g_off'] + half, kind)
        _close(to_gain.cpu().numpy(), back['to_gain'], back['to_gain_off'], kind)
        _close(to_bias.cpu().numpy(), back['to_bias'], back['to_bias_off'], kind)


@pytest.mark.parametrize('layout', ['row', 'class', 'any'])
@pytest.mark.parametrize('n,k', [(6, 5), (6, 300), (4, 2500)])
def test_norm_backward_against_differences(ops, n, k, layout):
    """<g, norm(s + t v) - norm(s - t v)> / 2 t against <norm_backward(g), v>: with t = 2^-6 the difference is off by t^2 / 6 times the third
    derivative, below 6 |g|_1 max|v|^3 where rstd is below 1.5, and by the error of norm over t."""
    torch, scores = ops
    r = np.random.default_rng(k)
    z, g, v = r.standard_normal((n, k)), r.standard_normal((n, k)), r.uniform(-1, 1, (n, k))
    z, v = np.round(z * 256) / 256, np.round(v * 64) / 64
    gain = (1 + 0.2 * r.standard_normal(k)).astype(np.float32)
    t = 2.0 ** -6
    call = lambda x: scores.norm(_tensor(torch, x, 'f32', layout), _dev(torch, gain))   # noqa: E731
    _, mean, rstd = call(z)
    scale = float(rstd.max())
    out = scores.norm_backward(_tensor(torch, g, 'f32', layout), _tensor(torch, z, 'f32', layout), mean, rstd, _dev(torch, gain))[0]
    g32 = g.astype(np.float32).astype(np.float64)
    slope = (g32 * (call(z + t * v)[0].double() - call(z - t * v)[0].double()).cpu().numpy()).sum(1) / (2 * t)
    want = (out.double().cpu().numpy() * v).sum(1)
    ga = np.abs(g32 * gain)
    off = t ** 2 / 6 * 6 * scale ** 3 * np.sqrt((ga ** 2).sum(1) * k) + (np.abs(g32) * ref.norm(z, gain)['y_off']).sum(1) / t * 1.5 + 1e-4
    assert (np.abs(slope - want) <= off).all()


@pytest.mark.parametrize('layout,n,k', [('class', 6, 5), ('class', 6, 100), ('row', 6, 5), ('row', 6, 300), ('row', 6, 9001), ('any', 6, 50), ('class', 6, 2000)])
def test_norm_of_unusual_numbers(ops, layout, n, k):
    torch, scores = ops
    z = np.full((n, k), 2.5)               # no variance
    z[1] = -np.inf
    z[2, 1] = np.nan
    z[3, 0] = np.inf
    z[4] = -np.inf
    z[4, 3] = 1e6                          # one class
    z[5] = 1e4 + np.arange(k) % 2          # a mean far larger than the deviation
    t = _tensor(torch, z, 'f32', layout)
    y, mean, rstd = (x.cpu().numpy() for x in scores.norm(t))
    assert (y[0] == 0).all() and (y[1] == -np.inf).all() and mean[1] == 0 and rstd[1] == 0
    assert np.isnan(y[2]).all() and not np.isfinite(y[3]).any()
    assert y[4, 3] == 0 and (np.delete(y[4], 3) == -np.inf).all() and mean[4] == 1e6
    want = ref.norm(z[5:])
    _close(mean[5:], want['mean'], want['mean_off'], 'mean')
    _close(y[5:], want['y'], want['y_off'], 'y')
    # rows without a class, and with one, have no gradient
    g = torch.ones_like(t)
    out, to_gain, to_bias = scores.norm_backward(g, t, _dev(torch, mean), _dev(torch, rstd))
    out = out.cpu().numpy()
    assert (out[1] == 0).all() and (out[4] == 0).all() and np.isnan(out[2]).all()


def test_no_rows(ops):
    torch, scores = ops
    z = torch.empty(0, 9, device='cuda')
    assert scores.sample(z, torch.empty(0, device='cuda'))[0].shape == (0,)
    assert scores.norm(z)[0].shape == (0, 9)
    f = torch.empty(0, device='cuda')
    out, to_gain, to_bias = scores.norm_backward(z, z, f, f)
    assert out.shape == (0, 9) and not to_gain.any() and not to_bias.any()
    i = torch.empty(0, 2, dtype=torch.int32, device='cuda')
    loss, logs, pairs = scores.feedback(z, i, i.float(), gives='pairs')
    assert loss.shape == (0,) and logs.shape == (0, 2) and pairs.shape == (0, 9, 2)


def test_a_run_of_all(ops):
    """As they are used together: a teacher's rules, a row's draws, what they earn, the gradient through norm, a graph of it all replayed on
    new numbers."""
    torch, scores = ops
    n, k = 300, 90
    g = torch.Generator(device='cuda').manual_seed(1)
    raw = torch.randn(k, n, device='cuda', generator=g).t()
    u, prize = torch.rand(n, 4, device='cuda', generator=g), torch.randn(k, device='cuda', generator=g)
    gain, bias = torch.ones(k, device='cuda'), torch.zeros(k, device='cuda')

    def once():
        z, mean, rstd = scores.norm(raw, gain, bias)
        z2 = scores.adjust(z, bias=bias, presence=0.1)
        ids, logs, _ = scores.sample(z2, u, temperature=0.8)
        loss, now, grad = scores.feedback(z2, ids, prize[ids.long()], old=logs, temperature=0.8, clip=0.2, entropy=0.01)
        return ids, logs, now, loss, *scores.norm_backward(grad, raw, mean, rstd, gain)
    eager = [x.clone() for x in once()]
    assert torch.allclose(eager[1], eager[2], atol=1e-5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            beside = once()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, beside))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = once()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(eager, kept))
    raw.copy_(torch.randn(n, k, device='cuda', generator=g))
    u.copy_(torch.rand(n, 4, device='cuda', generator=g))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(once(), kept))
    assert not torch.equal(kept[0], eager[0])


@pytest.mark.parametrize('by', ['row', 'class'])
def test_offsets_beyond_31_bits(ops, by):
    """Lines 2^30 + 8 cells apart: the last one starts behind 2^32 bytes and 2^31 cells."""
    torch, scores = ops
    lines, cells, apart = 3, 40, (1 << 30) + 8
    base = torch.zeros(2 * apart + cells, dtype=torch.bfloat16, device='cuda')
    z = torch.as_strided(base, (lines, cells), (apart, 1))
    r = np.random.default_rng(1)
    z.copy_(torch.from_numpy(_make(r, lines, cells)))
    z = z if by == 'row' else z.t()
    small = z.contiguous() if by == 'row' else z.t().contiguous().t()
    n = z.size(0)
    u, ids = torch.rand(n, device='cuda'), torch.randint(0, 3, (n,), device='cuda', dtype=torch.int32)
    for a, b in zip(scores.sample(z, u, top_p=0.9), scores.sample(small, u, top_p=0.9)):
        assert torch.equal(a, b)
    for a, b in zip(scores.feedback(z, ids, u), scores.feedback(small, ids, u)):
        assert torch.equal(a, b)
    out = torch.as_strided(torch.zeros_like(base), z.shape, z.stride())
    y, mean, rstd = scores.norm(z, out=out)
    want = scores.norm(small)
    assert torch.equal(y, want[0]) and torch.equal(mean, want[1])
    for a, b in zip(scores.norm_backward(out, z, mean, rstd), scores.norm_backward(want[0], small, mean, rstd)):
        assert torch.equal(a, b)


def test_refusals(ops):
    torch, scores = ops
    z = torch.zeros(4, 9, device='cuda')
    u, i = torch.rand(4, device='cuda'), torch.zeros(4, dtype=torch.int32, device='cuda')
    f = torch.zeros(4, device='cuda')
    for call in (lambda: scores.sample(z, u.half()), lambda: scores.sample(z, u[:3]), lambda: scores.sample(z, torch.rand(4, 129, device='cuda')),
                 lambda: scores.sample(z, torch.rand(4, 0, device='cuda')), lambda: scores.sample(z, torch.rand(4, 2, device='cuda')[:, 0]), lambda: scores.sample(z, u.cpu()),
                 lambda: scores.sample(z, 0.5), lambda: scores.sample(z, u, top_k=u), lambda: scores.sample(z, u, top_k=2.5), lambda: scores.sample(z, u, temperature=i),
                 lambda: scores.sample(z, u, top_p=f[:2]), lambda: scores.sample(z.cpu(), u), lambda: scores.sample(z.double(), u), lambda: scores.sample(z[0], u),
                 lambda: scores.feedback(z, i.long(), f), lambda: scores.feedback(z, i, f.double()), lambda: scores.feedback(z, i, f[:2]), lambda: scores.feedback(z, i, f, kl=0.1),
                 lambda: scores.feedback(z, i, f, gives='all'), lambda: scores.feedback(z, i, f, old=f[None]), lambda: scores.feedback(z, i, f, weights=f[:1]),
                 lambda: scores.norm(z, gain=f), lambda: scores.norm(z, out=z.half()), lambda: scores.norm(z, out=z.clone().requires_grad_()),
                 lambda: scores.norm_backward(z.half(), z, f, f), lambda: scores.norm_backward(z, z, f[:1], f), lambda: scores.norm_backward(z, z, f, f, gain=f)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: scores.sample(z, u, temperature=-1.0), lambda: scores.sample(z, u, temperature=float('nan')), lambda: scores.sample(z, u, top_p=1.5),
                 lambda: scores.sample(z, u, min_p=-0.1), lambda: scores.sample(z, u, top_k=-1), lambda: scores.feedback(z, i, f, temperature=0.0),
                 lambda: scores.feedback(z, i, f, clip=-0.1), lambda: scores.feedback(z, i, f, clip=(1.5, 0.2)), lambda: scores.feedback(z, i, f, entropy=-1.0),
                 lambda: scores.norm(z, eps=0.0), lambda: scores.norm(z, eps=float('nan'))):
        with pytest.raises(RuntimeError):
            call()
    torch.cuda.synchronize()
