"""The operators on scores where rows, lists and arguments are at their edges; definitions and bounds are those of tests/scores_ref.py."""
import numpy as np
import pytest

import scores_ref as ref
from test_gpu_scores import _close, _given, _make, _teacher, _tensor, ops  # noqa: F401

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


LAYOUTS = [('class', 12, 6), ('class', 12, 90), ('row', 12, 6), ('row', 12, 400), ('row', 12, 9001), ('any', 12, 50), ('class', 12, 2000), ('any', 3, 20000)]


@pytest.mark.parametrize('layout,n,k', LAYOUTS)
def test_terms_that_weigh_nothing(ops, layout, n, k):
    """A distance that is infinite counts for nothing where alpha is 0, and neither does a whole row of weight 0: the loss is that of the
    labels, or 0.  Gradients and pairs likewise."""
    torch, scores = ops
    r = np.random.default_rng(n + k)
    z = _make(r, n, k)
    ids, logits, lse = _teacher(r, z, 4, 1.0)
    ids[:, 3] = (ids[:, 2] + 1) % k   # (a class may stand there twice)
    labels = ids[:, 1].copy()
    for i in range(0, n, 3):
        z[i, ids[i, 0]] = -np.inf                                                 # a listed class is masked
    for i in range(1, n, 3):
        z[i] = np.where(np.isin(np.arange(k), ids[i]), z[i], -np.inf)             # ... or all that are not listed
    z[n - 1] = -np.inf                                                            # ... or all
    t = _tensor(torch, z, 'f32', layout)
    dev = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()   # noqa: E731
    weights = r.random(n).astype(np.float32) + 0.5
    weights[::2] = 0
    weights[n - 1] = 0
    for T in (1.0, 1.7):
        for use_lse in (True, False):
            L = lse if use_lse else None
            # alpha = 0 (the row without any score has no finite label term either: left to its weight)
            want = ref.distill(_given(t), np.full_like(ids, -1), logits, L, labels, None, T, 0.0)
            for gives in ('loss', 'gradient', 'pairs'):
                loss, g = scores.distill(t, dev(ids), dev(logits), lse=dev(L), labels=dev(labels), temperature=T, alpha=0.0, gives=gives)
                _close(loss.cpu().numpy(), want['loss'], want['loss_off'], (T, use_lse, gives))
            assert np.isfinite(want['loss'][:n - 1]).all() and np.isinf(want['loss'][n - 1])
            _close(g[..., 0].cpu().numpy(), want['g'], want['g_off'], (T, use_lse))
            # weights of 0
            one = ref.distill(_given(t), ids, logits, L, labels, None, T, 0.6)
            want = ref.distill(_given(t), ids, logits, L, labels, weights, T, 0.6)
            assert np.isinf(one['loss'][weights == 0]).any()
            for gives in ('loss', 'gradient', 'pairs'):
                loss, g = scores.distill(t, dev(ids), dev(logits), lse=dev(L), labels=dev(labels), weights=dev(weights), temperature=T, alpha=0.6, gives=gives)
                _close(loss.cpu().numpy(), np.where(weights == 0, 0.0, want['loss']), np.where(weights == 0, 0.0, want['loss_off']), (T, use_lse, gives))
            _close(g[..., 0].cpu().numpy(), want['g'], want['g_off'], (T, use_lse))
            assert bool((g[..., 0][dev(weights == 0)] == 0).all())


def test_a_set_of_no_masks_is_refused(ops):
    torch, scores = ops
    z = torch.randn(4, 70, device='cuda')
    none = torch.zeros(0, 3, dtype=torch.int32, device='cuda')
    row = torch.zeros(4, dtype=torch.int32, device='cuda')
    for bad in (dict(allowed=none), dict(allowed=none, allowed_row=row), dict(allowed=torch.zeros(3, 3, dtype=torch.int32, device='cuda'))):
        with pytest.raises(ValueError, match='allowed'):
            scores.adjust(z, **bad)
    assert scores.adjust(z[:0], allowed=none).shape == (0, 70) and scores.adjust(z[:0], allowed=none, allowed_row=row[:0]).shape == (0, 70)
    assert bool((scores.adjust(z, allowed=torch.zeros(1, 3, dtype=torch.int32, device='cuda'), allowed_row=row) == -float('inf')).all())


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('k', [6, 45, 250, 1000, 1024])
def test_a_slice_of_one_row_is_that_row(ops, kind, k):
    """One row taken out of a matrix by class, as a view and as a copy of its own, gets the bits that it has among the others."""
    torch, scores = ops
    r = np.random.default_rng(k)
    z = _tensor(torch, _make(r, 70, k), kind, 'class+')
    v, i, lse = scores.top(_tensor(torch, _make(r, 70, k), 'f32', 'row'), min(k, 9), temperature=1.5)
    y = torch.from_numpy(r.integers(-1, k, 70).astype(np.int32)).cuda()
    bias, given = torch.randn(k, device='cuda'), torch.arange(71, device='cuda')
    top, adjusted = scores.top(z, 5, temperature=1.5), scores.adjust(z, bias=bias, history=(given, y), presence=0.3, repetition=1.2)
    for gives in ('loss', 'gradient', 'pairs'):
        par = dict(temperature=1.5, alpha=0.6, gives=gives)
        whole = scores.distill(z, i, v, lse=lse, labels=y, **par)
        for n in (0, 31, 32, 69):
            one = slice(n, n + 1)
            for part in (z[one], z[one].t().contiguous().t()):
                got = scores.distill(part, i[one], v[one], lse=lse[one], labels=y[one], **par)
                assert torch.equal(got[0], whole[0][one]) and (gives == 'loss' or torch.equal(got[1], whole[1][one])), (gives, n, part.stride())
                assert all(torch.equal(a, b[one]) for a, b in zip(scores.top(part, 5, temperature=1.5), top))
                got = scores.adjust(part, bias=bias, history=(given[:2], y[one]), presence=0.3, repetition=1.2)
                assert torch.equal(got, adjusted[one])


def test_results_beside_what_is_read(ops):
    """In place with a row of the scores as the bias is refused; what lies in the gaps of a matrix, or shares its lines, is not."""
    torch, scores = ops
    z = torch.randn(6, 40, device='cuda')
    before = z.clone()
    for bias in (z[0], z[5]):
        with pytest.raises(RuntimeError, match='share memory'):
            scores.adjust(z, out=z, bias=bias)
    with pytest.raises(RuntimeError, match='share memory'):
        scores.adjust(z, out=z, history=(torch.arange(7, device='cuda'), z[2, :6].view(torch.int32)))
    assert torch.equal(z, before)
    assert torch.equal(scores.adjust(z, bias=z[3]), z + z[3])
    # records of scores, a bias and room, one behind the other
    rec = torch.randn(6, 100, device='cuda')
    want = rec[:, :40] + rec[2, 40:80]
    scores.adjust(rec[:, :40], out=rec[:, :40], bias=rec[2, 40:80])
    assert torch.equal(rec[:, :40], want)
    by_class = torch.randn(40, 100, device='cuda')
    part, bias = by_class[:, :30].t(), by_class[7, 40:80]
    want = part + bias
    assert torch.equal(scores.adjust(part, out=part, bias=bias), want)
    column = rec[:, 41:42]
    want = column + rec[1, 50:51]
    assert torch.equal(scores.adjust(column, out=column, bias=rec[1, 50:51]), want)
    one = by_class[:, 3:4].t()
    want = one + bias
    assert torch.equal(scores.adjust(one, out=one, bias=bias), want)
    with pytest.raises(RuntimeError, match='share memory'):
        scores.adjust(part, out=part, bias=by_class[7, 20:60])


def test_results_in_place_and_autograd(ops):
    """The operators are not recorded by autograd: a tensor that a recorded operation keeps for its backward pass is known to have
    changed, and one that takes part itself is refused as a place for results."""
    torch, scores = ops
    x = torch.randn(4, 30, device='cuda', requires_grad=True)
    bias = torch.ones(30, device='cuda')
    y = x.exp()               # (the backward pass reads y)
    for out in (x, y):
        with pytest.raises(ValueError, match='autograd'):
            scores.adjust(out, out=out, bias=bias)
    y.sum().backward()
    y = x.exp()
    scores.adjust(y.detach(), out=y.detach(), bias=bias)
    with pytest.raises(RuntimeError, match='modified'):
        y.sum().backward()
    with torch.no_grad():
        want = x + 1
        scores.adjust(x, out=x, bias=bias)
        assert torch.equal(x, want) and x.requires_grad
    with torch.inference_mode():
        z = torch.randn(4, 30, device='cuda')
        want = z + 1
        assert torch.equal(scores.adjust(z, out=z, bias=bias), want)
    # results require no gradient, whatever the scores do; distill's gradient is what backward() takes
    w = torch.randn(30, 30, device='cuda', requires_grad=True)
    student = torch.randn(4, 30, device='cuda') @ w
    v, i, lse = scores.top(student, 3)
    assert not v.requires_grad and not lse.requires_grad and not scores.adjust(student, bias=bias).requires_grad
    loss, grad = scores.distill(student, i, v + 1, temperature=2.0)
    assert not loss.requires_grad
    student.backward(grad)
    assert w.grad is not None and bool(w.grad.abs().sum() > 0)


@pytest.mark.parametrize('layout', ['row', 'row+', 'class', 'any'])
def test_as_many_classes_as_there_may_be(ops, layout):
    """2^20 classes, the last ones among the chosen, listed, masked and given ones."""
    torch, scores = ops
    n, k = 2, 1 << 20
    r = np.random.default_rng(5)
    z = r.standard_normal((n, k))
    z[:, k - 1] = 9.0
    z[1, k - 2] = 9.0
    z[0, :3] = [8.0, -np.inf, 7.5]
    t = _tensor(torch, z, 'f32', layout)
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()   # noqa: E731
    values, ids, lse, off = ref.top(_given(t), 4, 1.5)
    got = scores.top(t, 4, temperature=1.5)
    assert np.array_equal(got[1].cpu().numpy(), ids) and np.array_equal(got[0].cpu().numpy(), values)
    _close(got[2].cpu().numpy(), lse, off, 'lse')
    past = (np.array([0, 2, 3]), np.array([k - 1, k - 1, 0], np.int32))
    bias, allowed = r.standard_normal(k).astype(np.float32), np.ones((1, k), bool)
    allowed[0, [5, k - 2]] = False
    want, off = ref.adjust(_given(t), bias, allowed, np.zeros(n, np.int32), past, repetition=1.5, frequency=0.25, presence=0.5)
    got = scores.adjust(t, bias=dev(bias), allowed=dev(np.packbits(allowed, axis=1, bitorder='little').view(np.int32)),
                        allowed_row=dev(np.zeros(n, np.int32)), history=(dev(past[0]), dev(past[1])), repetition=1.5, frequency=0.25, presence=0.5)
    _close(_given(got), want, off + ref.U * np.abs(np.where(np.isfinite(want), want, 0)), 'adjust')
    ids = np.array([[k - 1, 0, 77], [k - 2, k - 1, 3]], np.int32)
    logits = r.standard_normal((n, 3)).astype(np.float32) + 8
    lse = np.array([9.5, 10.0], np.float32)
    y = np.array([k - 1, 4], np.int32)
    want = ref.distill(_given(t), ids, logits, lse, y, None, 1.5, 0.6)
    loss, pairs = scores.distill(t, dev(ids), dev(logits), lse=dev(lse), labels=dev(y), temperature=1.5, alpha=0.6, gives='pairs')
    _close(loss.cpu().numpy(), want['loss'], want['loss_off'], 'loss')
    _close(pairs[..., 0].cpu().numpy(), want['g'], want['g_off'], 'g')
    _close(pairs[..., 1].cpu().numpy(), want['h'], want['h_off'], 'h')
    loss, grad = scores.distill(t, dev(ids), dev(logits), lse=dev(lse), labels=dev(y), temperature=1.5, alpha=0.6)
    _close(_given(grad), want['g'], want['g_off'], 'gradient')


@pytest.mark.parametrize('layout,n,k', [('class', 12, 20), ('class', 12, 90), ('class', 12, 1000), ('row', 12, 400), ('row', 12, 9001), ('any', 12, 50), ('class', 12, 2000), ('any', 3, 20000)])
def test_masses_that_no_float_holds_are_none(ops, layout, n, k):
    """A class to which the teacher gives e^-200 of its mass (a float holds e^-103) counts as if it had none, also where the student masks
    it: the distance stays finite, however the scores are laid out."""
    torch, scores = ops
    r = np.random.default_rng(k)
    z = _make(r, n, k)
    ids, logits, lse = _teacher(r, z, 5, 1.0)
    logits[:, 4] = logits[:, 0] - 200
    z[np.arange(n), ids[:, 4]] = -np.inf
    t = _tensor(torch, z, 'f32', layout)
    without = ids.copy()
    without[:, 4] = -1
    dev = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()   # noqa: E731
    for L in (lse, None):
        want = ref.distill(_given(t), without, logits, L, None, None, 1.0, 1.0)
        loss, _ = scores.distill(t, dev(ids), dev(logits), lse=dev(L), gives='loss')
        assert np.isfinite(want['loss']).all()
        _close(loss.cpu().numpy(), want['loss'], want['loss_off'], L is None)
