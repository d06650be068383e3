"""Drawing classes and learning from draws where rows, limits and arguments are at their edges; definitions and bounds are those of
tests/draws_ref.py."""
import numpy as np
import pytest

import draws_ref as ref
from scores_ref import HALF, TINY
from test_gpu_draws import _check_feedback, _check_sample, _dev, _draws, _masked
from test_gpu_scores import _close, _given, _make, _tensor, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def _half(kind, v):
    return HALF[kind] * np.abs(np.where(np.isfinite(v), v, 0)) * (1 + 2.0 ** -8) + TINY[kind] if kind != 'f32' else 0


def _check_norm(ops, t, gt, kind, gain, bias, what):
    torch, scores = ops
    want = ref.norm(_given(t), gain, bias)
    y, mean, rstd = scores.norm(t, _dev(torch, gain), _dev(torch, bias))
    _close(mean.cpu().numpy(), want['mean'], want['mean_off'], what + ('mean',))
    _close(rstd.cpu().numpy(), want['rstd'], want['rstd_off'], what + ('rstd',))
    _close(_given(y), want['y'], want['y_off'] + _half(kind, want['y']), what + ('y',))
    back = ref.norm_backward(_given(gt), _given(t), mean.cpu().numpy(), rstd.cpu().numpy(), gain)
    for weights in (True, False):
        out, to_gain, to_bias = scores.norm_backward(gt, t, mean, rstd, _dev(torch, gain), weights=weights)
        _close(_given(out), back['g'], back['g_off'] + _half(kind, back['g']), what + ('g', weights))
        if weights:
            _close(to_gain.cpu().numpy(), back['to_gain'], back['to_gain_off'], what + ('to_gain',))
            _close(to_bias.cpu().numpy(), back['to_bias'], back['to_bias_off'], what + ('to_bias',))


# lengths around what the kernels' registers hold, rows that begin on 16 bytes and rows that do not
@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('n,k', [(3, 512), (40, 513), (3, 1024), (3, 2048), (2, 2049), (3, 8192), (2, 8200), (2, 16384), (1, 16385), (1, 32768), (1, 65536), (1, 65537), (1, 131072),
                                 (1, 131073)])
def test_lengths_where_kernels_change(ops, n, k, kind):
    torch, _ = ops
    r = np.random.default_rng(k + n)
    for layout in ('row', 'row+') if k > 1024 else ('row', 'class', 'row+'):
        z = _masked(r, _make(r, n, k), 0.05)
        t = _tensor(torch, z, kind, layout)
        for limits in ({}, dict(top_k=40, top_p=0.9), dict(top_p=0.97, temperature=1.4)):
            _check_sample(ops, t, r.random((n, 3)), limits, (kind, layout))
        classes, gains, old, reference = _draws(r, _given(t), 3, 1.3, (0.2, 0.2))
        _check_feedback(ops, t, kind, classes, gains, (kind, layout), old=old, reference=reference, temperature=1.3, clip=(0.2, 0.2), kl=0.1, entropy=0.05)
        gt = _tensor(torch, r.standard_normal((n, k)), kind, layout)
        gain, bias = (1 + 0.2 * r.standard_normal(k)).astype(np.float32), r.standard_normal(k).astype(np.float32)
        _check_norm(ops, t, gt, kind, gain, bias, (kind, layout))


@pytest.mark.parametrize('kind', ['f32', 'f16'])
@pytest.mark.parametrize('n,k,shift', [(1300, 1100, 0), (1300, 2048, 0), (700, 5000, 0), (400, 2003, 1), (310, 9000, 3)])
def test_many_long_rows(ops, n, k, shift, kind):
    """More rows than the GPU works on at once, several at a time; some of them with masked classes, and not all from a 16-byte boundary on."""
    torch, _ = ops
    r = np.random.default_rng(k)
    z = _make(r, n, k + 8)
    z[5::7] = np.where(r.random((z[5::7].shape)) < 0.3, -np.inf, z[5::7])
    z[n // 3] = -np.inf
    t = _tensor(torch, z, kind, 'row')[:, shift:shift + k]
    gt = _tensor(torch, r.standard_normal((n, k + 24)), kind, 'row')[:, 2 * shift + 1 if shift else 0:][:, :k]
    gain, bias = (1 + 0.2 * r.standard_normal(k)).astype(np.float32), r.standard_normal(k).astype(np.float32)
    _check_norm(ops, t, gt, kind, gain, bias, (kind, n, k))
    u = r.random(n)
    _check_sample(ops, t, u, dict(top_k=20, min_p=0.01), (kind, n, k))
    classes, gains, old, _ = _draws(r, _given(t), 1, 1.0, None)
    _check_feedback(ops, t, kind, classes, gains, (kind, n, k), old=old, entropy=0.01)


@pytest.mark.parametrize('ties', [False, True])
@pytest.mark.parametrize('layout,n,k', [('class', 40, 300), ('class', 35, 900), ('row', 1100, 700), ('row', 5, 3000), ('row', 3, 30001), ('row+', 2, 70000), ('class', 6, 1500)])
def test_limits_that_leave_many(ops, layout, n, k, ties):
    """More scores than a list has room for are left, or reach the border, or equal it."""
    torch, _ = ops
    r = np.random.default_rng(k)
    z = r.standard_normal((n, k))
    z = np.round(z * 4) / 4 if ties else z
    z[0] = 0.25                                     # all equal
    z[1] = np.where(np.arange(k) % 3, 1.0, 2.0)     # two values
    t = _tensor(torch, z, 'f32', layout)
    for limits in (dict(top_k=k // 2), dict(top_k=k - 1, temperature=3.0), dict(top_p=0.5), dict(top_p=0.999), dict(top_p=0.0), dict(min_p=0.001), dict(min_p=1.0),
                   dict(min_p=0.01, top_p=0.9), dict(top_k=k // 3, top_p=0.7, min_p=0.05), dict(top_k=1), dict(top_k=1100, top_p=0.95), dict(top_p=0.9, temperature=1e30)):
        _check_sample(ops, t, r.random((n, 2)), limits, (layout, ties, str(limits)))


def test_limits_per_row_that_differ(ops):
    """Rows without limits beside rows with a few classes left and rows with nearly all, in one tile and in one launch."""
    torch, _ = ops
    for layout, n, k in (('class', 200, 250), ('row', 1200, 250), ('row', 60, 20000), ('class', 130, 20)):
        r = np.random.default_rng(n)
        t = _tensor(torch, _make(r, n, k), 'bf16', layout)
        limits = dict(temperature=r.choice([0.0, 0.6, 1.0, 5.0], n).astype(np.float32), top_k=r.choice([0, 0, 1, 30, k - 1, k, 3 * k], n).astype(np.int32),
                      top_p=r.choice([1.0, 0.9999, 0.9, 0.3], n).astype(np.float32), min_p=r.choice([0.0, 0.0, 1e-4, 0.2], n).astype(np.float32))
        _check_sample(ops, t, r.random((n, 17)), limits, (layout, n, k))
        for name in limits:   # one of them, the others as numbers
            _check_sample(ops, t, r.random(n), {name: limits[name]}, (layout, n, k, name))


@pytest.mark.parametrize('layout', ['row', 'row+', 'class', 'any'])
def test_as_many_classes_as_there_may_be(ops, layout):
    """2^20 classes, the last ones among the likeliest and the drawn ones."""
    torch, _ = ops
    n, k = 2, 1 << 20
    r = np.random.default_rng(5)
    z = r.standard_normal((n, k))
    z[:, k - 1] = 9.0
    z[1, k - 2] = 9.0
    z[0, :3] = [8.0, -np.inf, 7.5]
    t = _tensor(torch, z, 'f32', layout)
    u = np.array([[0.0, 0.5, 1 - 2.0 ** -30], [0.1, 0.7, 0.999999]])
    for limits in ({}, dict(top_k=3), dict(top_p=0.2), dict(min_p=0.5, top_p=0.9)):
        _check_sample(ops, t, u, limits, (layout, str(limits)))
    classes = np.array([[k - 1, 1], [k - 2, 4]], np.int32)
    _check_feedback(ops, t, 'f32', classes, np.ones((2, 2), np.float32), (layout,), entropy=0.1)
    _check_norm(ops, t, _tensor(torch, r.standard_normal((n, k)), 'f32', layout), 'f32', r.standard_normal(k).astype(np.float32), None, (layout,))


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('k', [6, 45, 250, 1000])
def test_a_slice_of_one_row_is_that_row(ops, kind, k):
    """One row taken out of a matrix by class, as a view and as a copy of its own, gets the bits that it has among the others."""
    torch, scores = ops
    r = np.random.default_rng(k)
    z = _tensor(torch, _make(r, 70, k), kind, 'class+')
    g = _tensor(torch, r.standard_normal((70, k)), kind, 'class')
    c, a = _dev(torch, r.integers(0, k, (70, 3)).astype(np.int32)), torch.randn(70, 3, device='cuda')
    u, gain = torch.rand(70, 3, device='cuda'), torch.rand(k, device='cuda')
    drawn, loss, normed = scores.sample(z, u, top_p=0.9), scores.feedback(z, c, a, entropy=0.1, gives='pairs'), scores.norm(z, gain)
    back = scores.norm_backward(g, z, normed[1], normed[2], gain, weights=False)[0]
    for n in (0, 31, 32, 69):
        one = slice(n, n + 1)
        for part in (z[one], z[one].t().contiguous().t()):
            assert torch.equal(scores.sample(part, u[one], top_p=0.9)[0], drawn[0][one])
            assert all(torch.equal(x, y[one]) for x, y in zip(scores.feedback(part, c[one], a[one], entropy=0.1, gives='pairs'), loss))
            assert all(torch.equal(x, y[one]) for x, y in zip(scores.norm(part, gain), normed))
            got = scores.norm_backward(g[one], part, normed[1][one].contiguous(), normed[2][one].contiguous(), gain, weights=False)[0]
            assert torch.equal(got, back[one])


def test_results_beside_what_is_read(ops):
    torch, scores = ops
    z = torch.randn(6, 40, device='cuda')
    for gain in (z[0], z[5]):
        with pytest.raises(RuntimeError, match='share memory'):
            scores.norm(z, gain, out=z)
    with pytest.raises(RuntimeError, match='share memory'):
        scores.norm(z[:, :39], out=z[:, 1:])
    rec = torch.randn(6, 100, device='cuda')   # records of scores, a gain and room
    want = scores.norm(rec[:, :40].clone(), rec[2, 40:80].clone())[0]
    scores.norm(rec[:, :40], rec[2, 40:80], out=rec[:, :40])
    assert torch.equal(rec[:, :40], want)


def test_autograd(ops):
    """The operators are not recorded: results require no gradient, their gradients are what backward() takes, and a tensor that a
    recorded operation keeps is known to have changed."""
    torch, scores = ops
    w = torch.randn(30, 30, device='cuda', requires_grad=True)
    s = torch.randn(4, 30, device='cuda') @ w
    y, mean, rstd = scores.norm(s)
    ids, logs, every = scores.sample(y, torch.rand(4, 2, device='cuda'))
    loss, now, grad = scores.feedback(y, ids, torch.ones(4, 2, device='cuda'), old=logs)
    assert not any(x.requires_grad for x in (y, mean, rstd, logs, every, loss, now, grad))
    s.backward(scores.norm_backward(grad, s, mean, rstd, weights=False)[0])
    assert bool((w.grad.abs() > 0).any())
    x = torch.randn(4, 30, device='cuda', requires_grad=True)
    y = x.exp()
    with pytest.raises(ValueError, match='autograd'):
        scores.norm(y, out=y)
    scores.norm(y.detach(), out=y.detach())
    with pytest.raises(RuntimeError, match='modified'):
        y.sum().backward()


def test_two_graphs_in_turn(ops):
    """Captured one after the other, replayed in turn and on two streams at once: each has memory of its own."""
    torch, scores = ops
    z, g = torch.randn(2000, 3000 // 2, device='cuda'), torch.randn(2000, 3000 // 2, device='cuda')
    gain = torch.rand(1500, device='cuda')
    _, mean, rstd = scores.norm(z)
    graphs, kept = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept.append(scores.norm_backward(g * (i + 1), z, mean, rstd, gain))
        graphs.append(graph)
    want = [scores.norm_backward(g * (i + 1), z, mean, rstd, gain) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for turn in range(3):
        for i in (0, 1) if turn % 2 else (1, 0):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    for a, b in zip(kept, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
