"""The operators on scores (thundergbm_b200/scores.py, tgbm_scores_*) against their definitions in 64 bits: layouts, types, sizes where
kernels change over, masks that leave nothing, ties, infinities, lists with gaps and repeats; bounds are those of tests/scores_ref.py,
which count the roundings."""
import numpy as np
import pytest

import scores_ref as ref

pytestmark = pytest.mark.gpu
TYPES = ['f32', 'f16', 'bf16']


@pytest.fixture(scope='module')
def ops(gpu):
    import torch
    from thundergbm_b200 import scores
    return torch, scores


def _type(torch, kind):
    return {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}[kind]


def _tensor(torch, z, kind, layout):
    """z (rows x classes, NumPy) on the GPU in a layout: 'row', 'class', each with room behind ('+'), 'any': no stride of 1."""
    t = torch.from_numpy(np.ascontiguousarray(z)).to(_type(torch, kind))
    n, k = t.shape
    if layout.startswith('row'):
        pad = 3 if layout.endswith('+') else 0
        s = torch.full((n, k + pad), 7.0, dtype=t.dtype, device='cuda')[:, :k]
    elif layout.startswith('class'):
        pad = 5 if layout.endswith('+') else 0
        s = torch.full((k, n + pad), 7.0, dtype=t.dtype, device='cuda')[:, :n].t()
    else:
        s = torch.full((n, k, 2), 7.0, dtype=t.dtype, device='cuda')[:, :, 0]
    s.copy_(t)
    return s


def _given(t):
    return t.float().cpu().numpy()   # what the kernel reads: after the rounding to its type


def _make(r, n, k, ties=False):
    z = r.standard_normal((n, k)) * 2 + 8 * (r.random((n, k)) < 5 / k)
    return np.round(z * 2) / 2 if ties else z


def _close(got, want, off, what):
    got, want = np.asarray(got, np.float64), np.asarray(want)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True), what
    assert np.isfinite(got[fine]).all(), what
    far = np.abs(got[fine] - want[fine]) - np.broadcast_to(off, want.shape)[fine]
    assert far.size == 0 or far.max() <= 0, (what, far.max(), np.argwhere(fine)[np.argmax(far)])


# sizes: one row, rows and classes around a warp, a tile, several tiles; more classes than a block holds at once
SIZES = [(1, 1), (1, 7), (5, 1), (33, 2), (70, 3), (257, 7), (31, 31), (100, 32), (65, 33), (40, 100), (33, 250), (7, 257), (3, 1000), (2, 1025),
         (5, 4097), (2, 8193), (1, 20011), (3, 70001)]


def _history(r, n, k, most):
    lengths = r.integers(0, most + 1, n)
    lengths[:: 3] = 0
    ptr = np.concatenate([[0], lengths.cumsum()]).astype(np.int64)
    ids = (k * r.random(ptr[-1]) ** 2).astype(np.int32)
    ids[r.random(ids.size) < 0.1] = -1
    ids[r.random(ids.size) < 0.05] = k + 3
    return ptr, ids


def _bits(allowed):
    m, k = allowed.shape
    padded = np.ones((m, (k + 31) // 32 * 32), bool)
    padded[:, :k] = allowed
    return np.packbits(padded, axis=1, bitorder='little').view(np.int32)


@pytest.mark.parametrize('layout', ['row', 'class', 'row+', 'class+', 'any'])
@pytest.mark.parametrize('n,k', SIZES)
def test_adjust(ops, n, k, layout):
    torch, scores = ops
    r = np.random.default_rng(n * 1000 + k)
    for kind, masks, with_bias, most in (('f32', 'own', True, 40), ('bf16', 'shared', False, 300), ('f16', 'none', True, 5), ('f32', 'shared', True, 0)):
        z = _tensor(torch, _make(r, n, k), kind, layout)
        allowed = None if masks == 'none' else r.random((n if masks == 'own' else 3, k)) < 0.6
        row = r.integers(-1, 4, n).astype(np.int32) if masks == 'shared' else None   # (3: no such mask)
        bias = r.standard_normal(k).astype(np.float32) if with_bias else None
        history = _history(r, n, k, most) if most else None
        par = dict(repetition=1.3, frequency=0.11, presence=0.7)
        dev = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()   # noqa: E731
        want, off = ref.adjust(_given(z), bias, allowed, row, history, **par)
        before = z.clone()
        got = scores.adjust(z, bias=dev(bias), allowed=None if allowed is None else dev(_bits(allowed)), allowed_row=dev(row),
                            history=None if history is None else tuple(map(dev, history)), **par)
        assert got.dtype == z.dtype and got.shape == z.shape and torch.equal(z, before)
        off = off + ref.HALF[kind] * np.abs(np.where(np.isfinite(want), want, 0)) * (1 + 2.0 ** -8) + ref.TINY[kind]
        _close(_given(got), want, off, (kind, masks))
        # in place, and into a buffer of another layout
        other = _tensor(torch, np.zeros((n, k)), kind, 'class+' if layout == 'row' else 'row+')
        scores.adjust(z, out=other, bias=dev(bias), allowed=None if allowed is None else dev(_bits(allowed)), allowed_row=dev(row),
                      history=None if history is None else tuple(map(dev, history)), **par)
        assert torch.equal(other, got)
        scores.adjust(z, out=z, bias=dev(bias), allowed=None if allowed is None else dev(_bits(allowed)), allowed_row=dev(row),
                      history=None if history is None else tuple(map(dev, history)), **par)
        assert torch.equal(z, got)


@pytest.mark.parametrize('layout', ['row', 'class', 'row+', 'class+', 'any'])
@pytest.mark.parametrize('n,k', SIZES)
def test_top(ops, n, k, layout):
    torch, scores = ops
    r = np.random.default_rng(n * 1000 + k + 1)
    for kind, m, temperature, ties in (('f32', 1, 1.0, False), ('f32', 5, 0.5, True), ('bf16', 20, 2.0, False), ('f16', 64, 1.0, True), ('f32', 128, 1.7, False)):
        z = _make(r, n, k, ties)
        z[r.random((n, k)) < 0.1] = -np.inf
        z[0, : k // 2] = -np.inf
        z[n // 2] = -np.inf if n > 1 else z[n // 2]
        z[-1] = 1.5 if n > 2 else z[-1]        # all equal
        t = _tensor(torch, z, kind, layout)
        got = scores.top(t, m, temperature=temperature)
        values, ids, lse, off = ref.top(_given(t), m, temperature)
        assert got[0].dtype == got[2].dtype == torch.float32 and got[1].dtype == torch.int32
        assert np.array_equal(got[1].cpu().numpy(), ids), (kind, m)
        assert np.array_equal(got[0].cpu().numpy(), values), (kind, m)
        _close(got[2].cpu().numpy(), lse, off, (kind, m))


@pytest.mark.parametrize('order', ['up', 'down', 'comb', 'block'])
@pytest.mark.parametrize('layout,n,k', [('row', 3, 50021), ('row', 200, 1000), ('class', 70, 300), ('row', 9, 5000)])
def test_top_of_ordered_rows(ops, order, layout, n, k):
    """Rows whose largest scores all fall to the same thread, warp or tile."""
    torch, scores = ops
    z = np.tile(np.arange(k, dtype=np.float64) / 64, (n, 1))
    if order == 'down':
        z = z[:, ::-1].copy()
    elif order == 'comb':     # every 256th (and 32nd) class stands out
        z = np.where(np.arange(k) % 256 == 5, 5000.0, 0) + np.where(np.arange(k) % 32 == 5, 3000.0, 0) + z
        z = np.tile(z[0], (n, 1))
    elif order == 'block':
        z[:, k // 3: k // 3 + 200] += 4000
    t = _tensor(torch, z, 'f32', layout)
    for m in (1, 7, 33, 128):
        values, ids, lse, off = ref.top(_given(t), m)
        got = scores.top(t, m)
        assert np.array_equal(got[1].cpu().numpy(), ids) and np.array_equal(got[0].cpu().numpy(), values)
        _close(got[2].cpu().numpy(), lse, off, (order, m))


@pytest.mark.parametrize('kind', TYPES)
@pytest.mark.parametrize('layout,n,k', [('class', 40, 5), ('class', 40, 100), ('row', 40, 5), ('row', 40, 300), ('row', 6, 9001), ('any', 6, 40)])
def test_top_of_unusual_numbers(ops, kind, layout, n, k):
    torch, scores = ops
    r = np.random.default_rng(k)
    low = float(torch.finfo(_type(torch, kind)).min)
    z = _make(r, n, k)
    z[0] = low                               # masked by the type's lowest value, all of it
    z[1] = low
    z[1, k - 2] = 1.0
    z[2] = np.where(np.arange(k) % 2, 0.0, -0.0)   # the zeros are equal
    z[3, 1] = np.nan
    z[4] = np.nan
    z[5, :] = -np.inf
    z[5, k - 1] = low
    t = _tensor(torch, z, kind, layout)
    values, ids, lse, off = ref.top(_given(t), min(k, 8))
    got = scores.top(t, min(k, 8))
    assert np.array_equal(got[1].cpu().numpy(), ids)
    assert np.array_equal(got[0].cpu().numpy(), values)
    _close(got[2].cpu().numpy(), lse, off, kind)


def _teacher(r, z, m, temperature, gaps=False):
    """The m largest of a teacher near z; gaps: entries of no class, classes that stand twice, a row without any."""
    n, k = z.shape
    x = (0.8 * np.where(np.isfinite(z), z, 0) + 1.2 * r.standard_normal((n, k))).astype(np.float32)
    ids = np.full((n, m), -1, np.int32)
    logits = np.full((n, m), -np.inf, np.float32)
    order = np.argsort(-x, axis=1, kind='stable')[:, :m]
    ids[:, :order.shape[1]], logits[:, :order.shape[1]] = order, np.take_along_axis(x, order, 1)
    x = x.astype(np.float64) / temperature
    lse = (x.max(1) + np.log(np.exp(x - x.max(1, keepdims=True)).sum(1)) + 1e-4).astype(np.float32)
    if gaps:
        ids[r.random(ids.shape) < 0.2] = -1
        ids[r.random(ids.shape) < 0.1] = k + 1
        if m > 2:
            ids[:: 2, m // 2] = ids[:: 2, 0]
            ids[:: 3, m - 1] = ids[:: 3, 1]
        ids[0] = -1
        logits[n // 2] = -np.inf
    return ids, logits, lse


def _check_distill(ops, t, kind, ids, logits, logits_kind, lse, labels, weights, temperature, alpha, what):
    torch, scores = ops
    dev = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()   # noqa: E731
    tl = dev(logits).to(_type(torch, logits_kind))
    want = ref.distill(_given(t), ids, _given(tl), lse, labels, weights, temperature, alpha)
    args = dict(lse=dev(lse), labels=dev(labels), weights=dev(weights), temperature=temperature, alpha=alpha)
    loss, none = scores.distill(t, dev(ids), tl, gives='loss', **args)
    assert none is None
    _close(loss.cpu().numpy(), want['loss'], want['loss_off'], what + ('loss',))
    loss, grad = scores.distill(t, dev(ids), tl, gives='gradient', **args)
    assert grad.dtype == t.dtype and grad.shape == t.shape
    _close(loss.cpu().numpy(), want['loss'], want['loss_off'], what + ('loss',))
    off = want['g_off'] + (ref.HALF[kind] * np.abs(want['g']) * (1 + 2.0 ** -8) + ref.TINY[kind] if kind != 'f32' else 0)
    _close(_given(grad), want['g'], off, what + ('gradient',))
    loss, pairs = scores.distill(t, dev(ids), tl, gives='pairs', **args)
    assert pairs.dtype == torch.float32 and tuple(pairs.shape) == (*t.shape, 2)
    p = pairs.cpu().numpy()
    _close(p[..., 0], want['g'], want['g_off'], what + ('pairs g',))
    _close(p[..., 1], want['h'], want['h_off'], what + ('pairs h',))
    _close(loss.cpu().numpy(), want['loss'], want['loss_off'], what + ('loss',))
    return want


@pytest.mark.parametrize('layout', ['row', 'class', 'row+', 'class+', 'any'])
@pytest.mark.parametrize('n,k', SIZES)
def test_distill(ops, n, k, layout):
    torch, scores = ops
    r = np.random.default_rng(n * 1000 + k + 2)
    for kind, lk, m, T, a, with_lse, gaps in (('f32', 'f32', 3, 1.0, 1.0, False, False), ('f32', 'bf16', 16, 2.0, 0.7, True, True),
                                              ('bf16', 'bf16', 40, 2.0, 1.0, True, False), ('f16', 'f32', 128, 1.0, 0.4, False, True),
                                              ('f32', 'f16', 5, 0.8, 0.0, True, False)):
        t = _tensor(torch, _make(r, n, k), kind, layout)
        ids, logits, lse = _teacher(r, _given(t), m, T, gaps)
        labels = r.integers(-1, k + 1, n).astype(np.int32) if a < 1 else None
        weights = r.random(n).astype(np.float32) if gaps else None
        _check_distill(ops, t, kind, ids, logits, lk, lse if with_lse else None, labels, weights, T, a, (kind, m, T, a))


@pytest.mark.parametrize('layout,n,k', [('class', 12, 6), ('class', 12, 90), ('row', 12, 6), ('row', 12, 400), ('row', 12, 9001), ('any', 12, 50)])
def test_distill_of_unusual_numbers(ops, layout, n, k):
    """Students that mask classes, or all of them, or stand far from everything the teacher lists or leaves out."""
    torch, scores = ops
    r = np.random.default_rng(k)
    z = _make(r, n, k)
    ids, logits, lse = _teacher(r, z, 4, 1.0)
    far = np.arange(k)[None, :] != ids[:, :1]
    z[0] = -np.inf                                   # nothing is left: the loss is infinite, the gradient -q
    z[1] = np.where(np.isin(np.arange(k), ids[1]), z[1], -np.inf)   # what is not listed is masked
    z[2, ids[2, 0]] = -np.inf                        # ... or the teacher's first choice
    z[3] = np.finfo(np.float32).min
    z[4] = np.where(np.isin(np.arange(k), ids[4]), z[4] + 300, z[4])    # the rest has no mass that a float holds
    z[5] = np.where(np.isin(np.arange(k), ids[5]), z[5] - 300, z[5])    # ... the listed ones
    z[6] = np.where(far[6], z[6], 200.0)
    lse[7] = 50.0                                    # nearly all mass is left out
    lse[8] = lse[8] - 3                              # more than all mass is listed
    logits[9, 1:] = -np.inf
    t = _tensor(torch, z.astype(np.float32), 'f32', layout)
    labels = r.integers(0, k, n).astype(np.int32)
    labels[2] = ids[2, 0]
    for use_lse in (True, False):
        want = _check_distill(ops, t, 'f32', ids, logits, 'f32', lse if use_lse else None, None, None, 1.0, 1.0, (use_lse,))
        assert np.isinf(want['loss'][0]) and np.isinf(want['loss'][2])
        _check_distill(ops, t, 'f32', ids, logits, 'f32', lse if use_lse else None, labels, None, 1.5, 0.5, (use_lse, 'labels'))


@pytest.mark.parametrize('layout,n,k,m,T,a,rest', [('class', 3, 5, 3, 1.0, 1.0, True), ('class', 3, 40, 6, 2.0, 0.6, True), ('row', 2, 70, 8, 1.3, 0.5, False),
                                                   ('row', 2, 33, 33, 1.0, 1.0, True)])
def test_distill_gradient_against_differences(ops, layout, n, k, m, T, a, rest):
    """The kernel's gradient is the slope of the 64-bit loss: central differences with h = 2^-14 are off by h^2 |f'''| / 6 and by
    rounding, 2^-53 |f| / h; the third derivative of the loss is at most 2 w alpha T^2 / T^3 + 2 per class."""
    torch, scores = ops
    r = np.random.default_rng(k + m)
    z = _make(r, n, k)
    t = _tensor(torch, z, 'f32', layout)
    s = _given(t).astype(np.float64)
    ids, logits, lse = _teacher(r, s, m, T)
    labels = r.integers(0, k, n).astype(np.int32) if a < 1 else None
    args = (ids, logits, lse if rest else None, labels, None, T, a)
    dev = lambda x: None if x is None else torch.from_numpy(x).cuda()   # noqa: E731
    _, grad = scores.distill(t, dev(ids), dev(logits), lse=dev(args[2]), labels=dev(labels), temperature=T, alpha=a)
    off = ref.distill(s, *args)['g_off']
    h = 2.0 ** -14
    for c in range(k):
        up, down = s.copy(), s.copy()
        up[:, c] += h
        down[:, c] -= h
        lo, hi = ref.distill(down, *args)['loss'], ref.distill(up, *args)['loss']
        _close(_given(grad)[:, c], (hi - lo) / (2 * h), off[:, c] + h * h * (2 / T + 2) / 6 + 2.0 ** -50 * (1 + np.abs(hi)) / h, c)


@pytest.mark.parametrize('k', [5, 40])
def test_alpha_zero_gives_the_pairs_of_the_softmax_objective(ops, k):
    torch, scores = ops
    r = np.random.default_rng(k)
    z = _make(r, 50, k).astype(np.float32)
    t = _tensor(torch, z, 'f32', 'class')
    y = r.integers(0, k, 50).astype(np.int32)
    none = torch.full((50, 1), -1, dtype=torch.int32, device='cuda')
    _, pairs = scores.distill(t, none, torch.zeros(50, 1, device='cuda'), labels=torch.from_numpy(y).cuda(), temperature=2.0, alpha=0.0, gives='pairs')
    e = np.exp(z.astype(np.float64) - z.max(1, keepdims=True))
    p = e / e.sum(1, keepdims=True)
    g = p - (np.arange(k) == y[:, None])
    h = np.maximum(2 * p * (1 - p), 1e-16)
    bounds = ref.distill(z, np.full((50, 1), -1), np.zeros((50, 1), np.float32), None, y, None, 2.0, 0.0)
    _close(pairs[..., 0].cpu().numpy(), g, bounds['g_off'], 'g')
    _close(pairs[..., 1].cpu().numpy(), h, bounds['h_off'], 'h')


def test_no_rows(ops):
    torch, scores = ops
    z = torch.empty(0, 9, device='cuda')
    assert scores.adjust(z).shape == (0, 9)
    assert scores.top(z, 3)[0].shape == (0, 3)
    i = torch.empty(0, 2, dtype=torch.int32, device='cuda')
    loss, pairs = scores.distill(z, i, i.float(), gives='pairs')
    assert loss.shape == (0,) and pairs.shape == (0, 9, 2)


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
    for a, b in zip(scores.top(z, 3), scores.top(small, 3)):
        assert torch.equal(a, b)
    bias = torch.randn(z.size(1), device='cuda')
    out = torch.zeros_like(base)
    out = torch.as_strided(out, z.shape, z.stride())
    scores.adjust(z, bias=bias, out=out)
    assert torch.equal(out, scores.adjust(small, bias=bias))
    ids, logits = scores.top(small, 2)[1], scores.top(small, 2)[0]
    for a, b in zip(scores.distill(z, ids, logits), scores.distill(small, ids, logits)):
        assert torch.equal(a, b)


def _set_up(torch, scores, n, k, by):
    g = torch.Generator(device='cuda').manual_seed(n + k)
    z = torch.randn((n, k) if by == 'row' else (k, n), device='cuda', generator=g) * 3
    z = z if by == 'row' else z.t()
    bias = torch.randn(k, device='cuda', generator=g)
    ids = torch.randint(0, k, (n, 6), device='cuda', generator=g, dtype=torch.int32)
    logits = torch.randn(n, 6, device='cuda', generator=g)
    ptr = torch.arange(0, 4 * n + 1, 4, device='cuda')
    past = torch.randint(0, k, (4 * n,), device='cuda', generator=g, dtype=torch.int32)

    def chain():
        a = scores.adjust(z, bias=bias, history=(ptr, past), presence=0.5)
        v, i, lse = scores.top(a, 6, temperature=2.0)
        loss, pairs = scores.distill(z, i, v, lse=lse, temperature=2.0, gives='pairs')
        _, grad = scores.distill(z, ids, logits, alpha=0.5, labels=i[:, 0].contiguous(), temperature=2.0)
        return a, v, i, lse, loss, pairs, grad
    return z, chain


@pytest.mark.parametrize('by,n,k', [('class', 1000, 7), ('class', 500, 200), ('row', 300, 50), ('row', 4, 30011)])
def test_streams_graphs_and_repeats(ops, by, n, k):
    """The operators one after the other: on another stream, captured and replayed on new scores, twice the same bits, and a captured
    run beside an eager one."""
    torch, scores = ops
    z, chain = _set_up(torch, scores, n, k, by)
    want = chain()
    assert all(torch.equal(a, b) for a, b in zip(chain(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = chain()
    z.copy_(z.flip(0).clone())
    want = [t.clone() for t in chain()]
    side.wait_stream(torch.cuda.current_stream())
    graph.replay()
    with torch.cuda.stream(side):
        beside = [chain() for _ in range(3)]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, want))
    assert all(torch.equal(a, b) for run in beside for a, b in zip(run, want))


def test_what_lies_beside_is_left_alone(ops):
    """Rooms behind rows and columns of the outputs keep what they hold."""
    torch, scores = ops
    for by, shape in (('row', (37, 50)), ('row', (5, 9003)), ('class', (37, 50)), ('class', (70, 5))):
        n, k = shape
        z = torch.randn(n, k, device='cuda')
        z = z if by == 'row' else z.t().contiguous().t()
        buf = torch.full((n + 4, k + 9) if by == 'row' else (k + 4, n + 9), 5.0, device='cuda')
        out = buf[2:2 + n, 3:3 + k] if by == 'row' else buf[2:2 + k, 3:3 + n].t()
        scores.adjust(z, out=out, bias=torch.ones(k, device='cuda'))
        assert torch.equal(out, z + 1)
        out.fill_(5.0)
        assert bool((buf == 5.0).all())


def test_lists_that_are_slices(ops):
    torch, scores = ops
    z = torch.randn(60, 80, device='cuda')
    v, i, _ = scores.top(z, 30)
    want = scores.distill(z, i[:, :9].contiguous(), v[:, :9].contiguous(), gives='pairs')
    got = scores.distill(z, i[:, :9], v[:, :9], gives='pairs')
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(ops):
    torch, scores = ops
    z = torch.randn(8, 40, device='cuda')
    v, i, lse = scores.top(z, 4)
    bad = [lambda: scores.top(z.cpu(), 2), lambda: scores.top(z.double(), 2), lambda: scores.top(z[0], 2), lambda: scores.top(z, 0), lambda: scores.top(z, 129),
           lambda: scores.top(z, 2, temperature=0.0), lambda: scores.top(z, 2, temperature=float('nan')), lambda: scores.top(z, 2, temperature=-1.0),
           lambda: scores.adjust(z, out=z[:, ::2]), lambda: scores.adjust(z, out=torch.empty(8, 1, device='cuda').expand(8, 40)),
           lambda: scores.adjust(z[:4], out=z[1:5]), lambda: scores.adjust(z, bias=torch.zeros(39, device='cuda')),
           lambda: scores.adjust(z, bias=torch.zeros(40)), lambda: scores.adjust(z, allowed=torch.zeros(8, 1, dtype=torch.int32, device='cuda')),
           lambda: scores.adjust(z, allowed=torch.zeros(3, 2, dtype=torch.int32, device='cuda')),
           lambda: scores.adjust(z, allowed_row=torch.zeros(8, dtype=torch.int32, device='cuda')),
           lambda: scores.adjust(z, history=(torch.zeros(8, dtype=torch.int64, device='cuda'), i.view(-1))),
           lambda: scores.adjust(z, history=(torch.zeros(9, dtype=torch.int32, device='cuda'), i.view(-1))),
           lambda: scores.adjust(z, repetition=0.0), lambda: scores.adjust(z, presence=float('inf')),
           lambda: scores.distill(z, i.long(), v), lambda: scores.distill(z, i, v[:, :3]), lambda: scores.distill(z, i[:7], v[:7]),
           lambda: scores.distill(z, i, v, gives='both'), lambda: scores.distill(z, i, v, alpha=1.5), lambda: scores.distill(z, i, v, lse=lse[:5]),
           lambda: scores.distill(z, i, v, labels=i[:, 0].long()), lambda: scores.distill(z, i.t().contiguous().t(), v),
           lambda: scores.distill(z, i[:, :0], v[:, :0]), lambda: scores.distill(z, i.cpu(), v)]
    for j, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail(f'call {j} was taken')
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(scores.top(z, 4), (v, i, lse)))
    # two halves of one matrix, side by side, may be in and out
    wide = torch.randn(8, 80, device='cuda')
    want = wide[:, :40] + 1
    assert torch.equal(scores.adjust(wide[:, :40], out=wide[:, 40:], bias=torch.ones(40, device='cuda')), want)


@pytest.mark.parametrize('layout,n,k', [('class', 6, 6), ('class', 6, 90), ('row', 6, 6), ('row', 6, 400), ('row', 6, 9001), ('any', 6, 50), ('class', 6, 5000), ('class', 6, 9001)])
def test_distill_where_all_that_is_left_is_far_below_zero(ops, layout, n, k):
    """Nothing but a few listed scores is above -inf, and they lie hundreds below 0 (or above): shares are those of the same scores moved
    to 0."""
    r = np.random.default_rng(k)
    z = _make(r, n, k)
    ids, logits, lse = _teacher(r, z, 4, 1.0)
    for i, by in enumerate((-300, -90, 300, -3000, 0)):
        z[i] = np.where(np.isin(np.arange(k), ids[i]), z[i] + by, -np.inf)
    t = _tensor(ops[0], z.astype(np.float32), 'f32', layout)
    labels = ids[:, 1].copy()
    for T in (1.0, 1.5):
        for use_lse in (True, False):
            _check_distill(ops, t, 'f32', ids, logits, 'f32', lse if use_lse else None, labels, None, T, 0.5, (T, use_lse))


@pytest.mark.parametrize('kind', TYPES)
@pytest.mark.parametrize('m', [1, 20, 64, 74, 128])
def test_top_of_the_lowest_numbers_among_masked_ones(ops, kind, m):
    """Long rows with nothing but the type's lowest value here and there, each in another thread's hands."""
    torch, scores = ops
    low = float(torch.finfo(_type(torch, kind)).min)
    z = np.full((3, 9001), -np.inf)
    step = 16 // (4 if kind == 'f32' else 2)
    z[0, : 75 * step: step] = low
    z[1, : 75 * step: step] = low
    z[1, 5000] = low / 2
    z[2, ::7] = low
    t = _tensor(torch, z, kind, 'row')
    values, ids, lse, off = ref.top(_given(t), m)
    got = scores.top(t, m)
    assert np.array_equal(got[1].cpu().numpy(), ids) and np.array_equal(got[0].cpu().numpy(), values)
    _close(got[2].cpu().numpy(), lse, off, kind)


@pytest.mark.parametrize('layout,n,k', [('class', 40, 90), ('row', 40, 90), ('class', 12, 900), ('row', 12, 9001), ('any', 12, 50)])
def test_loss_where_nearly_all_mass_is_left_to_the_rest(ops, layout, n, k):
    """At a high temperature the listed classes hold little on both sides, and nearly the same: what is left of the loss is of second order
    in the difference of the two.  An error e of the sum over the unlisted classes moves it by (their difference) e; the
    logarithms of the shares of the rest, and the listed terms, are off by a few steps of the listed mass times what multiplies it."""
    torch, scores = ops
    r = np.random.default_rng(k)
    z = r.standard_normal((n, k)) * 1.5
    T = 6.0
    ids, logits, lse = _teacher(r, z, 3, T)
    t = _tensor(torch, z, 'f32', layout)
    dev = lambda x: torch.from_numpy(x).cuda()   # noqa: E731
    loss, _ = scores.distill(t, dev(ids), dev(logits), lse=dev(lse), temperature=T, gives='loss')
    s = _given(t).astype(np.float64) / T
    want = ref.distill(_given(t), ids, logits, lse, None, None, T, 1.0)['loss']
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    ps = np.take_along_axis(p, ids, 1).sum(1)
    q = np.exp(logits.astype(np.float64) / T - lse[:, None].astype(np.float64))
    far = np.abs(np.log(q)).max(1) + np.abs(np.log(np.take_along_axis(p, ids, 1))).max(1)
    off = T * T * (np.abs(q.sum(1) - ps) * ref.sum_error(3, k) + 8 * ref.U * (q.sum(1) + ps) * (1 + far)) + ref.U * np.abs(want)
    assert (off < 2e-4 * T * T).all()
    _close(loss.cpu().numpy(), want, off, k)
