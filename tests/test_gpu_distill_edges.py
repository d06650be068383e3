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


def _teacher_of(n, classes, seed):
    r = np.random.default_rng(seed)
    logits = r.standard_normal((n, classes)) * 2
    ids = np.argsort(-logits, axis=1)[:, :3].astype(np.int32)
    return ids, np.take_along_axis(logits, ids, 1).astype(np.float32), np.log(np.exp(logits / 2).sum(1)).astype(np.float32)


def _rows(n, classes, seed):
    from thundergbm_b200.synth import dense_to_csr
    r = np.random.default_rng(seed)
    y = r.integers(0, classes, n)
    y[:classes] = np.arange(classes)
    return dense_to_csr(r.integers(1, 30, (n, 5)).astype(np.float32), y.astype(np.float32))


def test_a_refused_teacher_leaves_the_one_before(gpu):
    from thundergbm_b200.booster import Booster
    d, t = _rows(1500, 4, 1), _teacher_of(1500, 4, 2)
    par = dict(objective='multi:softprob', num_class=4, depth=4, n_trees=3, hist_mode='exact')
    a, b = Booster(d, **par), Booster(d, **par)
    for x in (a, b):
        x.set_teacher(*t, 2.0, 0.6)
    for bad in (dict(alpha=2.0), dict(temperature=0.0)):
        with pytest.raises(RuntimeError):
            a.set_teacher(*_teacher_of(1500, 4, 3), **bad)
    with pytest.raises(ValueError):
        a.set_teacher(t[0][:5], t[1], t[2])
    assert a.teacher_loss() == b.teacher_loss()
    a.boost(3)
    b.boost(3)
    assert a.trees().tobytes() == b.trees().tobytes()
    other = _teacher_of(1500, 4, 3)
    c, d2 = Booster(d, **par), Booster(d, **par)
    c.set_teacher(*t, 2.0, 0.6)
    c.set_teacher(other[0], other[1], None, 1.0, 0.9)     # (another one takes its place)
    d2.set_teacher(other[0], other[1], None, 1.0, 0.9)
    c.boost(3)
    d2.boost(3)
    assert c.trees().tobytes() == d2.trees().tobytes()


def _rank(rank, world, port, q):
    import os
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for p in (root, os.path.join(root, 'tests')):
        sys.path.insert(0, p)
    import torch
    import torch.distributed as dist
    from thundergbm_b200.booster import Booster, Comm
    os.environ['MASTER_ADDR'] = '127.0.0.1'
    os.environ['MASTER_PORT'] = str(port)
    os.environ.setdefault('NCCL_NVLS_ENABLE', '0')
    os.environ['TGBM_COMM_TIMEOUT_S'] = '60'
    torch.cuda.set_device(rank)
    dist.init_process_group('gloo', rank=rank, world_size=world)
    uid = [Comm.unique_id() if rank == 0 else None]
    dist.broadcast_object_list(uid, src=0)
    comm = Comm(uid[0], rank, world)
    d, t = _rows(3000, 4, 1), _teacher_of(3000, 4, 2)
    lo, hi = 3000 * rank // world, 3000 * (rank + 1) // world
    b = Booster(d.rows(lo, hi), comm=comm, objective='multi:softprob', num_class=4, depth=4, n_trees=3, hist_mode='exact')
    mine = tuple(x[lo:hi] for x in t)
    refused = []
    for bad in (dict(alpha=2.0), dict(temperature=3.0), dict(lse=None), dict(ids=mine[0][:5])):   # of rank 1 alone
        args = dict(ids=mine[0], logits=mine[1], lse=mine[2], temperature=2.0, alpha=0.6)
        if rank == 1:
            args.update(bad)
        try:
            b.set_teacher(**args)
            refused.append(False)
        except (ValueError, RuntimeError):
            refused.append(True)
    b.set_teacher(*mine, 2.0, 0.6)
    b.boost(3)
    q.put((rank, refused, b.trees().tobytes()))
    b.close()
    comm.close()
    dist.barrier()
    dist.destroy_process_group()


def test_ranks_take_a_teacher_together(gpu):
    """What one rank refuses, or says something else for, no rank takes; what they take grows the trees of one GPU.  Skipped on one GPU."""
    import os
    import torch
    import torch.multiprocessing as mp
    if torch.cuda.device_count() < 2:
        pytest.skip('needs 2 GPUs')
    from thundergbm_b200.booster import Booster
    b = Booster(_rows(3000, 4, 1), objective='multi:softprob', num_class=4, depth=4, n_trees=3, hist_mode='exact')
    b.set_teacher(*_teacher_of(3000, 4, 2), 2.0, 0.6)
    b.boost(3)
    want = b.trees().tobytes()
    b.close()
    ctx = mp.get_context('spawn')
    q = ctx.Queue()
    port = 28600 + os.getpid() % 1000
    procs = [ctx.Process(target=_rank, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = [q.get(timeout=300) for _ in procs]
    for p in procs:
        p.join(timeout=120)
    for rank, refused, trees in res:
        assert refused == [True] * 4 and trees == want, rank


@pytest.mark.parametrize('classes,n,top,with_lse', [(1100, 1300, 40, True), (1100, 1300, 3, False), (5600, 5600, 5, True)])
def test_boosters_of_more_than_a_thousand_classes(gpu, classes, n, top, with_lse):
    """Tiles and, of still more classes, a block per row: roots hold the sums of the definition, in the first round and in the second."""
    from thundergbm_b200.booster import Booster
    r = np.random.default_rng(classes + top)
    d = _rows(n, classes, classes)
    y = d.y.astype(np.int32)
    ids = np.stack([r.permutation(classes)[:top] for _ in range(n)]).astype(np.int32)
    ids[::3, 0] = y[::3]
    logits = (r.standard_normal((n, top)) * 2).astype(np.float32)
    lse = (np.log(np.exp(logits.astype(np.float64) / 1.5).sum(1)) + r.uniform(0.01, 2.0, n)).astype(np.float32) if with_lse else None
    b = Booster(d, objective='multi:softprob', num_class=classes, depth=1, n_trees=2, learning_rate=1.0, hist_mode='exact')
    b.set_teacher(ids, logits, lse, 1.5, 0.7)
    for stop in (0, 1):
        s = b.ypred().T.copy() if stop else np.zeros((n, classes), np.float32)
        want = ref.distill(s, ids, logits, lse, y, None, 1.5, 0.7)
        loss = b.teacher_loss()
        assert abs(loss - want['loss'].mean()) <= want['loss_off'].mean() + 2.0 ** -40 * abs(want['loss']).sum()
        b.boost(1)
        _check_roots(b.trees()[stop], want, n, 18)
    b.close()


@pytest.mark.parametrize('n,classes', [(1, 5), (300, 5), (300, 40)])
def test_entries_of_predict_top_under_rules(gpu, n, classes):
    """Every entry that comes back, class by class: the score is the class's under the rules, the classes are those with the largest ones,
    and a row that runs out of allowed classes ends in -1."""
    from thundergbm_b200.thundergbm import TGBMClassifier
    r = np.random.default_rng(classes + n)
    d = _rows(1200, classes, classes)
    x = np.zeros((1200, 5), np.float32)
    x[np.repeat(np.arange(1200), np.diff(d.row_ptr)), d.col] = d.val
    m = TGBMClassifier(depth=4, n_trees=5, learning_rate=0.4, objective='multi:softprob', verbose=0)
    m.fit(x, d.y)
    rows = x[:n]
    s = np.zeros((n, classes), np.float32)
    all_ids, all_values, _ = m.predict_top(rows, classes)
    assert (np.sort(all_ids, 1) == np.arange(classes)).all()
    np.put_along_axis(s, all_ids, all_values, 1)
    bias = r.standard_normal(classes).astype(np.float32)
    allowed = r.random((4, classes)) < 0.5
    allowed[0] = False
    allowed[0, classes // 2] = True
    allowed[1] = False
    row = r.integers(-1, 4, n)
    past = [r.integers(0, classes, r.integers(0, 6)).tolist() for _ in range(n)]
    ptr = np.concatenate([[0], np.cumsum([len(h) for h in past])])
    flat = np.array([c for h in past for c in h], np.int32)
    par = dict(repetition=1.2, frequency=0.1, presence=0.3)
    k = 4
    ids, values, lse = m.predict_top(rows, k, bias=bias, allowed=allowed, allowed_row=row, history=past, temperature=1.5, **par)
    want, off = ref.adjust(s, bias, allowed, row, (ptr, flat), **par)
    off = off + ref.U * np.abs(np.where(np.isfinite(want), want, 0)) * (1 + 2.0 ** -18)   # (rounded once more, to the float that is kept)
    for i in range(n):
        can = int((want[i] > -np.inf).sum())
        got = ids[i][:min(k, can)]
        assert (ids[i][can:] == -1).all() and (values[i][can:] == -np.inf).all()
        assert len(set(got.tolist())) == got.size and (got >= 0).all() and (got < classes).all()
        assert (np.abs(values[i][:got.size] - want[i][got]) <= off[i][got]).all()
        assert (np.diff(values[i][:got.size]) <= 0).all()
        rest = np.setdiff1d(np.flatnonzero(want[i] > -np.inf), got)
        if rest.size:   # none that was left out is larger than the last one by more than both may be off
            assert (want[i][rest] - off[i][rest] <= want[i][got[-1]] + off[i][got[-1]]).all()
        if can == 0:
            assert lse[i] == -np.inf
