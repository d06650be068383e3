"""Operators on the scores of many classes, as measurable cases.

A booster of K classes keeps one raw score per row and class, all rows of a class side by side ("by class", the layout of
`Booster.ypred()` and of `predict_raw`); a neural network that teaches one keeps the scores of a row side by side ("by row",
often in 16 bits).  Three operators work on either:

adjust   penalties for classes that a row was given before, a bias per class, classes that a row may not have
top      the k largest scores of every row with their classes (ties: the lower class first) and the row's log-sum-exp
distill  distance of a student's scores from a teacher's largest ones, mixed with the loss on hard labels: the loss per row,
         its gradient, or the (gradient, hessian) pairs that trees are grown from

`prepare` makes scores in the layout and type they come in, with the masks, histories and teacher's scores that go with them.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
_BYTES = {'f32': 4, 'f16': 2, 'bf16': 2}


def _adjust(rows, classes, by='class', type='f32', **more):
    c = dict(do='adjust', rows=rows, classes=classes, by=by, type=type, pad=0, bias=True, masks=1, history=0,
             repetition=1.0, frequency=0.0, presence=0.0)
    c.update(more)
    return c


def _top(rows, classes, k, by='class', type='f32', **more):
    c = dict(do='top', rows=rows, classes=classes, k=k, by=by, type=type, pad=0, temperature=1.0)
    c.update(more)
    return c


def _distill(rows, classes, k, by='class', type='f32', **more):
    c = dict(do='distill', rows=rows, classes=classes, k=k, by=by, type=type, pad=0, temperature=1.0, alpha=1.0, rest=True,
             weights=False, gives='pairs')
    c.update(more)
    return c


def listed():
    named = [
        # one request at a time: a row of a model with many classes, its mask, what it was given before
        ('adjust 1x1000', _adjust(1, 1000, 'row', masks=1, history=64, repetition=1.2, frequency=0.1, presence=0.1)),
        # a batch scored by a booster: prior correction and a few sets of eligible classes shared by the rows
        ('adjust 50003x250', _adjust(50_003, 250, masks=16, history=24, repetition=1.1, presence=0.2)),
        # scores of a teacher network before its largest ones are kept: a mask per row, long histories
        ('adjust 256x131072 bf16', _adjust(256, 131_072, 'row', 'bf16', masks=256, history=4096, repetition=1.1,
                                           frequency=0.05, presence=0.1)),
        # the answer of a booster for one row
        ('top 5 of 1x1000', _top(1, 1000, 5)),
        # covtype: the three likeliest of seven classes for every row of the set
        ('top 3 of 581012x7', _top(581_012, 7, 3)),
        # candidates of a recommender's first stage, odd number of rows
        ('top 20 of 50003x250', _top(50_003, 250, 20, temperature=0.7)),
        # what is kept of a teacher network's scores
        ('top 64 of 1024x131072 bf16', _top(1024, 131_072, 64, 'row', 'bf16', temperature=2.0)),
        # one boosting round on the reference's small set: launches, not bytes
        ('distill 1605x5', _distill(1_605, 5, 3, alpha=0.5, rest=False)),
        # one boosting round on covtype from a teacher's three likeliest classes and the labels
        ('distill 581012x7', _distill(581_012, 7, 3, temperature=2.0, alpha=0.7, rest=False)),
        # one boosting round of many classes from a teacher's sixteen largest scores, the rest of its mass in one bucket
        ('distill 50003x250', _distill(50_003, 250, 16, temperature=1.5, alpha=0.8, weights=True)),
        # a wide student by row in 16 bits: loss and gradient
        ('distill 2048x65536 bf16', _distill(2048, 65_536, 64, 'row', 'bf16', temperature=2.0, gives='gradient')),
        # the same distance as a metric: rows of an odd length, no gradient
        ('distill 333x50021 f16', _distill(333, 50_021, 20, 'row', 'f16', alpha=0.9, rest=False, gives='loss')),
    ]
    return [dict(name=n, **c) for n, c in named]


def draw(rng):
    """One more case of the same ranges; cost bounded by the largest listed one."""
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    do = rng.choice(['adjust', 'top', 'distill'])
    by = rng.choice(['class', 'class', 'row'])
    if by == 'class':
        classes = log_int(3, 1000)
        rows = log_int(1, min(600_000, 12_000_000 // classes))
        kind = rng.choice(['f32', 'f32', 'f32', 'f16', 'bf16'])
        pad = rng.choice([0, 0, 5, 32])
    else:
        classes = log_int(3, 131_072)
        rows = log_int(1, min(50_000, 24_000_000 // classes))
        kind = rng.choice(['f32', 'f16', 'bf16'])
        pad = rng.choice([0, 0, 3, 64])
    if do == 'adjust':
        history = rng.choice([0, log_int(2, max(2, min(4096, classes))), log_int(2, max(2, min(400, classes)))])
        history = min(history, 8_000_000 // rows)
        return _adjust(rows, classes, by, kind, pad=pad, bias=rng.random() < 0.7,
                       masks=rng.choice([0, 1, min(rows, 16), rows if rows * classes <= 40_000_000 else 16]), history=history,
                       repetition=rng.choice([1.0, 1.1, 1.5]), frequency=rng.choice([0.0, 0.2]), presence=rng.choice([0.0, 0.3]))
    k = min(classes, log_int(1, 128), max(1, 8_000_000 // rows))
    if do == 'top':
        return _top(rows, classes, k, by, kind, pad=pad, temperature=rng.choice([1.0, 0.7, 2.0]))
    return _distill(rows, classes, k, by, kind, pad=pad, temperature=rng.choice([1.0, 1.0, 2.0, 3.5]),
                    alpha=rng.choice([1.0, 1.0, 0.7, 0.3]), rest=rng.random() < 0.5, weights=rng.random() < 0.3,
                    gives=rng.choice(['pairs', 'pairs', 'gradient', 'loss'] if by == 'class' else ['gradient', 'gradient', 'loss', 'pairs']))


# ------------------------------------------------------------------ inputs
def _scores(case, gen, spread):
    """rows x classes: what sums of leaves and output layers look like -- most classes close together, a few so far above
    that they hold much of the mass."""
    n, k, t = case['rows'], case['classes'], _TYPES[case['type']]
    few = min(0.2, 40.0 / k)
    above = 3.0 - math.log(few)
    long, short = (k, n) if case['by'] == 'class' else (n, k)
    s = torch.empty(long, short + case['pad'], device='cuda', dtype=t)
    step = max(1, (1 << 26) // max(1, short))
    for lo in range(0, long, step):
        part = s[lo:lo + step, :short]
        x = torch.randn(part.shape, device='cuda', generator=gen) * spread
        x += above * (torch.rand(part.shape, device='cuda', generator=gen) < few)
        part.copy_(x)
    s = s[:, :short]
    return s.t() if case['by'] == 'class' else s


def _popular(n, k, gen):
    """Classes that come back: small numbers far more often than large ones."""
    u = torch.rand(n, device='cuda', generator=gen)
    return (k * u ** 3).to(torch.int32).clamp_(0, k - 1)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(int(seed))
    n, k = case['rows'], case['classes']
    s = dict(case=dict(case), scores=_scores(case, gen, 1.5))
    if case['do'] == 'adjust':
        s['bias'] = 0.5 * torch.randn(k, device='cuda', generator=gen) if case['bias'] else None
        s['allowed'] = s['allowed_row'] = s['history'] = None
        if case['masks']:
            words = (k + 31) // 32
            bits = torch.randint(-2 ** 31, 2 ** 31, (2, case['masks'], words), device='cuda', generator=gen, dtype=torch.int64)
            s['allowed'] = (bits[0] | bits[1]).to(torch.int32)   # three of four classes
            s['allowed_row'] = torch.randint(0, case['masks'], (n,), device='cuda', generator=gen, dtype=torch.int32)
        if case['history']:
            lengths = torch.randint(0, case['history'] + 1, (n,), device='cuda', generator=gen)
            ptr = torch.zeros(n + 1, device='cuda', dtype=torch.int64)
            ptr[1:] = lengths.cumsum(0)
            s['history'] = (ptr, _popular(int(ptr[-1]), k, gen))
    elif case['do'] == 'distill':
        # the teacher: near the student where it is sure; its largest scores, as they are stored, in the student's type
        m, step = case['k'], max(1, (1 << 26) // k)
        ids, logits, lse = [], [], []
        for lo in range(0, n, step):
            x = 0.8 * s['scores'][lo:lo + step].float() + 1.2 * torch.randn((min(step, n - lo), k), device='cuda', generator=gen)
            v, i = x.topk(m, dim=1)
            ids.append(i.to(torch.int32)); logits.append(v.to(_TYPES[case['type']]))
            lse.append(torch.logsumexp(x / case['temperature'], 1))
        s['ids'], s['logits'] = torch.cat(ids), torch.cat(logits)
        s['lse'] = torch.cat(lse) if case['rest'] else None
        s['labels'] = None
        if case['alpha'] < 1:
            y = s['ids'][:, 0].clone()
            other = torch.randint(0, k, (n,), device='cuda', generator=gen, dtype=torch.int32)
            pick = torch.rand(n, device='cuda', generator=gen)
            y = torch.where(pick < 0.2, other, y)
            s['labels'] = torch.where(pick > 0.95, torch.full_like(y, -1), y)   # a few rows have no label
        s['weights'] = torch.rand(n, device='cuda', generator=gen) + 0.5 if case['weights'] else None
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    case = state['case']
    if own:
        from thundergbm_b200 import scores
        if case['do'] == 'adjust':
            return scores.adjust(state['scores'], bias=state['bias'], allowed=state['allowed'], allowed_row=state['allowed_row'],
                                 history=state['history'], repetition=case['repetition'], frequency=case['frequency'],
                                 presence=case['presence'])
        if case['do'] == 'top':
            return scores.top(state['scores'], case['k'], temperature=case['temperature'])
        loss, grad = scores.distill(state['scores'], state['ids'], state['logits'], lse=state['lse'], labels=state['labels'],
                                    weights=state['weights'], temperature=case['temperature'], alpha=case['alpha'],
                                    gives=case['gives'])
        return (loss,) if grad is None else (loss, grad)
    return {'adjust': _plain_adjust, 'top': _plain_top, 'distill': _plain_distill}[case['do']](state, case)


def _plain_adjust(state, case):
    z = state['scores'].float()
    n, k = z.shape
    if state['history'] is not None:
        ptr, ids = state['history']
        row = torch.repeat_interleave(torch.arange(n, device='cuda'), ptr[1:] - ptr[:-1], output_size=ids.numel())
        count = torch.zeros(n, k, device='cuda').index_put_((row, ids.long()), torch.ones(1, device='cuda'), accumulate=True)
        seen = count > 0
        z = torch.where(seen, torch.where(z > 0, z / case['repetition'], z * case['repetition']), z)
        z = z - case['frequency'] * count - case['presence'] * seen
    if state['bias'] is not None:
        z = z + state['bias']
    if state['allowed'] is not None:
        c = torch.arange(k, device='cuda')
        word = state['allowed'][state['allowed_row'].long()][:, c >> 5]
        z = torch.where(((word >> (c & 31)) & 1) == 1, z, -math.inf)
    return z.to(state['scores'].dtype)


def _plain_top(state, case):
    z = state['scores'].float()
    lse = _log_sum_exp(z / case['temperature'])
    left = z.clone()
    values, ids = [], []
    for _ in range(case['k']):
        i = left.argmax(1, keepdim=True)   # the first of equals
        v = left.gather(1, i)
        left.scatter_(1, i, -math.inf)
        values.append(v)
        ids.append(torch.where(v == -math.inf, -1, i).to(torch.int32))
    return torch.cat(values, 1), torch.cat(ids, 1), lse


def _log_sum_exp(x):
    top = x.amax(1, keepdim=True)
    return (top + (x - top).exp().sum(1, keepdim=True).log())[:, 0]


def _plain_distill(state, case):
    t, a, kind = case['temperature'], case['alpha'], state['scores'].dtype
    s, ids = state['scores'].float(), state['ids'].long()
    n, k = s.shape
    w = state['weights'] if state['weights'] is not None else torch.ones(n, device='cuda')
    # the teacher's few numbers in 64 bits: what is left of its mass is a difference of nearly equal ones
    u = state['logits'].double() / t
    log_q = u - (state['lse'].double()[:, None] if case['rest'] else torch.logsumexp(u, 1, keepdim=True))
    q = log_q.exp()
    mass = q.sum(1)
    rest = (1 - mass).clamp_min(0) if case['rest'] and case['k'] < k else torch.zeros_like(mass)
    total = (mass + rest).float()[:, None]
    at_t = s / t
    top = at_t.amax(1, keepdim=True)
    e = (at_t - top).exp()
    over = e.sum(1, keepdim=True)
    p = e / over
    log_p = (at_t.gather(1, ids) - top).double() - over.double().log()
    term = (q * (log_q - log_p)).sum(1)
    q = q.float()
    grad = p * total
    if case['rest'] and case['k'] < k:
        p_rest = (e.scatter(1, ids, 0.0).sum(1) / over[:, 0]).double()
        term = term + torch.where(rest > 0, rest * (rest / p_rest).log(), 0.0)
        factor = (rest / p_rest).float()[:, None]
        listed = torch.zeros_like(p).scatter_(1, ids, 1.0)
        grad = grad - p * factor * (1 - listed)
    grad = a * t * grad.scatter_add(1, ids, -q)
    loss = a * t * t * term
    hess = a * p * (1 - p)
    if state['labels'] is not None:
        y = state['labels'].long()
        has = (y >= 0)
        y = y.clamp_min(0)[:, None]
        top = s.amax(1, keepdim=True)
        e = (s - top).exp()
        over = e.sum(1, keepdim=True)
        p1 = e / over
        hard = (1 - a) * has.float()[:, None]
        loss = loss + hard[:, 0] * (over.double().log() - (s.gather(1, y) - top).double())[:, 0]
        grad = grad + hard * p1.scatter_add(1, y, -torch.ones_like(y, dtype=torch.float32))
        hess = hess + hard * p1 * (1 - p1)
    loss = (w * loss).float()
    if case['gives'] == 'loss':
        return (loss,)
    grad = w[:, None] * grad
    if case['gives'] == 'gradient':
        return loss, grad.to(kind)
    return loss, torch.stack((grad, (2 * w[:, None] * hess).clamp_min(1e-16)), 2)


# ------------------------------------------------------------------ floors
def work(case):
    n, k = case['rows'], case['classes']
    cells, s = n * k, _BYTES[case['type']]
    if case['do'] == 'adjust':
        given = n * case['history'] // 2
        masks = min(case['masks'], n)
        return {'bytes': 2 * cells * s + 4 * k * bool(case['bias']) + masks * ((k + 31) // 32) * 4 + 4 * n * bool(masks) +
                4 * given + 8 * (n + 1) * bool(case['history']), 'flops': 2 * cells + 4 * given}
    if case['do'] == 'top':
        return {'bytes': cells * s + n * (8 * case['k'] + 4), 'flops': 4 * cells}
    out = {'loss': 0, 'gradient': s, 'pairs': 8}[case['gives']]
    per_row = case['k'] * (4 + s) + 4 + 4 * bool(case['rest']) + 4 * (case['alpha'] < 1) + 4 * bool(case['weights'])
    two = 2 if case['alpha'] < 1 and case['temperature'] != 1 else 1
    return {'bytes': cells * (s + out) + n * per_row, 'flops': cells * (4 * two + (6 * two if out else 0))}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {'adjust': _exact_adjust, 'top': _exact_top, 'distill': _exact_distill}[case['do']](s, case)


def _exact_adjust(s, case):
    n, k = case['rows'], case['classes']
    z = s['scores'].double().contiguous()
    if s['history'] is not None:
        ptr, ids = s['history']
        length = ptr.diff()
        cell = torch.arange(n, device='cuda').repeat_interleave(length) * k + ids
        cell, count = torch.unique(cell, return_counts=True)
        flat = z.view(-1)
        v = flat[cell]
        v = torch.where(v > 0, v / case['repetition'], v * case['repetition'])
        flat[cell] = v - count * case['frequency'] - case['presence']
    if s['bias'] is not None:
        z += s['bias'].double()
    if s['allowed'] is not None:
        shift = torch.arange(32, device='cuda', dtype=torch.int32)
        bits = torch.bitwise_and(s['allowed'][:, :, None] >> shift, 1).reshape(case['masks'], -1)[:, :k]
        z.masked_fill_(bits[s['allowed_row'].long()] == 0, -math.inf)
    return z


def _exact_top(s, case):
    n, k, m = case['rows'], case['classes'], case['k']
    values, ids, lse = [], [], []
    step = max(1, (1 << 24) // k)
    for lo in range(0, n, step):
        z = s['scores'][lo:lo + step].double()
        v, i = torch.sort(z, dim=1, descending=True, stable=True)
        values.append(v[:, :m].clone()); ids.append(i[:, :m].to(torch.int32))
        lse.append(torch.logsumexp(z / case['temperature'], 1))
    return torch.cat(values), torch.cat(ids), torch.cat(lse)


def _exact_distill(s, case):
    n, k, t, a = case['rows'], case['classes'], case['temperature'], case['alpha']
    losses, grads = [], []
    step = max(1, (1 << 25) // k)
    for lo in range(0, n, step):
        part = slice(lo, min(n, lo + step))
        z = s['scores'][part].double().contiguous().requires_grad_(case['gives'] != 'loss')
        ids, u = s['ids'][part].long(), s['logits'][part].double() / t
        w = s['weights'][part].double() if s['weights'] is not None else torch.ones(z.shape[0], device='cuda', dtype=torch.float64)
        log_p = (z / t).log_softmax(1)
        if case['rest']:
            log_q = u - s['lse'][part].double()[:, None]
        else:
            log_q = u.log_softmax(1)
        q = log_q.exp()
        soft = (q * (log_q - log_p.gather(1, ids))).sum(1)
        if case['rest'] and case['k'] < k:
            left = (1 - q.sum(1)).clamp_min(0)
            log_rest = torch.logsumexp(log_p.scatter(1, ids, -math.inf), 1)
            soft = soft + torch.xlogy(left, left) - left * log_rest
        loss = a * t * t * soft
        p = log_p.detach().exp()
        hess = a * p * (1 - p)
        if s['labels'] is not None:
            y = s['labels'][part].long()
            log_p1 = z.log_softmax(1)
            has = (y >= 0).double() * (1 - a)
            loss = loss - has * log_p1.gather(1, y.clamp_min(0)[:, None])[:, 0]
            p1 = log_p1.detach().exp()
            hess = hess + has[:, None] * p1 * (1 - p1)
        loss = w * loss
        losses.append(loss.detach())
        if case['gives'] != 'loss':
            g, = torch.autograd.grad(loss.sum(), z)
            grads.append(g if case['gives'] == 'gradient' else
                         torch.stack((g, (2 * w[:, None] * hess).clamp_min(1e-16)), 2))
    return (torch.cat(losses),) if case['gives'] == 'loss' else (torch.cat(losses), torch.cat(grads))
