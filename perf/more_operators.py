"""Drawing answers from the scores of many classes and learning from what came of them, as measurable cases.

A booster of K classes keeps one raw score per row and class, all rows of a class side by side ("by class", the layout of
`Booster.ypred()` and of `predict_raw`); a neural network keeps the scores of a row side by side ("by row", often in 16 bits).
A score of -inf is a class that the row may not have.  Four operators work on either:

sample         a class for every given random number, after temperature, top-k, min-p and top-p
norm           every row's scores at mean 0 and variance 1 over its classes, then a gain and a bias per class
norm_backward  the gradient of that, with the gradients of gain and bias
feedback       loss on classes that were drawn and the gains that followed (clipped importance ratio, distance from a reference,
               entropy), with its gradient or the (gradient, hessian) pairs that trees are grown from

`prepare` makes scores in the layout and type they come in, with the random numbers, draws and gradients that go with them.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
_BYTES = {'f32': 4, 'f16': 2, 'bf16': 2}


def _sample(rows, classes, draws=1, by='class', type='f32', **more):
    c = dict(do='sample', rows=rows, classes=classes, draws=draws, by=by, type=type, pad=0, masked=0.0, temperature=1.0, top_k=0,
             top_p=1.0, min_p=0.0, each=False)
    c.update(more)
    return c


def _norm(rows, classes, by='class', type='f32', **more):
    c = dict(do='norm', rows=rows, classes=classes, by=by, type=type, pad=0, masked=0.0, weights=True)
    c.update(more)
    return c


def _norm_backward(rows, classes, by='class', type='f32', **more):
    return dict(_norm(rows, classes, by, type, **more), do='norm_backward')


def _feedback(rows, classes, draws=1, by='class', type='f32', **more):
    c = dict(do='feedback', rows=rows, classes=classes, draws=draws, by=by, type=type, pad=0, masked=0.0, temperature=1.0, old=True,
             reference=False, weights=False, clip=0.2, kl=0.0, entropy=0.0, gives='pairs')
    c.update(more)
    return c


def listed():
    named = [
        # one request at a time
        ('sample 1x1000', _sample(1, 1000, by='row', top_k=50, top_p=0.95, temperature=0.8)),
        # covtype: a class for every row of the set, for logged decisions or bootstrap labels
        ('sample 581012x7', _sample(581_012, 7)),
        # candidates of a recommender's first stage with some variety, odd number of rows
        ('sample 50003x250', _sample(50_003, 250, masked=0.1, temperature=0.7, min_p=0.02, top_p=0.9)),
        # a serving batch of a network with many classes: every request has its own temperature and limits
        ('sample 256x131072 bf16', _sample(256, 131_072, by='row', type='bf16', each=True)),
        # several answers for every row, nothing cut off; rows of an odd length
        ('sample 16 of 333x50021 f16', _sample(333, 50_021, 16, 'row', 'f16', temperature=0.9)),
        # scores of a booster made comparable with another model's; one of ten classes not allowed
        ('norm 50003x250', _norm(50_003, 250, masked=0.1, weights=False)),
        # scores of a wide network, gain and bias per class
        ('norm 2048x65536 bf16', _norm(2048, 65_536, 'row', 'bf16')),
        # learning gain and bias behind a booster's scores
        ('norm_backward 50003x250', _norm_backward(50_003, 250)),
        # a step of a network's training; rows of an odd length
        ('norm_backward 4096x8191 bf16', _norm_backward(4096, 8191, 'row', 'bf16')),
        # one boosting round on the reference's small set: launches, not bytes
        ('feedback 1605x5', _feedback(1_605, 5)),
        # one boosting round from four logged answers for every row
        ('feedback 4 of 50003x250', _feedback(50_003, 250, 4, weights=True, entropy=0.01)),
        # a step of a wide network's training from its own answers
        ('feedback 1024x131072 bf16', _feedback(1024, 131_072, 1, 'row', 'bf16', reference=True, kl=0.05, entropy=0.003, gives='gradient')),
    ]
    return [dict(name=n, **c) for n, c in named]


def draw(rng):
    """One more case of the same ranges; cost bounded by the largest listed one."""
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    do = rng.choice(['sample', 'sample', 'norm', 'norm_backward', 'feedback', 'feedback'])
    by = rng.choice(['class', 'class', 'row', 'row'])
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
    common = dict(pad=pad, masked=rng.choice([0.0, 0.0, 0.1, 0.5]))
    if do in ('norm', 'norm_backward'):
        make = _norm if do == 'norm' else _norm_backward
        return make(rows, classes, by, kind, weights=rng.random() < 0.7, **common)
    draws = min(rng.choice([1, 1, log_int(2, 64)]), max(1, 8_000_000 // rows))
    temperature = round(rng.uniform(0.5, 1.5), 3) if rng.random() < 0.6 else 1.0
    if do == 'sample':
        return _sample(rows, classes, draws, by, kind, temperature=temperature, each=rng.random() < 0.25,
                       top_k=rng.choice([0, 0, log_int(1, min(classes, 1000))]), top_p=rng.choice([1.0, round(rng.uniform(0.5, 0.99), 3)]),
                       min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.005, 0.2), 4)]), **common)
    return _feedback(rows, classes, draws, by, kind, temperature=temperature, old=rng.random() < 0.8, reference=rng.random() < 0.4,
                     weights=rng.random() < 0.4, clip=rng.choice([0.0, 0.2, 0.3]), kl=rng.choice([0.0, 0.05, 0.2]),
                     entropy=rng.choice([0.0, 0.003, 0.05]), gives=rng.choice(['pairs', 'gradient', 'loss'] if by == 'class' else
                                                                             ['gradient', 'gradient', 'loss', 'pairs']), **common)


# ------------------------------------------------------------------ inputs
def _like_scores(case, gen, fill):
    """rows x classes in the case's layout; fill(shape) makes a piece of it."""
    n, k, t = case['rows'], case['classes'], _TYPES[case['type']]
    long, short = (k, n) if case['by'] == 'class' else (n, k)
    s = torch.empty(long, short + case['pad'], device='cuda', dtype=t)
    step = max(1, (1 << 26) // max(1, short))
    for lo in range(0, long, step):
        part = s[lo:lo + step, :short]
        part.copy_(fill(part.shape))
    s = s[:, :short]
    return s.t() if case['by'] == 'class' else s


def _scores(case, gen):
    """What sums of leaves and output layers look like -- most classes close together, a few so far above that they hold much of
    the mass; masked classes, and where there are any one row without another one."""
    few = min(0.2, 40.0 / case['classes'])
    above = 3.0 - math.log(few)

    def fill(shape):
        x = torch.randn(shape, device='cuda', generator=gen) * 1.5
        x += above * (torch.rand(shape, device='cuda', generator=gen) < few)
        if case['masked']:
            x.masked_fill_(torch.rand(shape, device='cuda', generator=gen) < case['masked'], -math.inf)
        return x
    s = _like_scores(case, gen, fill)
    if case['masked'] and case['rows'] > 2:
        s[case['rows'] // 2] = -math.inf
    return s


def _pick(gen, n, values, dtype):
    i = torch.randint(0, len(values), (n,), device='cuda', generator=gen)
    return torch.tensor(values, device='cuda', dtype=dtype)[i]


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(int(seed))
    n, k = case['rows'], case['classes']
    s = dict(case=dict(case), scores=_scores(case, gen))
    if case['do'] == 'sample':
        shape = (n,) if case['draws'] == 1 else (n, case['draws'])
        s['uniform'] = torch.rand(shape, device='cuda', generator=gen, dtype=torch.float64)
        if case['each']:   # numbers that the requests of a batch come with: 0 and 1 switch a limit off
            s['temperature'] = _pick(gen, n, [0.6, 0.8, 1.0, 1.2], torch.float32)
            s['top_k'] = _pick(gen, n, [0, 0, 1, 20, 50, 200], torch.int32)
            s['top_p'] = _pick(gen, n, [1.0, 0.95, 0.9, 0.5], torch.float32)
            s['min_p'] = _pick(gen, n, [0.0, 0.0, 0.02, 0.1], torch.float32)
        else:
            s.update({name: case[name] for name in ('temperature', 'top_k', 'top_p', 'min_p')})
    elif case['do'] in ('norm', 'norm_backward'):
        s['gain'] = s['bias'] = None
        if case['weights']:
            s['gain'] = 1 + 0.2 * torch.randn(k, device='cuda', generator=gen)
            s['bias'] = 0.3 * torch.randn(k, device='cuda', generator=gen)
        if case['do'] == 'norm_backward':
            s['grad'] = _like_scores(case, gen, lambda shape: 0.1 * torch.randn(shape, device='cuda', generator=gen))
            s['mean'], s['rstd'] = (x.float() for x in _moments(s['scores'].double() if n * k < 1 << 25 else s['scores'].float()))
    else:
        # answers of a model near this one, logged with their log-probabilities; a few are missing
        m, step, t = case['draws'], max(1, (1 << 25) // (k * case['draws'])), case['temperature']
        classes, old = [], []
        for lo in range(0, n, step):
            x = s['scores'][lo:lo + step].float()
            x = (x + 0.15 * torch.randn(x.shape, device='cuda', generator=gen)) / t
            noise = torch.rand((x.shape[0], m, k), device='cuda', generator=gen).clamp_min_(1e-30)
            a = (x[:, None] - (-noise.log_()).log_()).argmax(2)
            classes.append(a)
            old.append((x - torch.logsumexp(x, 1, keepdim=True)).gather(1, a))
        a, old = torch.cat(classes), torch.cat(old)
        missing = torch.rand((n, m), device='cuda', generator=gen) < 0.03
        s['classes'] = torch.where(missing, -1, a).to(torch.int32)
        s['gains'] = torch.randn((n, m), device='cuda', generator=gen)
        old = torch.where(old > -math.inf, old, torch.zeros_like(old))   # (rows without a class; NaN)
        s['old'] = old if case['old'] else None
        s['reference'] = old + 0.2 * torch.randn((n, m), device='cuda', generator=gen) if case['reference'] else None
        s['weights'] = torch.rand(n, device='cuda', generator=gen) + 0.5 if case['weights'] else None
    return s


def _moments(x, eps=1e-5):
    """(mean, 1 / sqrt(variance + eps)) of every row over the classes that it may have; 0, 0 where there are none"""
    there = x > -math.inf
    count = there.sum(1).to(x.dtype)
    x = torch.where(there, x, 0)
    mean = x.sum(1) / count.clamp_min(1)
    var = torch.where(there, x - mean[:, None], 0).square().sum(1) / count.clamp_min(1)
    return mean, torch.where(count > 0, 1 / (var + eps).sqrt(), 0)


# ------------------------------------------------------------------ one pass
def run(state):
    case = state['case']
    if own:
        from thundergbm_b200 import scores
        if case['do'] == 'sample':
            return scores.sample(state['scores'], state['uniform'], temperature=state['temperature'], top_k=state['top_k'],
                                 top_p=state['top_p'], min_p=state['min_p'])
        if case['do'] == 'norm':
            return scores.norm(state['scores'], state['gain'], state['bias'])
        if case['do'] == 'norm_backward':
            grad, gain, bias = scores.norm_backward(state['grad'], state['scores'], state['mean'], state['rstd'], state['gain'],
                                                    weights=case['weights'])
            return (grad, gain, bias) if case['weights'] else (grad,)
        loss, logs, grad = scores.feedback(state['scores'], state['classes'], state['gains'], old=state['old'],
                                           reference=state['reference'], weights=state['weights'], temperature=case['temperature'],
                                           clip=case['clip'] or None, kl=case['kl'] if case['reference'] else 0.0, entropy=case['entropy'], gives=case['gives'])
        return (loss, logs) if grad is None else (loss, logs, grad)
    return {'sample': _plain_sample, 'norm': _plain_norm, 'norm_backward': _plain_norm_backward,
            'feedback': _plain_feedback}[case['do']](state, case)


def _column(v, n):
    return v.double()[:, None] if isinstance(v, torch.Tensor) else torch.full((n, 1), v, device='cuda', dtype=torch.float32).double()


def _plain_sample(state, case):
    # in 64 bits: which class a random number falls on is decided next to borders between sums of many terms
    z = state['scores'].double()
    n, k = z.shape
    u = state['uniform'].reshape(n, -1).contiguous()
    e = ((z - z.amax(1, keepdim=True)) / _column(state['temperature'], n)).exp()
    e = torch.where(z > -math.inf, e, 0)
    limit = _column(state['top_k'], n)
    limit = torch.where(limit > 0, limit, k)
    place = torch.arange(k, device='cuda')[None]
    order = z.argsort(dim=1, descending=True, stable=True)
    w = e.gather(1, order)
    w = torch.where((w >= _column(state['min_p'], n)) & (place < limit), w, 0)
    before = w.cumsum(1) - w
    w = torch.where(before < _column(state['top_p'], n) * w.sum(1, keepdim=True), w, 0)
    kept = torch.zeros_like(e).scatter_(1, order, w)
    sums = kept.cumsum(1)
    mass = sums[:, -1:].contiguous()
    i = torch.searchsorted(sums, u * mass, right=True).clamp_max(k - 1)
    weight = kept.gather(1, i)
    logs = (weight / mass).log()
    none = mass == 0
    logs = torch.where(none, -math.inf, logs)
    overall = torch.where(none, -math.inf, (weight / e.sum(1, keepdim=True)).log())
    i = torch.where(none, -1, i).to(torch.int32)
    shape = state['uniform'].shape
    return i.reshape(shape), logs.float().reshape(shape), overall.float().reshape(shape)


def _plain_norm(state, case):
    s = state['scores']
    x = s.float()
    mean, rstd = _moments(x)
    y = (x - mean[:, None]) * rstd[:, None]
    if state['gain'] is not None:
        y = y * state['gain'] + state['bias']
    return torch.where(x > -math.inf, y, -math.inf).to(s.dtype), mean, rstd


def _plain_norm_backward(state, case):
    s = state['scores']
    x, g = s.float(), state['grad'].float()
    there = x > -math.inf
    count = there.sum(1, keepdim=True).clamp_min(1)
    rstd = state['rstd'][:, None]
    x = torch.where(there, (x - state['mean'][:, None]) * rstd, 0)
    g = torch.where(there, g, 0)
    a = g if state['gain'] is None else g * state['gain']
    c1 = a.sum(1, keepdim=True) / count
    c2 = (a * x).sum(1, keepdim=True) / count
    out = torch.where(there, rstd * (a - c1 - x * c2), 0).to(s.dtype)
    return (out, (g * x).sum(0), g.sum(0)) if case['weights'] else (out,)


def _plain_feedback(state, case):
    t, kind = case['temperature'], state['scores'].dtype
    s = state['scores'].float()
    n, k = s.shape
    a, gains = state['classes'].long(), state['gains']
    z = s / t
    top = z.amax(1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0)
    e = (z - top).exp()
    over = e.sum(1, keepdim=True)
    log_over = over.log()
    p = torch.where(over > 0, e / over, 0)
    at = a.clamp_min(0)
    score = z.gather(1, at)
    counts = (a >= 0) & (score > -math.inf)
    lp = torch.where(counts, score - top - log_over, -math.inf)
    some = torch.where(counts, lp, 0)
    old = some if state['old'] is None else state['old']
    r = (some - old).exp()
    near = r.clamp(1 - case['clip'], 1 + case['clip']) if case['clip'] else r
    term = -torch.minimum(r * gains, near * gains)
    c = torch.where(r * gains <= near * gains, -r * gains, 0)
    if case['kl'] and state['reference'] is not None:
        d = state['reference'] - some
        term = term + case['kl'] * (d.exp() - d - 1)
        c = c + case['kl'] * (1 - d.exp())
    number = counts.sum(1, keepdim=True)
    has = number > 0
    share = torch.where(counts, 1 / number.clamp_min(1), 0)
    w = (state['weights'] if state['weights'] is not None else torch.ones(n, device='cuda'))[:, None]
    log_p = torch.where(e > 0, z - top - log_over, 0)
    h = -(p * log_p).sum(1, keepdim=True)
    b = case['entropy'] * has
    loss = w * ((share * term).sum(1, keepdim=True) - b * h)
    loss = torch.where(has, loss, 0)[:, 0]
    if case['gives'] == 'loss':
        return loss, lp
    c = torch.where(counts, share * c, 0)
    grad = (w / t) * (p * (b * (log_p + h) - c.sum(1, keepdim=True))).scatter_add(1, at, c)
    if case['gives'] == 'gradient':
        return loss, lp, grad.to(kind)
    curve = 2 * w / (t * t) * (c.abs().sum(1, keepdim=True) + b)
    return loss, lp, torch.stack((grad, (curve * p * (1 - p)).clamp_min(1e-16)), 2)


# ------------------------------------------------------------------ floors
def work(case):
    n, k = case['rows'], case['classes']
    cells, s = n * k, _BYTES[case['type']]
    if case['do'] == 'sample':
        return {'bytes': cells * s + n * (20 * case['draws'] + 16 * case['each']), 'flops': 4 * cells}
    if case['do'] == 'norm':
        return {'bytes': 2 * cells * s + 8 * n + 8 * k * case['weights'], 'flops': 8 * cells}
    if case['do'] == 'norm_backward':
        return {'bytes': 3 * cells * s + 8 * n + 12 * k * case['weights'], 'flops': 14 * cells}
    out = {'loss': 0, 'gradient': s, 'pairs': 8}[case['gives']]
    per_row = case['draws'] * (12 + 4 * case['old'] + 4 * case['reference']) + 4 + 4 * case['weights']
    return {'bytes': cells * (s + out) + n * per_row, 'flops': cells * (6 + 6 * bool(out))}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {'sample': _exact_sample, 'norm': _exact_norm, 'norm_backward': _exact_norm_backward,
                'feedback': _exact_feedback}[case['do']](s, case)


def _exact_sample(s, case):
    n, k = case['rows'], case['classes']
    draws = s['uniform'].reshape(n, -1)
    each = {name: _column(s[name], n) for name in ('temperature', 'top_k', 'top_p', 'min_p')}
    ids, logs, overall = [], [], []
    step = max(1, (1 << 24) // k)
    for lo in range(0, n, step):
        part = slice(lo, min(n, lo + step))
        lp = (s['scores'][part].double() / each['temperature'][part]).log_softmax(1)   # NaN in rows without a class
        lp = lp.nan_to_num(nan=-math.inf)
        best, order = lp.sort(dim=1, descending=True, stable=True)
        keep = best > -math.inf
        keep &= best >= best[:, :1] + each['min_p'][part].log()
        limit = each['top_k'][part]
        keep &= (torch.arange(k, device='cuda') < limit) | (limit <= 0)
        q = best.masked_fill(~keep, -math.inf)
        q = (q - q.logsumexp(1, keepdim=True)).exp().nan_to_num(nan=0.0)
        inside = torch.ones_like(keep)
        inside[:, 1:] = q.cumsum(1)[:, :-1] < each['top_p'][part]
        keep &= inside
        some = keep.any(1)[:, None]
        allowed = torch.zeros_like(keep).scatter_(1, order, keep)
        masked = lp.masked_fill(~allowed, -math.inf)
        masked = masked - masked.logsumexp(1, keepdim=True)
        upto = masked.exp().nan_to_num(nan=0.0).cumsum(1)
        i = torch.searchsorted(upto, draws[part].contiguous() * upto[:, -1:], right=True).clamp_max(k - 1)
        ids.append(torch.where(some, i, -1).to(torch.int32))
        logs.append(torch.where(some, masked.gather(1, i), -math.inf))
        overall.append(torch.where(some, lp.gather(1, i), -math.inf))
    shape = s['uniform'].shape
    return torch.cat(ids).reshape(shape), torch.cat(logs).reshape(shape), torch.cat(overall).reshape(shape)


def _exact_norm(s, case):
    n, k = case['rows'], case['classes']
    out = torch.empty(n, k, device='cuda', dtype=torch.float64)
    means, rstds = [], []
    step = max(1, (1 << 24) // k)
    for lo in range(0, n, step):
        z = s['scores'][lo:lo + step].double()
        there = z != -math.inf
        number = there.sum(1, keepdim=True)
        mean = z.masked_fill(~there, 0).sum(1, keepdim=True) / number
        var = ((z - mean) ** 2).masked_fill(~there, 0).sum(1, keepdim=True) / number
        rstd = (var + 1e-5).rsqrt()
        y = (z - mean) * rstd
        if s['gain'] is not None:
            y = y * s['gain'].double() + s['bias'].double()
        out[lo:lo + step] = y.masked_fill(~there, -math.inf)
        means.append(mean.nan_to_num(nan=0.0)[:, 0]); rstds.append(rstd.nan_to_num(nan=0.0)[:, 0])
    return out, torch.cat(means), torch.cat(rstds)


def _exact_norm_backward(s, case):
    n, k = case['rows'], case['classes']
    grads = torch.empty(n, k, device='cuda', dtype=torch.float64)
    gain = s['gain'].double() if s['gain'] is not None else torch.ones(k, device='cuda', dtype=torch.float64)
    to_gain, to_bias = torch.zeros_like(gain), torch.zeros_like(gain)
    step = max(1, (1 << 24) // k)
    for lo in range(0, n, step):
        part = slice(lo, min(n, lo + step))
        z = s['scores'][part].double()
        there = z != -math.inf
        number = there.sum(1, keepdim=True)
        rstd = s['rstd'][part].double()[:, None]
        hat = ((z - s['mean'][part].double()[:, None]) * rstd).masked_fill(~there, 0)
        gy = s['grad'][part].double().masked_fill(~there, 0)
        to_gain += (gy * hat).sum(0)
        to_bias += gy.sum(0)
        a = gy * gain
        inner = a - (a.sum(1, keepdim=True) + hat * (a * hat).sum(1, keepdim=True)) / number
        grads[part] = (rstd * inner).masked_fill(~there, 0)
    return (grads, to_gain, to_bias) if case['weights'] else (grads,)


def _exact_feedback(s, case):
    n, k, t = case['rows'], case['classes'], case['temperature']
    losses, logs, grads = [], [], []
    step = max(1, (1 << 24) // k)
    for lo in range(0, n, step):
        part = slice(lo, min(n, lo + step))
        z = s['scores'][part].double().contiguous().requires_grad_(case['gives'] != 'loss')
        masked = z.detach() == -math.inf
        empty = masked.all(1, keepdim=True)
        lp = (z.masked_fill(masked, -1e300).masked_fill(empty, 0) / t).log_softmax(1)   # (a mask without infinities, for their gradients)
        a = s['classes'][part].long()
        counts = (a >= 0) & ~masked.gather(1, a.clamp_min(0))
        at = lp.gather(1, a.clamp_min(0))
        now = torch.where(counts, at, 0)
        old = s['old'][part].double() if s['old'] is not None else now.detach()
        r, gains = (now - old).exp(), s['gains'][part].double()
        term = -r * gains
        if case['clip']:
            held = (now - old).clamp(math.log1p(-case['clip']), math.log1p(case['clip'])).exp()
            term = torch.where(r.detach() * gains <= held.detach() * gains, term, -held.detach() * gains)
        if case['kl'] and s['reference'] is not None:
            d = s['reference'][part].double() - now
            term = term + case['kl'] * (d.expm1() - d)
        number = counts.sum(1)
        has = number > 0
        w = s['weights'][part].double() if s['weights'] is not None else torch.ones(z.shape[0], device='cuda', dtype=torch.float64)
        p = lp.exp()
        h = -torch.where(masked, 0, p * lp).sum(1)
        loss = (term * counts).sum(1) / number.clamp_min(1) - case['entropy'] * h
        loss = torch.where(has, w * loss, 0)
        losses.append(loss.detach())
        logs.append(torch.where(counts, at.detach(), -math.inf))
        if case['gives'] == 'loss':
            continue
        g, = torch.autograd.grad(loss.sum(), z, retain_graph=case['gives'] == 'pairs')
        if case['gives'] == 'pairs':
            # what one draw's loss changes with its log-probability
            c, = torch.autograd.grad((term * counts).sum(), at)
            each = c.abs().sum(1) / number.clamp_min(1) + case['entropy'] * has
            p = p.detach().masked_fill(masked, 0)
            h = (2 * w * each / (t * t))[:, None] * p * (1 - p)
            g = torch.stack((g, h.clamp_min(1e-16)), 2)
        grads.append(g)
    return (torch.cat(losses), torch.cat(logs)) if case['gives'] == 'loss' else (torch.cat(losses), torch.cat(logs), torch.cat(grads))
