"""sample, feedback, norm and norm_backward from their definitions, in 64 bits with NumPy, and how far float arithmetic may be off."""
import numpy as np

from scores_ref import U, f32, sum_error

SLACK = 1 + 2.0 ** -18


def _per_row(v, n, none):
    return np.full(n, none) if v is None else np.full(n, f32(v)) if np.isscalar(v) else np.asarray(v, np.float64)


def sample(z, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """(classes, logs, all_logs, bounds on the errors of both): what a draw is left to has its mass in doubles, good to 2^-33, and logs are
    rounded once; the mass of all classes may be a sum of floats (the relative error of that is the error of its log)"""
    z = z.astype(np.float64)
    n, k = z.shape
    u2 = u.reshape(n, -1).astype(np.float64)
    T, K, P, M = _per_row(temperature, n, 1.0), _per_row(top_k, n, 0), _per_row(top_p, n, 1.0), _per_row(min_p, n, 0.0)
    ids = np.full(u2.shape, -1, np.int32)
    logs, every, off = np.full(u2.shape, np.nan), np.full(u2.shape, np.nan), np.zeros(u2.shape)
    for i in range(n):
        s = z[i]
        if not np.isfinite(T[i]) or T[i] < 0 or np.isnan(s).any() or s.max() == np.inf:
            continue
        if s.max() == -np.inf:
            logs[i] = every[i] = -np.inf
            continue
        if T[i] == 0:
            ids[i], logs[i], every[i] = np.argmax(s), 0, 0
            continue
        w = np.where(s > -np.inf, np.exp((s - s.max()) / T[i]), 0)
        off[i] = sum_error((w * np.where(w > 0, (s.max() - s) / T[i], 0)).sum() / w.sum(), k)
        order = np.argsort(-s, kind='stable')
        order = order[s[order] > -np.inf]
        if M[i] > 0:
            order = order[w[order] >= min(M[i], 1.0)]
        if K[i] > 0:
            order = order[:int(K[i])]
        if P[i] < 1:
            upto = np.cumsum(w[order])
            order = order[:np.searchsorted(upto, max(P[i], 0.0) * upto[-1], side='left') + 1]
        kept = np.zeros(k)
        kept[order] = w[order]
        upto = np.cumsum(kept)
        last = np.flatnonzero(kept)[-1]
        for d, v in enumerate(u2[i]):
            v = v if v > 0 else 0.0
            c = min(np.searchsorted(upto, v * upto[-1], side='right'), last)
            ids[i, d], logs[i, d], every[i, d] = c, np.log(w[c] / upto[-1]), np.log(w[c] / w.sum())
    size = lambda v: U * SLACK * np.abs(np.where(np.isfinite(v), v, 0))   # noqa: E731
    shape = u.shape
    return ids.reshape(shape), logs.reshape(shape), every.reshape(shape), (2.0 ** -32 + size(logs)).reshape(shape), (off * SLACK + size(every)).reshape(shape)


def feedback(s, classes, gains, old=None, reference=None, weights=None, temperature=1.0, clip=None, kl=0.0, entropy=0.0):
    """dict of loss, logs, g, h and bounds on their errors (before a rounding to 16 bits); 'gap': how near a ratio lies to where the
    gradient jumps"""
    s = s.astype(np.float64)
    n, k = s.shape
    shape = classes.shape
    two = lambda v: None if v is None else v.reshape(n, -1)   # noqa: E731
    classes, gains, old, reference = two(classes), two(gains).astype(np.float64), two(old), two(reference)
    T, b, q = f32(temperature), f32(entropy), f32(kl)
    low, high = (1.0, np.inf) if clip is None else clip
    low, high = f32(1 - f32(low)), f32(1 + f32(high))
    out = {name: np.zeros(n) for name in ('loss', 'loss_off')}
    out.update({name: np.zeros((n, k)) for name in ('g', 'h', 'g_off', 'h_off')})
    out['logs'], out['logs_off'] = np.full(classes.shape, -np.inf), np.zeros(classes.shape)
    out['gap'] = np.full(classes.shape, np.inf)
    out['h'][:], out['h_off'][:] = 1e-16, 1e-23   # (1e-16 as a float: off by at most 2^-24 of it, 6e-24)
    chain = (k / 32 + 41) * U
    for i in range(n):
        m = s[i].max()
        if m == -np.inf:
            continue
        y = (s[i] - m) / T
        e = np.exp(y)
        S = e.sum()
        lp, p = y - np.log(S), e / S
        far = np.where(e > 0, -y, 0)
        d = sum_error((p * far).sum(), k) + 2 * U
        each = d + far * 3 * U + 2.0 ** -22 + 4 * U
        H = np.log(S) + (p * far).sum()
        H_off = d + (p * far * (far * 3 * U + 2.0 ** -22 + chain)).sum() + (p * far).sum() * d + U * H
        w = 1.0 if weights is None else float(weights[i])
        c_sum, c_off_sum, size, term, term_off, J = 0.0, 0.0, 0.0, 0.0, 0.0, 0
        at, at_off = np.zeros(k), np.zeros(k)
        for j, a in enumerate(classes[i]):
            if not 0 <= a < k or s[i, a] == -np.inf:
                continue
            J += 1
            out['logs'][i, j], out['logs_off'][i, j] = lp[a], d + U * abs(lp[a])
            A = gains[i, j]
            with np.errstate(over='ignore', invalid='ignore'):
                r = np.exp(lp[a] - float(old[i, j])) if old is not None else 1.0
                out['gap'][i, j] = min(abs(r - low), abs(r - high)) / r
            held = min(max(r, low), high)
            t, c, off_t, off_c = 0.0, 0.0, 0.0, 0.0
            if A != 0:
                t = -min(r * A, held * A)
                c = -r * A if r * A <= held * A else 0.0
                if old is not None:
                    off_t, off_c = abs(r * A) * 2 * d, abs(c) * 2 * d
            if q:
                x = float(reference[i, j]) - lp[a]
                t += q * (np.expm1(x) - x)
                c += -q * np.expm1(x)
                off_t += q * (abs(np.expm1(x)) * d + np.exp(x) * d * d)
                off_c += q * np.exp(x) * 2 * d
            off_c += U * abs(c)
            term, c_sum, size, term_off, c_off_sum = term + t, c_sum + c, size + abs(c), term_off + off_t, c_off_sum + off_c
            at[a] += c
            at_off[a] += off_c + U * abs(c)
        if J == 0 or w == 0:
            continue
        out['loss'][i] = w * (term / J - b * H)
        out['loss_off'][i] = w * (term_off / J + b * H_off) + U * abs(out['loss'][i])
        inner = np.where(e > 0, lp + H, 0)
        yy = np.where(e > 0, np.abs(y), 0)
        out['g'][i] = w / T * ((at - c_sum * p) / J + b * p * inner)
        off = (abs(c_sum) * p * each + c_off_sum * p + at_off) / J
        off = off + b * p * (each * np.abs(inner) + yy * 4 * U + H_off + d + 3 * U * (yy + np.log(S) + H))
        off = off + 4 * U * (p * (abs(c_sum) / J + b * (yy + abs(H - np.log(S)))) + np.abs(at) / J)
        out['g_off'][i] = w / T * off + 4 * U * np.abs(out['g'][i])
        curve, curve_off = 2 * w / T ** 2 * (size / J + b), 2 * w / T ** 2 * c_off_sum / J
        out['h'][i] = np.maximum(curve * p * (1 - p), 1e-16)
        out['h_off'][i] = curve * p * (2 * each + 6 * U) + curve_off * p + 1e-23
    for name in ('g_off', 'h_off', 'loss_off', 'logs_off'):   # (results below 2^-126 may become 0)
        out[name] = out[name] * SLACK + 2.0 ** -120
    for name in ('logs', 'logs_off', 'gap'):
        out[name] = out[name].reshape(shape)
    return out


def norm(s, gain=None, bias=None, eps=1e-5):
    """dict of y, mean, rstd and bounds on their errors (that of y before a rounding to 16 bits); sums are chains of at most k / 32 + 40"""
    s = s.astype(np.float64)
    n, k = s.shape
    there = s != -np.inf
    c = there.sum(1)
    x = np.where(there, s, 0)
    chain = (k / 32 + 42) * U
    eps = f32(eps)
    with np.errstate(invalid='ignore', divide='ignore'):
        mean = np.where(c > 0, x.sum(1) / np.maximum(c, 1), 0)
        mean_off = chain * np.abs(x).sum(1) / np.maximum(c, 1) + U * abs(mean)
        dev = np.where(there, s - mean[:, None], 0)
        var = (dev ** 2).sum(1) / np.maximum(c, 1)
        rstd = np.where(c > 0, 1 / np.sqrt(var + eps), 0)
        # the variance about the rounded mean: larger by the square of what that is off; differences rounded
        rel = 0.5 * (var * (chain + 4 * U) + mean_off ** 2 + 2 * U * abs(mean) * mean_off) / (var + eps) + 3 * U
        y = dev * rstd[:, None]
        y_off = (rstd * mean_off)[:, None] + np.abs(y) * (rel[:, None] + 3 * U)
        g = np.ones(k) if gain is None else gain.astype(np.float64)
        b = np.zeros(k) if bias is None else bias.astype(np.float64)
        out = y * g + b
        off = np.abs(g) * y_off + U * (np.abs(y * g) + np.abs(out))
    return dict(y=np.where(there, out, -np.inf), y_off=off * SLACK, mean=mean, mean_off=mean_off * SLACK, rstd=rstd, rstd_off=rstd * rel * SLACK)


def norm_backward(gy, s, mean, rstd, gain=None):
    """dict of g, to_gain, to_bias and bounds on their errors (that of g before a rounding to 16 bits)"""
    s, mean, rstd = s.astype(np.float64), mean.astype(np.float64)[:, None], rstd.astype(np.float64)[:, None]
    n, k = s.shape
    there = s != -np.inf
    c = np.maximum(there.sum(1, keepdims=True), 1)
    gy = np.where(there, gy.astype(np.float64), 0)
    x = np.where(there, s - mean, 0) * rstd
    a = gy * (1.0 if gain is None else gain.astype(np.float64))
    chain = (k / 32 + 44) * U
    c1, c2 = a.sum(1, keepdims=True) / c, (a * x).sum(1, keepdims=True) / c
    off1, off2 = chain * np.abs(a).sum(1, keepdims=True) / c, (chain + 3 * U) * np.abs(a * x).sum(1, keepdims=True) / c
    g = rstd * np.where(there, a - c1 - x * c2, 0)
    off = rstd * (off1 + np.abs(x) * off2 + 5 * U * (np.abs(a) + np.abs(c1) + np.abs(x * c2))) + 2 * U * np.abs(g)
    rows = (n / 32 + 64) * U
    return dict(g=g, g_off=off * SLACK, to_gain=(gy * x).sum(0), to_gain_off=(rows + 4 * U) * np.abs(gy * x).sum(0) * SLACK,
                to_bias=gy.sum(0), to_bias_off=rows * np.abs(gy).sum(0) * SLACK)
