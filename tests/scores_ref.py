"""The operators on scores from their definitions, in 64 bits with NumPy, row by row, and how far float arithmetic may be off."""
import numpy as np

U = 2.0 ** -24   # half a step of a float, relative
HALF = {'f32': 2.0 ** -24, 'f16': 2.0 ** -11, 'bf16': 2.0 ** -8}
TINY = {'f32': 0.0, 'f16': 2.0 ** -25, 'bf16': 0.0}   # half a step of the smallest numbers


def f32(x):
    return float(np.float32(x))


def adjust(z, bias=None, allowed=None, allowed_row=None, history=None, repetition=1.0, frequency=0.0, presence=0.0):
    """(result, bound on the error of float arithmetic before the last rounding); allowed: masks x classes of truth values."""
    z = z.astype(np.float64).copy()
    n, k = z.shape
    r, f, p = f32(repetition), f32(frequency), f32(presence)
    off = np.zeros_like(z)
    if history is not None:
        ptr, ids = history
        for i in range(n):
            h = ids[ptr[i]:ptr[i + 1]]
            h = h[(h >= 0) & (h < k)]
            c = np.bincount(h, minlength=k)
            s = c > 0
            z1 = np.where(z[i] > 0, z[i] / r, z[i] * r)
            z2 = z1 - (c * f + p)
            with np.errstate(invalid='ignore'):
                off[i] = np.where(s, U * (abs(z1) + abs(c * f) + abs(c * f + p) + abs(z2)), 0)
            z[i] = np.where(s, z2, z[i])
    if bias is not None:
        z = z + bias.astype(np.float64)
        off += U * abs(z)
    if allowed is not None:
        row = np.arange(n) if allowed_row is None else allowed_row
        for i in range(n):
            if 0 <= row[i] < allowed.shape[0]:
                z[i][~allowed[row[i]]] = -np.inf
    return z, off * (1 + 2.0 ** -18)


def top(z, k, temperature=1.0):
    """(values, classes, lse, bound on the error of lse)"""
    z = z.astype(np.float64)
    n, m = z.shape
    T = f32(temperature)
    values, ids = np.full((n, k), -np.inf), np.full((n, k), -1, np.int32)
    lse, off = np.zeros(n), np.zeros(n)
    for i in range(n):
        can = np.flatnonzero(z[i] > -np.inf)   # (not NaN either)
        order = can[np.argsort(-z[i][can], kind='stable')][:k]
        values[i, :order.size], ids[i, :order.size] = z[i][order], order
        if np.isnan(z[i]).any():
            lse[i] = np.nan
        elif can.size == 0:
            lse[i] = -np.inf
        else:
            t = z[i].max()
            x = (z[i][can] - t) / T
            e = np.exp(x)
            lse[i] = t / T + np.log(e.sum())
            off[i] = sum_error((e * abs(x)).sum() / e.sum(), m) + U * abs(lse[i])
    return values, ids, lse, off * (1 + 2.0 ** -18)


def sum_error(far, k):
    """Relative error of a float sum of exponentials of k scores: the exponents (x, x c and c are rounded, `far` is the mean of |x|
    over the mass), the exponential (2^-22), additions one after the other in a chain of at most k / 32 + 40."""
    return far * 3 * U + 2.0 ** -22 + (k / 32 + 40) * U


def distill(s, ids, logits, lse=None, labels=None, weights=None, temperature=1.0, alpha=1.0):
    """dict of loss, g, h and bounds on their errors (before a rounding to 16 bits)"""
    s = s.astype(np.float64)
    n, k = s.shape
    T, a = f32(temperature), f32(alpha)
    out = {name: np.zeros(n) for name in ('loss', 'loss_off')}
    out.update({name: np.zeros((n, k)) for name in ('g', 'h', 'g_off', 'h_off')})
    with np.errstate(divide='ignore', invalid='ignore', over='ignore'):
        for i in range(n):
            w = 1.0 if weights is None else float(weights[i])
            ok = (ids[i] >= 0) & (ids[i] < k)
            j, t = ids[i][ok], logits[i][ok].astype(np.float64) / T
            has = t.size > 0 and t.max() > -np.inf
            L = float(lse[i]) if lse is not None else (t.max() + np.log(np.exp(t - t.max()).sum()) if has else 0.0)
            q = np.zeros(k)
            listed = np.zeros(k, bool)
            if has:
                np.add.at(q, j, np.exp(t - L))
                listed[j] = True
            r = max(0.0, 1 - q.sum()) if has and lse is not None and not listed.all() else 0.0
            Q = q.sum() + r

            def softmax(x):
                m = x.max()
                if m == -np.inf:
                    return np.zeros(k), np.full(k, -np.inf), np.zeros(k)
                e = np.exp(x - m)
                return e / e.sum(), x - m - np.log(e.sum()), np.where(e > 0, m - x, 0)
            p, lp, far = softmax(s[i] / T)
            p1, lp1, far1 = softmax(s[i])
            mean = lambda p, far: sum_error((p * far).sum(), k)   # noqa: E731
            d, d1 = mean(p, far), mean(p1, far1)                  # relative errors of the two sums
            each, each1 = d + far * 3 * U + 2.0 ** -22 + 4 * U, d1 + far1 * 3 * U + 2.0 ** -22 + 4 * U   # ... of the shares
            y = -1 if labels is None or not 0 <= labels[i] < k else int(labels[i])
            hard = 1 - a if y >= 0 else 0.0
            soft = a if has else 0.0
            share = np.zeros(k)   # of the unlisted classes' mass
            log_r, d_r = 0.0, 0.0
            if r > 0:
                if (s[i][~listed] > -np.inf).any():
                    m = s[i][~listed].max()
                    e = np.where(listed, 0, np.exp((s[i] - m) / T))
                    share = e / e.sum()
                    far_r = np.where(share > 0, (m - s[i]) / T, 0)
                    log_r = (m - s[i].max()) / T + np.log(e.sum()) - np.log(np.exp((s[i] - s[i].max()) / T).sum())
                    d_r = sum_error((share * far_r).sum(), k)
                    each = each + far_r * 3 * U + d_r
                else:
                    log_r = -np.inf
            kl = sum(q[c] * (np.log(q[c]) - lp[c]) for c in np.flatnonzero(q)) + (r * (np.log(r) - log_r) if r > 0 else 0.0)
            loss = w * ((soft * T * T * kl if soft else 0.0) + (hard * -lp1[y] if hard else 0.0))
            far_q = abs(np.where(q > 0, lp, 0)) + abs(np.log(np.where(q > 0, q, 1)))
            off = soft * T * T * (q.sum() * d + (q * far_q).sum() * 2 * U + r * (d + d_r + U * (abs(np.log(r)) + abs(log_r) + 2) if r > 0 else 0))
            off += soft * T * T * U * (abs(np.log(r / np.exp(log_r))) + 2) if r > 0 else 0.0   # (rest is rounded, 1 - sum q)
            off += hard * d1
            out['loss'][i], out['loss_off'][i] = loss, w * off + U * abs(loss)
            one = np.zeros(k)
            if y >= 0:
                one[y] = 1
            out['g'][i] = w * (soft * T * (Q * p - q - r * share) + hard * (p1 - one))
            out['g_off'][i] = w * (soft * T * ((Q * p + r * share) * each + (q + r * share) * 4 * U) + hard * (p1 * each1 + one * U)) + 4 * U * abs(out['g'][i]) + \
                w * 4 * U * (soft * T * (Q * p + q) + hard * p1)
            curve, curve1 = soft * p * (1 - p), hard * p1 * (1 - p1)
            out['h'][i] = np.maximum(2 * w * (curve + curve1), 1e-16)
            out['h_off'][i] = 2 * w * (soft * p * (2 * each + 4 * U) + hard * p1 * (2 * each1 + 4 * U)) + 1e-23
    # (results below 2^-126 may become 0)
    for name in ('g_off', 'h_off', 'loss_off'):
        out[name] = out[name] * (1 + 2.0 ** -18) + 2.0 ** -120
    return out
