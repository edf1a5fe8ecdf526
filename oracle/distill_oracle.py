"""Float64 statement of distillation from a teacher's top logits (numpy, CPU; test infrastructure only)."""
import numpy as np


def _lse(v):
    m = v.max() if v.size else -np.inf
    return m if not np.isfinite(m) else m + np.log(np.exp(v - m).sum())


def distill(z, values, index, targets=None, tail=None, T=1.0, alpha=1.0):
    """Row losses and the gradient of each row's loss (not divided by the batch)."""
    z = np.asarray(z, np.float64)
    B, C = z.shape
    loss, grad = np.zeros(B), np.zeros((B, C))
    for b in range(B):
        keep = index[b] >= 0
        idx, t = index[b][keep], np.asarray(values[b], np.float64)[keep] / T
        listed = np.zeros(C, bool)
        listed[idx] = True
        y = z[b] / T
        ly = _lse(y)
        soft = np.exp(y - ly)
        rest = -np.inf if tail is None else float(tail[b])
        ends = np.append(t, rest)
        lt = _lse(ends)
        if alpha > 0 and lt > -np.inf:
            logp = ends - lt
            p = np.exp(logp)
            logq = np.append(y[idx] - ly, (_lse(y[~listed]) - ly) if tail is not None else 0.0)
            on = p > 0
            loss[b] += alpha * T * T * (p[on] * (logp[on] - logq[on])).sum()
            d = soft.copy()
            np.subtract.at(d, idx, p[:-1])
            if tail is not None and p[-1] > 0:
                d[~listed] -= p[-1] * np.exp(y[~listed] - _lse(y[~listed]))
            grad[b] += alpha * T * d
        if alpha < 1.0 and targets[b] >= 0:
            l1 = _lse(z[b])
            loss[b] += (1 - alpha) * (l1 - z[b, targets[b]])
            h = np.exp(z[b] - l1)
            h[targets[b]] -= 1
            grad[b] += (1 - alpha) * h
    return loss, grad


def sizes(z, values, index, targets=None, tail=None, T=1.0, alpha=1.0):
    """Of every component of ``distill``'s gradient: the size of the terms that it is a sum of, and how far its exponents lie from the
    row's maximum, |z - max z| / min(T, 1) (what an error of the exponents' arguments is relative to)."""
    z = np.asarray(z, np.float64)
    B, C = z.shape
    mag, far = np.zeros((B, C)), np.zeros((B, C))
    for b in range(B):
        keep = index[b] >= 0
        idx, t = index[b][keep], np.asarray(values[b], np.float64)[keep] / T
        listed = np.zeros(C, bool)
        listed[idx] = True
        y = z[b] / T
        far[b] = (z[b].max() - z[b]) / min(T, 1.0)
        rest = -np.inf if tail is None else float(tail[b])
        ends = np.append(t, rest)
        lt = _lse(ends)
        if alpha > 0 and lt > -np.inf:
            p = np.exp(ends - lt)
            m = np.exp(y - _lse(y))
            np.add.at(m, idx, p[:-1])
            if tail is not None and p[-1] > 0:
                m[~listed] += p[-1] * np.exp(y[~listed] - _lse(y[~listed]))
            mag[b] += alpha * T * m
        if alpha < 1.0 and targets[b] >= 0:
            h = np.exp(z[b] - _lse(z[b]))
            h[targets[b]] += 1
            mag[b] += (1 - alpha) * h
    return mag, far
