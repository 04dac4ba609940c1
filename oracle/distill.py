"""Top-logit distillation, written from its definition in numpy and 64 bits
(include/pesti_sampler.h); the checker of the distillation tests."""
import numpy as np


def _log(x):
    with np.errstate(divide="ignore"):
        return np.log(x)


def row(x, idx, val, T, lse=None, w=1.0):
    """(loss, gradient [V], and the scale tolerances are counted in: p, Q + q_t,
    q_t / p_t) of one row; x, idx, val as numpy arrays of their exact values."""
    V = len(x)
    x = x.astype(np.float64)
    zero = np.zeros(V)
    if w == 0:
        return 0.0, zero, zero, 0.0, 0.0
    keep = (idx >= 0) & (idx < V)
    idx, t = idx[keep].astype(np.int64), val[keep].astype(np.float64) / T
    nan = np.full(V, np.nan)
    if np.isnan(x).any() or (x == np.inf).any() or np.isnan(t).any():
        return np.nan, nan, nan, np.nan, np.nan
    m = x.max()
    if m == -np.inf:
        p, logp = zero, np.full(V, -np.inf)
    else:
        z = (x - m) / T
        s = np.exp(z).sum()
        p, logp = np.exp(z) / s, z - np.log(s)
    if lse is None:
        if len(t) == 0 or t.max() == -np.inf:
            logq = np.full(len(t), -np.inf)
        else:
            logq = t - t.max() - np.log(np.exp(t - t.max()).sum())
    else:
        logq = t - float(lse)
    q = np.exp(logq)
    member = np.zeros(V, bool)
    member[idx] = True
    q_t = p_t = 0.0
    logp_t = 0.0
    if lse is not None:
        q_t = max(0.0, 1.0 - q.sum())
        rest = logp[~member]
        if rest.size == 0 or rest.max() == -np.inf:
            q_t = 0.0
        else:
            logp_t = rest.max() + np.log(np.exp(rest - rest.max()).sum())
            p_t = np.exp(logp_t)
            if p_t == 0.0:
                q_t = 0.0
    loss = 0.0
    for qj, lq, i in zip(q, logq, idx):
        if qj != 0:
            loss += qj * (lq - logp[i])
    if q_t != 0:
        loss += q_t * (np.log(q_t) - logp_t)
    total = q.sum() + q_t
    ratio = q_t / p_t if q_t != 0 else 0.0
    grad = p * total
    grad[~member] -= ratio * p[~member]
    np.subtract.at(grad, idx, q)
    return w * T * T * loss, w * T * grad, p, total, ratio


def batch(x, idx, val, T, lse=None, weight=None):
    out = [row(x[n], idx[n], val[n], T, None if lse is None else lse[n], 1.0 if weight is None else float(weight[n]))
           for n in range(x.shape[0])]
    return (np.array([o[0] for o in out]), np.stack([o[1] for o in out]), np.stack([o[2] for o in out]),
            np.array([o[3] for o in out]), np.array([o[4] for o in out]))
