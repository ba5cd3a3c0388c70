"""The divergence of a row of logits from a teacher's list in 64 bits, from the probabilities of distinct ids."""

import numpy as np


def divergence(row, tv, ti, T=1.0, lse=None, weight=1.0):
    """(loss, gradient [V], scale of the gradient's terms [V]); the row's logits are finite or -inf."""
    l = row.detach().double().cpu().numpy()
    t, ids = tv.detach().double().cpu().numpy() / T, ti.cpu().numpy()
    V = len(l)
    ok = (ids >= 0) & (ids < V)
    t, ids = t[ok], ids[ok]
    zero = np.zeros(V)
    if lse == -np.inf or (lse is None and (len(t) == 0 or t.max() == -np.inf)):
        return 0.0, zero, zero
    norm = lse if lse is not None else t.max() + np.log(np.exp(t - t.max()).sum())
    p = np.zeros(V)
    np.add.at(p, ids, np.exp(t - norm))
    x = (l - l.max()) / T if l.max() > -np.inf else l
    logq = x - np.log(np.exp(x).sum())
    q = np.exp(logq)
    seen = p > 0
    loss = float((p[seen] * (np.log(p[seen]) - logq[seen])).sum())
    grad, size = q - p, q + p
    if lse is not None:
        listed = np.zeros(V, bool)
        listed[ids] = True
        rest, other = max(0.0, 1.0 - p.sum()), q[~listed].sum()
        if (x[~listed] < -700).all() and rest <= 2.0 ** -17 + 2.0 ** -23 * abs(lse):
            rest = 0.0  # the rounding of the log-sum-exp: nothing is left but masked tokens
        if rest > 0:
            with np.errstate(divide="ignore"):
                loss += float(rest * (np.log(rest) - np.log(other)))
        share = rest / other if other > 0 else 0.0
        grad = np.where(listed, grad, q - q * share)
        size = np.where(listed, size, q + q * share)
    return loss, grad * weight / T, size * abs(weight) / T
