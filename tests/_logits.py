"""The operators on rows of logits in 64 bits, one row at a time on the host."""

import numpy as np
import torch


def values(row: torch.Tensor) -> np.ndarray:
    """float64 of a row, NaN as -infinity."""
    x = row.detach().double().cpu().numpy().copy()
    x[np.isnan(x)] = -np.inf
    return x


def order(l: np.ndarray) -> np.ndarray:
    """ids by (logit descending, id ascending)."""
    return np.argsort(-l, kind="stable")


def weights(l: np.ndarray, T: float) -> np.ndarray:
    if l.max() == -np.inf:
        return np.zeros_like(l)
    if not T > 0:
        w = np.zeros_like(l)
        w[int(l.argmax())] = 1.0
        return w
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((l - l.max()) / T)
    w[l == l.max()] = 1.0
    return np.nan_to_num(w, nan=0.0)


def draw(w: np.ndarray, u: float) -> int:
    if not w.sum() > 0:
        return -1
    cum = np.cumsum(w)
    over = np.nonzero((cum > u * cum[-1]) & (w > 0))[0]
    return int(over[0]) if len(over) else int(np.nonzero(w > 0)[0][-1])


def sample(row, u, T=1.0, top_k=0, top_p=1.0, min_p=0.0) -> int:
    l = values(row)
    if l.max() == -np.inf:
        return -1
    if not T > 0:
        return int(l.argmax())
    w, o = weights(l, T), order(l)
    n = len(l) if top_k <= 0 else min(int(top_k), len(l))
    if top_p < 1:
        mass = np.cumsum(w[o[:n]])
        before = np.concatenate([[0.0], mass[:-1]])
        n = max(1, int((before < top_p * mass[-1]).sum()))
    kept = np.zeros_like(w)
    kept[o[:n]] = w[o[:n]]
    kept[w < min(min_p, 1.0)] = 0.0
    return draw(kept, float(u))


def topk(row, k):
    """(float64 values, ids)."""
    l = values(row)
    ids = order(l)[:k]
    return l[ids], ids


def logsumexp(row, T=1.0) -> float:
    l = values(row)
    if not np.isfinite(l.max()):
        return float(l.max())
    return float(l.max() / T + np.log(np.exp((l - l.max()) / T).sum()))


def speculative(logits, draft, ids, u, T=1.0, Td=None):
    """(tokens, accepted) of one sequence: logits [n + 1, V], draft [n, V], ids [n], u [n + 1]."""
    Td = T if Td is None else Td
    n, V = len(ids), logits.shape[-1]
    tokens, j, q = [], 0, None

    def prob(row, t):
        w = weights(values(row), t)
        return w / w.sum() if w.sum() > 0 else w

    while j < n and 0 <= int(ids[j]) < V:
        p, q_j, d = prob(logits[j], T), prob(draft[j], Td), int(ids[j])
        if not float(u[j]) * q_j[d] < p[d]:
            q = q_j
            break
        tokens.append(d)
        j += 1
    p = prob(logits[j], T)
    rest = p if q is None else np.maximum(p - q, 0.0)
    if q is not None and not rest.sum() > 0:
        rest = p
    tokens.append(draw(rest, float(u[n])))
    return tokens + [-1] * (n - j), j


def distill(row, tv, ti, T=1.0, lse=None, weight=1.0):
    """(loss, gradient [V], scale of the gradient's terms [V]) in float64; infinities and NaN of the
    logits' row are left to the caller."""
    l = row.detach().double().cpu().numpy()
    t, ids = tv.detach().double().cpu().numpy() / T, ti.cpu().numpy()
    V = len(l)
    ok = (ids >= 0) & (ids < V)
    t, ids = t[ok], ids[ok]
    zero = np.zeros(V)
    if lse is None:
        if len(t) == 0 or t.max() == -np.inf:
            return 0.0, zero, zero
        logp = t - (t.max() + np.log(np.exp(t - t.max()).sum()))
    else:
        if lse == -np.inf:
            return 0.0, zero, zero
        logp = t - lse
    p = np.exp(logp)
    x = l / T
    logq = x - (x.max() + np.log(np.exp(x - x.max()).sum()))
    q = np.exp(logq)
    seen = p > 0
    loss = float((p[seen] * (logp[seen] - logq[ids[seen]])).sum())
    listed = np.zeros(V, bool)
    listed[ids] = True
    dense = np.zeros(V)
    np.add.at(dense, ids, p)
    grad, size = q - dense, q + dense
    if lse is not None:
        rest, other = max(0.0, 1.0 - p.sum()), q[~listed].sum()
        if rest > 0:
            with np.errstate(divide="ignore"):
                loss += float(rest * (np.log(rest) - np.log(other)))
        share = rest / other if other > 0 else 0.0
        grad = np.where(listed, grad, q - q * share)
        size = np.where(listed, size, q + q * share)
    return loss, grad * weight / T, size * abs(weight) / T
