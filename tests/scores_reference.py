"""Draws from rows of scores and the loss against a teacher's top entries in 64 bits, from their definitions.  Nothing here uses
the library."""
import numpy as np


def kept_weights(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Weights of a row's columns after all cuts, 0 for those that are cut off or not there."""
    x = np.asarray(x, dtype=np.float64)
    out = np.zeros(len(x))
    there = np.flatnonzero(x > -np.inf)          # NaN is not
    if len(there) == 0:
        return out
    order = there[np.argsort(-x[there], kind="stable")]
    best = x[order[0]]
    if not temperature > 0:
        temperature, top_k = 1.0, 1
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        w = np.where(x[order] == best, 1.0, np.exp((x[order] - best) / np.float64(temperature)))
    w = np.where(w > 2.0 ** -960, w, 0.0)        # what is below counts as nothing; so does no number
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    if top_p < 1:
        n = int(np.count_nonzero(np.cumsum(w) < np.float64(top_p) * w.sum())) + 1
        order, w = order[:max(1, n)], w[:max(1, n)]
    if min_p > 0:
        keep = w >= min(np.float64(min_p), 1.0)
        order, w = order[keep], w[keep]
    out[order] = w
    return out


def drawn(w, u, label, prob, slack):
    """Whether a label and its probability are those of the random number u, but for `slack` of the total next to a border."""
    total = w.sum()
    if total == 0:
        return label == -1 and prob == 0
    if not 0 <= label < len(w) or w[label] == 0:
        return False
    run = np.cumsum(w)
    target = min(max(float(u), 0.0), 1 - 2.0 ** -24) * total
    near = slack * total
    return bool(run[label] > target - near and run[label] - w[label] <= target + near and
                abs(prob - w[label] / total) <= 2.0 ** -23 * w[label] / total + 2.0 ** -149)


def distil(x, labels, teacher, temperature, whole=None):
    """(loss, gradient per unit of weight) of one row."""
    x, teacher, T = np.asarray(x, dtype=np.float64), np.asarray(teacher, dtype=np.float64), float(temperature)
    n = len(x)
    there = (labels >= 0) & (labels < n)
    l, t = labels[there], teacher[there] / T
    gradient = np.zeros(n)
    if np.isnan(x).any() or (x == np.inf).any():
        return np.nan, np.full(n, np.nan)
    if len(l) == 0 or not (x > -np.inf).any():
        return 0.0, gradient
    if whole is None:
        top = t.max()
        if top == -np.inf:
            return 0.0, gradient
        lse = top + np.log(np.exp(t - top).sum())
    else:
        lse = float(whole)
    log_p = t - lse
    p = np.exp(log_p)
    e = np.exp((x - x.max()) / T)
    with np.errstate(divide="ignore"):
        log_q = (x - x.max()) / T - np.log(e.sum())
    use = p > 0
    loss = T * T * float((p[use] * (log_p[use] - log_q[l[use]])).sum())
    gradient = T * p.sum() * e / e.sum()
    np.subtract.at(gradient, l, T * p)
    return loss, gradient
