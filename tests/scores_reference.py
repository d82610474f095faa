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
    w = np.nan_to_num(w)
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
