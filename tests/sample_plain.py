"""pa_sample's definition on the host, in 64 bits (numpy)."""
import math

import numpy as np


def weights(x, t):
    """Weights of one f64 row without NaN (they are -inf)."""
    top = x.max()
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((x - top) / t)
    w = np.where(x == -np.inf, 0.0, w)
    return np.where(x == top, 1.0, w)


def kept(x, t, k, p, m):
    """Kept columns, ascending, and their weights."""
    w = weights(x, t)
    order = np.argsort(-x, kind="stable")
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        sums = np.cumsum(w[order])
        order = order[:max(1, int(np.searchsorted(sums, p * sums[-1], "left")) + 1)]
    if m > 0:
        keep = w[order] >= m
        keep[0] = True
        order = order[keep]
    order = np.sort(order)
    return order, w[order]


def draw(x, u, t=1.0, k=0, p=1.0, m=0.0):
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    if x.max() == -np.inf:
        return 0
    if not t > 0:
        return int(np.argmax(x))
    order, w = kept(x, t, k, p, m)
    order, w = order[w > 0], w[w > 0]
    u = 0.0 if not u > 0 else u
    sums = np.cumsum(w)
    return int(order[min(len(order) - 1, int(np.searchsorted(sums, u * sums[-1], "right")))])


def margin(x, u, t, k, p, m):
    """How far the draw is from another one, relative to the total weight (the
    distance of u from the next border between two kept tokens, and of p from one
    between two that top-p parts), and the total weight."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    if x.max() == -np.inf or not t > 0:
        return 1.0, 1.0
    order, w = kept(x, t, k, p, m)
    sums = np.cumsum(w) / w.sum()
    got = np.abs(sums[:-1] - u).min() if len(sums) > 1 else 1.0
    if p < 1:
        full = weights(x, t)
        desc = np.argsort(-x, kind="stable")
        desc = desc[:k] if 0 < k < len(x) else desc
        c = np.cumsum(full[desc]) / full[desc].sum()
        got = min(got, np.abs(c - p).min())
    return got, w.sum()
