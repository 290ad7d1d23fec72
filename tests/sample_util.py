"""What ops.sample_tokens computes, in 64 bits, row by row from its definition."""
import math

import numpy as np


def allowed(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Indices that stay, in their order, and their weights; x: a row of float64."""
    order = np.lexsort((np.arange(len(x)), -x))                  # logit downwards, index upwards
    order = order[x[order] > -math.inf]
    if not temperature > 0:
        return order[:1], np.ones(1)
    with np.errstate(over="ignore"):
        w = np.exp((x[order] - x[order[0]]) / float(np.float32(temperature)))
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    n = len(order)
    top_p, min_p = float(np.float32(top_p)), float(np.float32(min_p))
    if top_p < 1:
        sums = np.cumsum(w)
        n = 1 if top_p <= 0 else min(n, int(np.searchsorted(sums, top_p * sums[-1])) + 1)
    n = min(n, max(1, int((w >= min(min_p, 1.0)).sum())))
    keep = np.sort(order[:n])
    back = np.argsort(order[:n])
    return keep, w[:n][back]


def sample(x, u, **how):
    """(token, log of its share) of one row."""
    if np.isnan(x).any() or (x == math.inf).any():
        return -1, math.nan
    if not (x > -math.inf).any():
        return -1, -math.inf
    keep, w = allowed(x, **how)
    some = w >= math.exp(-690)                                   # less is as good as excluded
    keep, w = keep[some], w[some]
    sums = np.cumsum(w)
    goal = float(np.float32(u)) * sums[-1] if u > 0 else 0.0
    at = min(int(np.searchsorted(sums, goal, side="right")), len(keep) - 1)
    return int(keep[at]), math.log(w[at] / sums[-1])
