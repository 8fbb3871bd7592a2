"""Token sampling with temperature, top-k, top-p and min-p, float64, one row at a time."""
from __future__ import annotations

import numpy as np


def kept(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(indices of the kept tokens, ascending; their probabilities) of one row."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    if x.max() == -np.inf:
        return np.zeros(0, np.int64), np.zeros(0)
    if not temperature > 0:
        return np.array([int(x.argmax())]), np.ones(1)
    e = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / temperature))
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        mass = e[order]
        before = np.cumsum(mass) - mass
        order = order[:max(1, int((before < top_p * mass.sum()).sum()))]
    order = np.sort(order[e[order] >= min(min_p, 1.0)])
    return order, e[order] / e[order].sum()


def token(x, u, **settings):
    """(token, log-probability); (-1, -inf) where nothing can be taken."""
    at, p = kept(x, **settings)
    if not len(at):
        return -1, -np.inf
    j = min(int((np.cumsum(p) <= u).sum()), len(at) - 1)
    return int(at[j]), float(np.log(p[j]))
