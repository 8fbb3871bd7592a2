"""Distillation loss on a teacher's top logits and its gradient, float64, row by row."""
from __future__ import annotations

import numpy as np


def _softmax(v, tau):
    """softmax(v / tau) and its logarithm, from differences to the maximum."""
    d = (v - v.max()) / tau
    return np.exp(d) / np.exp(d).sum(), d - np.log(np.exp(d).sum())


def loss_and_grad(z, q, ids, weight=None, tau=1.0, dloss=None):
    """z (T, V), q and ids (T, K) -> (loss (T,), dz (T, V))"""
    z, q = np.asarray(z, np.float64), np.asarray(q, np.float64)
    T, V = z.shape
    loss, dz = np.zeros(T), np.zeros((T, V))
    for t in range(T):
        w = 1.0 if weight is None else float(weight[t])
        at = [k for k in range(q.shape[1]) if 0 <= ids[t, k] < V and q[t, k] != -np.inf]
        if w == 0 or not at:
            continue
        p, logp = _softmax(q[t, at], tau)
        s, logs = _softmax(z[t], tau)
        g = s.copy()
        for pk, lk, k in zip(p, logp, at):
            v = ids[t, k]
            if pk > 0:
                loss[t] += pk * (lk - logs[v])
            g[v] -= pk
        loss[t] *= w * tau * tau
        dz[t] = (1.0 if dloss is None else float(dloss[t])) * w * tau * g
    return loss, dz
