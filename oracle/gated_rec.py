"""Gated linear recurrence in float64, token by token, with its adjoint.

Per feature: u = -c softplus(lam) sigmoid(r), a = exp(u), m = sqrt(1 - a^2),
h_t = a_t h_(t-1) + m_t sigmoid(i_t) x_t.  Sequences are given by offsets
``cu`` into (T, D) arrays (dense inputs: cu = multiples of L).
"""
from __future__ import annotations

import numpy as np


def _sigmoid(v):
    e = np.exp(-np.abs(v))
    return np.where(v >= 0, 1 / (1 + e), e / (1 + e))


def _parts(x, r, i, lam, c):
    x, r, i, lam = (np.asarray(v, np.float64) for v in (x, r, i, lam))
    soft = np.logaddexp(0.0, lam)
    sr, si = _sigmoid(r), _sigmoid(i)
    u = -c * soft * sr
    return x, sr, si, u, np.exp(u), np.sqrt(-np.expm1(2 * u)), lam


def fwd(x, r, i, lam, h0, cu, c=8.0):
    """-> (y (T, D), h_last (n, D))"""
    x, sr, si, u, a, m, lam = _parts(x, r, i, lam, c)
    n, d = len(cu) - 1, x.shape[1]
    y = np.zeros_like(x)
    h_last = np.zeros((n, d))
    for s in range(n):
        h = np.zeros(d) if h0 is None else np.asarray(h0[s], np.float64)
        for t in range(cu[s], cu[s + 1]):
            h = a[t] * h + m[t] * si[t] * x[t]
            y[t] = h
        h_last[s] = h
    return y, h_last


def bwd(x, r, i, lam, h0, cu, dy, dh_last, c=8.0):
    """-> (dx, dr, di (T, D), dlam (D,), dh0 (n, D))"""
    y, _ = fwd(x, r, i, lam, h0, cu, c)
    x, sr, si, u, a, m, lam = _parts(x, r, i, lam, c)
    n, d = len(cu) - 1, x.shape[1]
    G, prev = np.zeros_like(x), np.zeros_like(x)
    dh0 = np.zeros((n, d))
    for s in range(n):
        back = np.zeros(d) if dh_last is None else np.asarray(dh_last[s], np.float64)
        for t in range(cu[s + 1] - 1, cu[s] - 1, -1):
            G[t] = back + (0 if dy is None else np.asarray(dy[t], np.float64))
            back = a[t] * G[t]
            prev[t] = y[t - 1] if t > cu[s] else (0 if h0 is None else h0[s])
        dh0[s] = back
    dx = G * m * si
    di = dx * x * (1 - si)
    slope = np.divide(a * a, m, out=np.zeros_like(m), where=m != 0)
    du = G * (a * prev - slope * si * x)
    return dx, du * u * (1 - sr), di, -c * _sigmoid(lam) * (du * sr).sum(0), dh0
