"""Linear attention with a decay for each head in float64, token by token, with its adjoint.

Per head, a_t = exp(g_t): S_t = a_t S_(t-1) + k_t v_t^T, y_t = S_t^T q_t.  q, k (T, Hk, N), v (T, H, P), g (T, H); head h
reads query and key h // (H / Hk).  Sequences are given by offsets ``cu`` (dense inputs: multiples of L); rows outside
them have y and gradients 0.
"""
from __future__ import annotations

import numpy as np


def _wide(x, heads):
    x = np.asarray(x, np.float64)
    return np.repeat(x, heads // x.shape[1], axis=1)


def fwd(q, k, v, g, h0, cu, keep=False):
    """-> (y (T, H, P), h_last (n, H, N, P)); with keep also the state before every token"""
    v, g = np.asarray(v, np.float64), np.asarray(g, np.float64)
    heads = v.shape[1]
    q, k = _wide(q, heads), _wide(k, heads)
    n = len(cu) - 1
    y = np.zeros_like(v)
    last = np.zeros((n, heads, q.shape[2], v.shape[2]))
    states = np.zeros((v.shape[0],) + last.shape[1:]) if keep else None
    for s in range(n):
        h = np.zeros(last.shape[1:]) if h0 is None else np.asarray(h0[s], np.float64)
        for t in range(cu[s], cu[s + 1]):
            if keep:
                states[t] = h
            h = np.exp(g[t])[:, None, None] * h + k[t][:, :, None] * v[t][:, None, :]
            y[t] = np.einsum("hnp,hn->hp", h, q[t])
        last[s] = h
    return (y, last, states) if keep else (y, last)


def bwd(q, k, v, g, h0, cu, dy, dh):
    """-> (dq, dk (T, Hk, N), dv (T, H, P), dg (T, H), dh0 (n, H, N, P))"""
    shared = np.asarray(q).shape
    _, last, states = fwd(q, k, v, g, h0, cu, keep=True)
    v, g = np.asarray(v, np.float64), np.asarray(g, np.float64)
    heads = v.shape[1]
    q, k = _wide(q, heads), _wide(k, heads)
    dq, dk, dv, dg = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v), np.zeros_like(g)
    dh0 = np.zeros_like(last)
    for s in range(len(cu) - 1):
        ds = np.zeros(last.shape[1:]) if dh is None else np.asarray(dh[s], np.float64)
        for t in range(cu[s + 1] - 1, cu[s] - 1, -1):
            a = np.exp(g[t])[:, None, None]
            up = np.zeros_like(v[t]) if dy is None else np.asarray(dy[t], np.float64)
            now = a * states[t] + k[t][:, :, None] * v[t][:, None, :]
            ds = ds + q[t][:, :, None] * up[:, None, :]
            dq[t] = np.einsum("hnp,hp->hn", now, up)
            dk[t] = np.einsum("hnp,hp->hn", ds, v[t])
            dv[t] = np.einsum("hnp,hn->hp", ds, k[t])
            dg[t] = (a * ds * states[t]).sum((1, 2))
            ds = a * ds
        dh0[s] = ds
    split = lambda x: x.reshape(shared[0], shared[1], -1, shared[2]).sum(2)
    return split(dq), split(dk), dv, dg, dh0
