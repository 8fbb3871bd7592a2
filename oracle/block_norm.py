"""The norms of a linear-attention block in float64: the gated norm by groups of features and the residual addition
with its norm, each with its gradients.  Rows (T, D)."""
from __future__ import annotations

import numpy as np


def _norm(x, eps):
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return x * r, r


def _norm_back(x, r, dn):
    return r * (dn - x * r * r * (dn * x).mean(-1, keepdims=True))


def gated(x, gate, weight, groups, eps, dout=None):
    """-> out; with dout (out, dx, dgate, dweight)"""
    x, gate, weight = (np.asarray(v, np.float64) for v in (x, gate, weight))
    shape = x.shape
    split = lambda v: np.asarray(v, np.float64).reshape(v.shape[:-1] + (groups, -1))
    x, gate, weight = split(x), split(gate), split(weight)
    sig = 1 / (1 + np.exp(-gate))
    n, r = _norm(x, eps)
    out = (n * weight * gate * sig).reshape(shape)
    if dout is None:
        return out
    d = split(np.asarray(dout, np.float64))
    dx = _norm_back(x, r, d * weight * gate * sig)
    dz = d * n * weight * sig * (1 + gate * (1 - sig))
    return out, dx.reshape(shape), dz.reshape(shape), (d * n * gate * sig).sum(0).reshape(-1)


def add(residual, branch, weight, scale, eps, dres=None, dout=None):
    """-> (v, normed); with an upstream gradient also (dresidual, dbranch, dweight, dscale)"""
    residual, branch, weight = (np.asarray(v, np.float64) for v in (residual, branch, weight))
    s = 1.0 if scale is None else np.asarray(scale, np.float64)
    v = residual + s * branch
    n, r = _norm(v, eps)
    if dres is None and dout is None:
        return v, n * weight
    d = np.zeros_like(v) if dout is None else np.asarray(dout, np.float64)
    dv = (0.0 if dres is None else np.asarray(dres, np.float64)) + _norm_back(v, r, d * weight)
    return v, n * weight, dv, s * dv, (d * n).sum(0), (dv * branch).sum(0)
