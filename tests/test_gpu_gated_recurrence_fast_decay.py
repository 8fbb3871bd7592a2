"""Gated recurrence with decays far below one: every output that is
proportional to a decay keeps its relative accuracy, element by element,
however small the decay is.

Tolerance (derived): in fp32 the exponent U = c softplus(lam) sigmoid(r)
carries a relative error of a few 2^-23 (log1p, exp, two reciprocals), hence
a = e^-U one of U 2^-21, and 1 - sigmoid(r) one of 2^-22 / (1 - sigmoid(r));
exponentials, reciprocals and products add a constant of a few 2^-22, and the
neighbours' decays enter with U e^-U <= 0.4 of theirs.  So every element is
within 2^-20 (16 + U + 1 / (1 - sigmoid(r))) of the sum of its terms'
magnitudes, and 16-bit ones within 2^-8 (bf16) of it."""
import numpy as np
import pytest
import torch

from bc_mamba_b200 import interface as itf
from oracle import gated_rec as orc

pytestmark = pytest.mark.gpu
dev = "cuda"
C = 8.0


def _inputs(rows, d, n, lam, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    t = dict(x=rn(rows, d), r=1.5 + rn(rows, d), i=rn(rows, d), dy=rn(rows, d))
    t = {k: v.to(dtype).to(dev) for k, v in t.items()}
    t["lam"] = (lam + 0.1 * rn(d)).to(dev)
    t["h0"], t["dh"] = rn(n, d).to(dev), rn(n, d).to(dev)
    return t


def _np(t):
    return t.detach().double().cpu().numpy()


def _magnitudes(v, cu):
    """Per output the sum of its terms' magnitudes, and the tolerance's factor of each token."""
    x, r, i, dy, lam, h0, dh = v
    soft, sr, si = np.logaddexp(0.0, lam), 1 / (1 + np.exp(-r)), 1 / (1 + np.exp(-i))
    U = C * soft * sr
    a, m = np.exp(-U), np.sqrt(-np.expm1(-2 * U))
    b = m * si * np.abs(x)
    h, G = np.zeros_like(x), np.zeros_like(x)
    prev, m0 = np.zeros_like(x), np.zeros_like(h0)
    for s in range(len(cu) - 1):
        now = np.abs(h0[s])
        for t in range(cu[s], cu[s + 1]):
            prev[t] = now
            now = a[t] * now + b[t]
            h[t] = now
        back = np.abs(dh[s])
        for t in range(cu[s + 1] - 1, cu[s] - 1, -1):
            G[t] = np.abs(dy[t]) + back
            back = a[t] * G[t]
        m0[s] = back
    du = G * a * (prev + a / m * si * np.abs(x))
    wide = 2.0 ** -20 * (16 + U + 1 / (1 - sr))
    dr = du * U * (1 - sr)
    first = np.array([wide[cu[s]] if cu[s] < cu[s + 1] else np.zeros_like(lam) for s in range(len(cu) - 1)])
    dlam = (C / (1 + np.exp(-lam)) * du * sr * wide).sum(0)
    return dr * wide, dlam, m0 * first, h * wide


PLANS = [("serial", (1800, 5, 10)), ("grouped", (40, 7, 66)), ("dense", (2, 300, 66)), ("segments", (1, 9000, 6)),
         ("packed", (0, 7, 7, 200, 300)), ("packed runs", tuple(range(0, 5001, 50))), ("packed segments", (0, 6000, 12288, 20000))]


@pytest.mark.parametrize("lam", [2.0, 4.0, 6.0])
@pytest.mark.parametrize("name,shape", PLANS)
def test_gradients_keep_small_decays(name, shape, lam):
    packed = name.startswith("packed")
    d = 5 if packed else shape[2]
    cu = shape if packed else range(0, shape[0] * shape[1] + 1, shape[1])
    cu = [int(v) for v in cu]
    n = len(cu) - 1
    t = _inputs(cu[-1], d, n, lam, torch.float32, seed=n)
    view = (lambda v: v) if packed else (lambda v: v.reshape(shape[0], shape[1], d))
    leaves = {k: (view(t[k]) if k in "xri" else t[k]).clone().requires_grad_(True) for k in ("x", "r", "i", "lam", "h0")}
    y, h = itf.gated_recurrence(*(leaves[k] for k in ("x", "r", "i", "lam")), h0=leaves["h0"],
                                cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev) if packed else None)
    grads = torch.autograd.grad([y, h], [leaves[k] for k in ("r", "lam", "h0")], [view(t["dy"]), t["dh"]])
    v = [_np(t[k]) for k in ("x", "r", "i", "dy", "lam", "h0", "dh")]
    _, dr, _, dlam, dh0 = orc.bwd(v[0], v[1], v[2], v[4], v[5], cu, v[3], v[6])
    lims = _magnitudes(v, cu)
    for what, got, want, lim in zip(("dr", "dlam", "dh0"), grads, (dr, dlam, dh0), lims):
        err = np.abs(_np(got).reshape(want.shape) - want)
        assert (err <= lim).all(), f"{what}: {np.max(err / np.maximum(lim, 1e-300)):.3g} times the bound"


@pytest.mark.parametrize("lam", [2.0, 4.0, 6.0])
def test_states_keep_small_decays(lam):
    """Without inputs the state is a product of decays: by the scan and by the step."""
    t = _inputs(2 * 2, 33, 2, lam, torch.float32, seed=3)
    v = [_np(t[k]) for k in ("x", "r", "i", "dy", "lam", "h0", "dh")]
    v[0] = np.zeros_like(v[0])
    want, _ = orc.fwd(*v[:3], v[4], v[5], (0, 2, 4))
    U = C * np.logaddexp(0.0, v[4]) / (1 + np.exp(-v[1]))
    U = U.reshape(2, 2, 33).cumsum(1).reshape(4, 33)
    lim = 2.0 ** -20 * (16 + U) * np.abs(want)
    x, r, i = (t[k].reshape(2, 2, 33) for k in ("x", "r", "i"))
    y, _ = itf.gated_recurrence(torch.zeros_like(x), r, i, t["lam"], h0=t["h0"])
    assert (np.abs(_np(y).reshape(4, 33) - want) <= lim).all()
    h = t["h0"].clone()
    steps = torch.stack([itf.gated_recurrence_step(torch.zeros_like(x[:, 0]), r[:, k], i[:, k], t["lam"], h) for k in range(2)], 1)
    assert (np.abs(_np(steps).reshape(4, 33) - want) <= lim).all()


def test_bf16_gradients_of_tiny_decays_are_not_zero():
    t = _inputs(200, 40, 1, 6.0, torch.bfloat16, seed=5)
    r = (t["r"].float().abs() + 1).to(torch.bfloat16)                 # every U above 34: a below 2^-24
    leaf = r[None].clone().requires_grad_(True)
    y, _ = itf.gated_recurrence(t["x"][None], leaf, t["i"][None], t["lam"], h0=t["h0"])
    g, = torch.autograd.grad(y, leaf, t["dy"][None])
    v = [_np(t["x"]), _np(r), _np(t["i"]), _np(t["dy"]), _np(t["lam"]), _np(t["h0"]), np.zeros((1, 40))]
    _, want, _, _, _ = orc.bwd(v[0], v[1], v[2], v[4], v[5], (0, 200), v[3], None)
    lim = _magnitudes(v, (0, 200))[0] + 2.0 ** -8 * np.abs(want)
    assert np.abs(want).min() > 0 and (np.abs(_np(g)[0] - want) <= lim).all()
