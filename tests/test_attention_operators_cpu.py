"""CPU tests of the linear-attention block's operators: the oracles against differences and known answers, and the
refusals of the entry points before any kernel runs."""
import ctypes

import numpy as np
import pytest

from oracle import block_norm, decay_attn


@pytest.mark.parametrize("cu", [(0, 5, 10), (0, 0, 4, 4, 9), (0, 10)])
def test_attention_oracle_gradient_equals_differences(cu):
    """Central differences in float64: truncation ~eps^2 = 1e-10, rounding ~1e-15/eps = 1e-10; 1e-7 bounds both.  Rows
    behind the last sequence have neither outputs nor gradients."""
    rng = np.random.default_rng(0)
    n, T, H, Hk, N, P = len(cu) - 1, 10, 4, 2, 3, 2
    v = [rng.standard_normal((T, Hk, N)), rng.standard_normal((T, Hk, N)), rng.standard_normal((T, H, P)), -rng.random((T, H)),
         rng.standard_normal((n, H, N, P))]
    dy, dh = rng.standard_normal((T, H, P)), rng.standard_normal((n, H, N, P))

    def loss(w):
        y, h = decay_attn.fwd(*w, cu)
        return (y * dy).sum() + (h * dh).sum()

    grads = decay_attn.bwd(*v, cu, dy, dh)
    for k, g in enumerate(grads):
        if k < 4:
            assert (g[cu[-1]:] == 0).all()
        for at in np.ndindex(g.shape):
            up, down = [w.copy() for w in v], [w.copy() for w in v]
            up[k][at] += 1e-5
            down[k][at] -= 1e-5
            assert abs((loss(up) - loss(down)) / 2e-5 - g[at]) < 1e-7


def test_attention_oracle_known_answers():
    """Without decay a sum of outer products, with a dropped state the token's own alone."""
    q, k, v = np.ones((3, 1, 1)), np.array([1.0, 2, 3]).reshape(3, 1, 1), np.array([1.0, 10, 100]).reshape(3, 1, 1)
    y, h = decay_attn.fwd(q, k, v, np.zeros((3, 1)), np.full((1, 1, 1, 1), 5.0), (0, 3))
    assert y.reshape(-1).tolist() == [6, 26, 326] and h.reshape(-1).tolist() == [326]
    y, _ = decay_attn.fwd(q, k, v, np.full((3, 1), -np.inf), np.full((1, 1, 1, 1), 5.0), (0, 3))
    assert y.reshape(-1).tolist() == [1, 20, 300]


def test_norm_oracles_gradients_equal_differences():
    rng = np.random.default_rng(1)
    x, z, w, d = rng.standard_normal((3, 8)), rng.standard_normal((3, 8)), rng.standard_normal(8), rng.standard_normal((3, 8))
    _, *grads = block_norm.gated(x, z, w, 2, 1e-3, d)
    f = lambda *a: (block_norm.gated(*a, 2, 1e-3) * d).sum()
    r, b, s, dr = rng.standard_normal((3, 8)), rng.standard_normal((3, 8)), rng.standard_normal(8), rng.standard_normal((3, 8))
    grads2 = block_norm.add(r, b, w, s, 1e-3, dr, d)[2:]

    def f2(r, b, w, s):
        v, n = block_norm.add(r, b, w, s, 1e-3)
        return (v * dr).sum() + (n * d).sum()

    for fun, args, gs in ((f, (x, z, w), grads), (f2, (r, b, w, s), grads2)):
        for k, g in enumerate(gs):
            for at in np.ndindex(g.shape):
                up, down = [a.copy() for a in args], [a.copy() for a in args]
                up[k][at] += 1e-5
                down[k][at] -= 1e-5
                assert abs((fun(*up) - fun(*down)) / 2e-5 - g[at]) < 1e-7


class Attn(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("batch", "seqlen", "heads", "qk_heads", "dim_k", "dim_v")] + [
        ("cu_seqlens", ctypes.c_void_p), ("dtype", ctypes.c_int), ("fixed_decay", ctypes.c_int)] + [
        f for t in "qkvg" for f in [(t, ctypes.c_void_p)] + [(f"{t}_stride_{d}", ctypes.c_int64) for d in "bth"]] + [
        ("h0", ctypes.c_void_p), ("y", ctypes.c_void_p), ("h_last", ctypes.c_void_p), ("ckpt", ctypes.c_void_p), ("ckpt_bytes", ctypes.c_size_t),
        ("dy", ctypes.c_void_p)] + [(f"dy_stride_{d}", ctypes.c_int64) for d in "bth"] + [
        (n, ctypes.c_void_p) for n in ("dh_last", "dq", "dk", "dv", "dlog_decay", "dh0", "workspace")] + [("workspace_bytes", ctypes.c_size_t)]


class Gated(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int64), ("dim", ctypes.c_int64), ("groups", ctypes.c_int64), ("dtype", ctypes.c_int), ("eps", ctypes.c_float),
                ("rest", ctypes.c_int64 * 16)]


class Add(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int64), ("dim", ctypes.c_int64), ("dtype", ctypes.c_int), ("residual_dtype", ctypes.c_int), ("eps", ctypes.c_float),
                ("rest", ctypes.c_int64 * 24)]


def _call(name, args, *more):
    import bc_mamba_b200

    lib = bc_mamba_b200.load_library()
    lib.bcm_last_error.restype = ctypes.c_char_p
    f = getattr(lib, name)
    f.restype = ctypes.c_int
    f.argtypes = [ctypes.c_void_p] * (2 + len(more))
    return f(None if args is None else ctypes.byref(args), *more, None), lib.bcm_last_error()


@pytest.mark.parametrize("name,more", [("bcm_decay_attn_fwd", ()), ("bcm_decay_attn_bwd", ()), ("bcm_decay_attn_step", (None,))])
def test_attention_refusals(name, more):
    ok = dict(batch=0, seqlen=1, heads=4, qk_heads=2, dim_k=8, dim_v=8)
    assert _call(name, None, *more) == (1, f"{name[4:]}: null arguments".encode())
    for bad, why in [(dict(dim_k=129), b"more than 128"), (dict(heads=3), b"multiple"), (dict(dim_v=0), b"bad sizes"), (dict(heads=0), b"bad sizes"),
                     (dict(batch=-1), b"bad sizes"), (dict(dtype=3), b"unsupported dtype"), (dict(batch=1), b"null pointer"),
                     (dict(heads=1 << 20, qk_heads=1, dim_v=1 << 20), b"too large"), (dict(cu_seqlens=256), b"no sequence")]:
        status, text = _call(name, Attn(**{**ok, **bad}), *more)
        assert status == 1 and why in text, (bad, text)
    assert _call(name, Attn(**ok), *more) == (0, b"")


def test_attention_workspaces_do_not_need_a_device_call_to_be_sized():
    import bc_mamba_b200

    lib = bc_mamba_b200.load_library()
    for f in (lib.bcm_decay_attn_ckpt_bytes, lib.bcm_decay_attn_fwd_workspace_bytes, lib.bcm_decay_attn_bwd_workspace_bytes):
        f.restype, f.argtypes = ctypes.c_size_t, [ctypes.c_void_p]
    a = Attn(batch=2, seqlen=130, heads=4, qk_heads=2, dim_k=16, dim_v=64)
    # three chunks a sequence, states of 64 x 16
    assert lib.bcm_decay_attn_ckpt_bytes(ctypes.byref(a)) == 2 * 3 * 4 * 64 * 16 * 4
    # two heads to a query: two parts of dq and of dk
    assert lib.bcm_decay_attn_bwd_workspace_bytes(ctypes.byref(a)) >= 2 * 2 * 2 * 130 * 2 * 16 * 4
    assert lib.bcm_decay_attn_fwd_workspace_bytes(None) == 0


@pytest.mark.parametrize("name", ["bcm_gated_norm_fwd", "bcm_gated_norm_bwd"])
def test_gated_norm_refusals(name):
    ok = dict(rows=0, dim=8, groups=2, eps=1e-6)
    assert _call(name, None)[0] == 1
    for bad, why in [(dict(groups=3), b"bad sizes"), (dict(groups=0), b"bad sizes"), (dict(eps=0.0), b"eps"), (dict(eps=float("nan")), b"eps"),
                     (dict(eps=float("inf")), b"eps"), (dict(dim=8193, groups=1), b"more than 8192"), (dict(dtype=3), b"unsupported dtype"),
                     (dict(rows=1), b"null pointer")]:
        status, text = _call(name, Gated(**{**ok, **bad}))
        assert status == 1 and why in text, (bad, text)
    assert _call("bcm_gated_norm_fwd", Gated(**ok)) == (0, b"")


@pytest.mark.parametrize("name", ["bcm_add_norm_fwd", "bcm_add_norm_bwd"])
def test_add_norm_refusals(name):
    ok = dict(rows=0, dim=8, eps=1e-6)
    assert _call(name, None)[0] == 1
    for bad, why in [(dict(dim=0), b"bad sizes"), (dict(eps=-1.0), b"eps"), (dict(dim=8193), b"more than 8192"), (dict(dtype=1, residual_dtype=2), b"residual"),
                     (dict(rows=1), b"null pointer")]:
        status, text = _call(name, Add(**{**ok, **bad}))
        assert status == 1 and why in text, (bad, text)
    assert _call("bcm_add_norm_fwd", Add(**ok)) == (0, b"")


def test_cpu_tensors_are_refused():
    import torch

    from bc_mamba_b200 import interface as itf

    x = torch.zeros(1, 2, 3, 4)
    with pytest.raises(RuntimeError, match="v must be on CUDA"):
        itf.decay_attention(x, x, x, torch.zeros(3))
    with pytest.raises(RuntimeError, match="v must be on CUDA"):
        itf.decay_attention_step(x[0], x[0], x[0], torch.zeros(3), torch.zeros(2, 3, 4, 4))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        itf.gated_norm(x, x, torch.ones(4))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        itf.add_norm(x, x, torch.ones(4))
