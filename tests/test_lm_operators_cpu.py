"""CPU tests of the language-model operators: the oracles against differences
and known answers, and the refusals of the entry points before any kernel runs."""
import ctypes

import numpy as np
import pytest

from oracle import distill, gated_rec, sample


@pytest.mark.parametrize("cu", [(0, 7, 14), (0, 0, 5, 5, 14), (0, 14)])
def test_recurrence_oracle_gradient_equals_differences(cu):
    """Central differences in float64: truncation ~eps^2 = 1e-10, rounding ~1e-16/eps = 1e-11; 1e-7 bounds both."""
    rng = np.random.default_rng(0)
    n, d, T = len(cu) - 1, 3, cu[-1]
    v = [rng.standard_normal((T, d)) for _ in range(3)] + [rng.standard_normal(d), rng.standard_normal((n, d))]
    dy, dh = rng.standard_normal((T, d)), rng.standard_normal((n, d))

    def loss(w):
        y, h = gated_rec.fwd(*w, cu)
        return (y * dy).sum() + (h * dh).sum()

    grads = gated_rec.bwd(*v, cu, dy, dh)
    for k, g in enumerate(grads):
        for at in np.ndindex(g.shape):
            up, down = [w.copy() for w in v], [w.copy() for w in v]
            up[k][at] += 1e-5
            down[k][at] -= 1e-5
            assert abs((loss(up) - loss(down)) / 2e-5 - g[at]) < 1e-7


def test_recurrence_oracle_known_answers():
    """Gates far open and closed: r = -inf keeps the state, a huge decay drops it and takes x sigmoid(i)."""
    inf = np.full((2, 1), np.inf)
    y, h = gated_rec.fwd(np.ones((2, 1)), -inf, inf, np.zeros(1), np.full((1, 1), 3.0), (0, 2))
    assert (y == 3.0).all() and h[0, 0] == 3.0
    y, _ = gated_rec.fwd(np.full((2, 1), 2.0), inf, np.zeros((2, 1)), np.full(1, 1000.0), np.full((1, 1), 3.0), (0, 2))
    assert np.allclose(y, 1.0)


def test_distill_oracle_gradient_equals_differences():
    rng = np.random.default_rng(1)
    z, q = rng.standard_normal((4, 9)), rng.standard_normal((4, 3))
    ids = np.array([[0, 4, 8], [2, -1, 3], [5, 5, 1], [-1, 9, 40]])
    w, up = rng.random(4), rng.standard_normal(4)
    _, g = distill.loss_and_grad(z, q, ids, w, 1.7, up)
    f = lambda zz: (distill.loss_and_grad(zz, q, ids, w, 1.7)[0] * up).sum()
    for at in np.ndindex(z.shape):
        a, b = z.copy(), z.copy()
        a[at] += 1e-5
        b[at] -= 1e-5
        assert abs((f(a) - f(b)) / 2e-5 - g[at]) < 1e-8
    assert (g[3] == 0).all()


def test_distill_oracle_zero_at_the_teacher():
    """A student equal to the teacher on all tokens has loss 0 and gradient 0."""
    z = np.random.default_rng(2).standard_normal((3, 5))
    loss, g = distill.loss_and_grad(z, z, np.tile(np.arange(5), (3, 1)), None, 2.0)
    assert np.abs(loss).max() < 1e-14 and np.abs(g).max() < 1e-15


def test_sample_oracle_known_answers():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    assert sample.token(x, 0.05) == (0, pytest.approx(np.log(0.1)))
    assert sample.token(x, 0.49)[0] == 1 and sample.token(x, 0.51)[0] == 2 and sample.token(x, 0.99)[0] == 3
    assert list(sample.kept(x, top_k=2)[0]) == [1, 3]
    assert list(sample.kept(x, top_p=0.5)[0]) == [1, 3] and list(sample.kept(x, top_p=0.3)[0]) == [1]
    assert list(sample.kept(x, min_p=0.6)[0]) == [1, 3]
    assert list(sample.kept(np.zeros(5), top_k=2)[0]) == [0, 1]
    assert sample.token(np.full(3, -np.inf), 0.5) == (-1, -np.inf)
    assert sample.token(x, 0.9, temperature=0.0) == (1, 0.0)


def test_refusals_without_gpu():
    """The shim rejects CPU tensors, the C entry points bad arguments with BCM_ERR_INVALID_ARGUMENT (1) and a reason."""
    import torch

    import bc_mamba_b200
    from bc_mamba_b200 import interface as itf

    x = torch.zeros(1, 2, 3)
    with pytest.raises(RuntimeError, match="x must be on CUDA"):
        itf.gated_recurrence(x, x, x, torch.zeros(3))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        itf.gated_recurrence_step(x[0], x[0], x[0], torch.zeros(3), torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        itf.distill_topk(x[0], x[0], torch.zeros(2, 3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        itf.sample_tokens(x[0], torch.zeros(2))
    lib = bc_mamba_b200.load_library()
    lib.bcm_last_error.restype = ctypes.c_char_p
    for name in ("bcm_gated_rec_fwd", "bcm_gated_rec_bwd", "bcm_distill_fwd", "bcm_distill_bwd", "bcm_distill_fwd_grad", "bcm_sample_tokens"):
        f = getattr(lib, name)
        f.restype, f.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]
        assert f(None, None) == 1 and b"null arguments" in lib.bcm_last_error(), name
    f = lib.bcm_gated_rec_step
    f.restype = ctypes.c_int
    P, I = ctypes.c_void_p, ctypes.c_int64
    f.argtypes = [P, I, P, I, P, I, ctypes.c_int, I, I, P, ctypes.c_float, P, P, P]
    assert f(None, 0, None, 0, None, 0, 0, 2, 4, None, 8.0, None, None, None) == 1 and b"null pointer" in lib.bcm_last_error()
    assert f(None, 0, None, 0, None, 0, 3, 2, 4, None, 8.0, None, None, None) == 1 and b"unsupported dtype" in lib.bcm_last_error()
    # BCM_F64 (3) and a size of zero features, through the argument block
    block = (ctypes.c_int64 * 64)()
    block[0], block[1], block[2] = 1, 1, 0
    lib.bcm_gated_rec_fwd(ctypes.byref(block), None)
    assert b"bad sizes" in lib.bcm_last_error()
    # no sequence: nothing to do, and the error text is cleared
    assert lib.bcm_gated_rec_step(None, 0, None, 0, None, 0, 0, 0, 4, None, 8.0, None, None, None) == 0
    assert lib.bcm_last_error() == b""
