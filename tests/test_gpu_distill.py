"""GPU parity of the distillation loss on a teacher's top logits, and of its
gradient (autograd pair and one-call form), against the float64 oracle.

Tolerances (derived): the fp32 softmax carries an exponential of relative error
2^-22 + |z/tau| 2^-24 and sums in fixed trees, 1e-5 of the largest entry; the
loss adds terms of both signs of size |ln p| <= 30, 1e-5 of max(1, loss);
16-bit gradients are rounded once, half an ulp doubled, plus the type's
smallest subnormal."""
import math

import numpy as np
import pytest
import torch

from bc_mamba_b200 import interface as itf
from helpers import assert_close, assert_exact
from oracle import distill as orc

pytestmark = pytest.mark.gpu
dev = "cuda"
TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11 + 1e-5}


def _inputs(T, V, K, dtype, seed, qdtype=torch.float32, idtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    z = (3 * torch.randn(T, V, generator=g)).to(dtype).to(dev)
    ids = torch.rand(T, V, generator=g).topk(K, 1)[1].to(idtype).to(dev)
    q = (3 * torch.randn(T, K, generator=g)).to(qdtype).to(dev)
    return z, q, ids, (0.2 + torch.rand(T, generator=g)).to(dev), (torch.rand(T, generator=g) - 0.3).to(dev)


def _np(t):
    return t.detach().double().cpu().numpy()


def _check(z, q, ids, w, tau, up):
    args = (_np(z), _np(q), ids.cpu().numpy(), None if w is None else _np(w), tau)
    loss, dz = orc.loss_and_grad(*args, dloss=_np(up))
    _, dz1 = orc.loss_and_grad(*args)
    leaf = z.detach().clone().requires_grad_(True)
    got = itf.distill_topk(leaf, q, ids, weight=w, temperature=tau)
    lim = 1e-5 * np.maximum(1.0, np.abs(loss)) * (1 if w is None else max(1.0, float(w.max()))) * tau * tau
    assert got.dtype == torch.float32 and (np.abs(_np(got) - loss) <= lim).all()
    g, = torch.autograd.grad(got, leaf, up)
    assert g.dtype == z.dtype
    tol = TOL[z.dtype]
    tiny = 2.0 ** -24 if z.dtype == torch.float16 else 0.0

    def near(a, b):
        a = _np(a)
        assert (np.abs(a - b) <= tol * np.abs(b) + 1e-5 * np.abs(b).max() + tiny).all(), np.abs(a - b).max()

    near(g, dz)
    one, g1 = itf.distill_topk_with_grad(z, q, ids, weight=w, temperature=tau)
    assert_close(one, _np(got), 1e-6, "loss of the one-call form")
    near(g1, dz1)


@pytest.mark.parametrize("T,V,K", [(1, 1, 1), (3, 7, 2), (5, 256, 8), (2, 1023, 33), (4, 4099, 64), (2, 33001, 200), (1, 150001, 16),
                                   (3, 2048, 1024), (300, 129, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_loss_and_gradient(T, V, K, dtype):
    z, q, ids, w, up = _inputs(T, V, K, dtype, seed=T + V + K)
    _check(z, q, ids, w, 1.5, up)


@pytest.mark.parametrize("qdtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("idtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tau", [0.5, 1.0, 4.0])
def test_types_and_temperatures(qdtype, idtype, tau):
    z, q, ids, _, up = _inputs(6, 777, 20, torch.float32, 1, qdtype, idtype)
    _check(z, q, ids, None, tau, up)


def test_absent_entries_duplicates_and_empty_rows():
    z, q, ids, w, up = _inputs(8, 500, 12, torch.float32, seed=2)
    ids[0, 5:] = -1                       # a list that ends early, NaN in its unused places
    q[0, 5:] = math.nan
    ids[1, ::2] = 500                     # outside the vocabulary
    ids[1, 1] = 2 ** 40
    q[2, 3:] = -math.inf                  # masked by value
    ids[3] = ids[3, 0]                    # one token over and over
    ids[4, 4:8] = ids[4, 0:4]
    ids[5] = -1                           # nothing left
    q[6] = -math.inf
    w[7] = 0.0                            # a padding row of NaN
    z[5:8] = math.nan
    clean = z.clone()
    clean[5:8] = 0.0
    _check_rows = slice(0, 5)
    _check(z[_check_rows], q[_check_rows], ids[_check_rows], w[_check_rows], 2.0, up[_check_rows])
    loss, dz = itf.distill_topk_with_grad(z, q, ids, weight=w, temperature=2.0)
    assert_exact(loss[5:], torch.zeros(3), "loss of rows without a target")
    assert_exact(dz[5:], torch.zeros(3, 500), "gradient of rows without a target")
    leaf = z.clone().requires_grad_(True)
    g, = torch.autograd.grad(itf.distill_topk(leaf, q, ids, weight=w).sum(), leaf)
    assert_exact(g[5:], torch.zeros(3, 500), "autograd gradient of rows without a target")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_vocabulary(dtype):
    """Logits of -inf and of the type's lowest value take no mass and no gradient; one of them as a target
    makes the loss infinite, as the formula does."""
    z, q, ids, w, up = _inputs(4, 3001, 6, dtype, seed=3)
    mask = torch.rand(4, 3001, generator=torch.Generator().manual_seed(1)).to(dev) < 0.6
    mask.scatter_(1, ids, False)
    z[:2].masked_fill_(mask[:2], -math.inf)
    z[2:].masked_fill_(mask[2:], torch.finfo(dtype).min)
    _check(z, q, ids, w, 1.0, up)
    z[0, ids[0, 0]] = -math.inf
    loss, dz = itf.distill_topk_with_grad(z, q, ids)
    assert loss[0] == math.inf and torch.isfinite(loss[1:]).all() and torch.isfinite(dz).all()


def test_nan_and_spread():
    z, q, ids, w, up = _inputs(3, 900, 4, torch.float32, seed=4)
    z[1, 17] = math.nan
    loss, dz = itf.distill_topk_with_grad(z, q, ids)
    assert torch.isnan(loss[1]) and torch.isnan(dz[1]).all() and torch.isfinite(dz[[0, 2]]).all()
    z, q, ids, w, up = _inputs(3, 900, 4, torch.float32, seed=5)
    _check(z * 300, q * 30, ids, w, 1.0, up)          # exponentials far below the smallest float


def test_row_strides():
    z, q, ids, w, up = _inputs(5, 700, 9, torch.bfloat16, seed=6)
    wide = torch.zeros(5, 903, dtype=torch.bfloat16, device=dev)
    view = wide[:, 101:801]
    view.copy_(z)
    a = itf.distill_topk_with_grad(z, q, ids, weight=w)
    b = itf.distill_topk_with_grad(view, q, ids, weight=w)
    assert_close(a[0], _np(b[0]), 1e-6, "loss")
    assert_close(a[1], _np(b[1]), 2.0 ** -8, "gradient")
    leaf = view.detach().requires_grad_(True)
    g, = torch.autograd.grad(itf.distill_topk(leaf, q, ids, weight=w), leaf, torch.ones(5, device=dev))
    assert_close(g, _np(a[1]), 2.0 ** -8, "autograd gradient")
    turned = z.t().contiguous().t()                    # a strided last dimension is copied
    assert_close(itf.distill_topk(turned, q, ids, weight=w), _np(a[0]), 1e-6, "transposed")


def test_offsets_past_32_bits():
    V = 70000
    z, q, ids, w, up = _inputs(3, V, 5, torch.float16, seed=7)
    gap = (1 << 30) + 1
    big = torch.empty(2 * gap + V, dtype=torch.float16, device=dev)
    far = torch.as_strided(big, (3, V), (gap, 1))
    far.copy_(z)
    a, b = itf.distill_topk_with_grad(z, q, ids, weight=w), itf.distill_topk_with_grad(far, q, ids, weight=w)
    assert_close(a[0], _np(b[0]), 1e-6, "loss")
    assert_close(a[1], _np(b[1]), 2.0 ** -11, "gradient")
    del big, far
    T = (1 << 31) // V + 2                             # a gradient of more than 2^31 elements
    rows = z[:1].expand(T, V)
    loss, dz = itf.distill_topk_with_grad(rows, q[:1].expand(T, 5), ids[:1].expand(T, 5))
    assert_exact(loss, loss[:1].expand(T), "equal rows")
    assert_exact(dz[-1], dz[0], "last row")


def test_gradient_against_differences():
    z, q, ids, w, up = _inputs(3, 211, 7, torch.float32, seed=8)
    leaf = z.clone().requires_grad_(True)
    g, = torch.autograd.grad(itf.distill_topk(leaf, q, ids, weight=w, temperature=3.0), leaf, up)
    d = np.random.default_rng(1).standard_normal(z.shape)
    f = lambda s: float((orc.loss_and_grad(_np(z) + s * d, _np(q), ids.cpu().numpy(), _np(w), 3.0)[0] * _np(up)).sum())
    want = (f(1e-5) - f(-1e-5)) / 2e-5
    g = _np(g)
    assert abs((g * d).sum() - want) <= 1e-5 * np.abs(g).max() * np.abs(d).sum() + 1e-7


def test_empty_batch_and_stream():
    z, q, ids, w, up = _inputs(4, 3000, 8, torch.float32, seed=9)
    loss, dz = itf.distill_topk_with_grad(z[:0], q[:0], ids[:0])
    assert loss.shape == (0,) and dz.shape == (0, 3000)
    want = itf.distill_topk_with_grad(z, q, ids)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        late = torch.zeros_like(z)
        torch.cuda._sleep(20_000_000)
        late.copy_(z)
        got = itf.distill_topk_with_grad(late, q, ids)
    s.synchronize()
    assert_exact(got[0], want[0], "loss")
    assert_exact(got[1], want[1], "gradient")


def test_refusals():
    z, q, ids, w, up = _inputs(2, 50, 3, torch.float32, seed=10)
    ok = dict(logits=z, teacher_logits=q, teacher_ids=ids)
    for bad, match in [(dict(logits=z.double()), "float32, float16 or bfloat16"), (dict(logits=z[0]), "\\(T, V\\)"),
                       (dict(teacher_ids=ids.short()), "int32 or int64"), (dict(teacher_ids=ids[:, :2]), "teacher_ids"),
                       (dict(teacher_logits=q[:1], teacher_ids=ids[:1]), "teacher_logits"), (dict(weight=w[:1]), "weight"),
                       (dict(weight=w.half()), "weight"), (dict(temperature=0.0), "temperature"), (dict(temperature=math.inf), "temperature"),
                       (dict(teacher_logits=torch.zeros(2, 0, device=dev), teacher_ids=ids[:, :0]), "k must be"),
                       (dict(teacher_logits=torch.zeros(2, 1025, device=dev), teacher_ids=torch.zeros(2, 1025, dtype=torch.int64, device=dev)), "k must be"),
                       (dict(logits=z.cpu()), "CUDA")]:
        for f in (itf.distill_topk, itf.distill_topk_with_grad):
            with pytest.raises(RuntimeError, match=match):
                f(**{**ok, **bad})


def test_second_derivatives_are_refused():
    z, q, ids, w, up = _inputs(2, 50, 3, torch.float32, seed=11)
    z.requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(itf.distill_topk(z, q, ids).sum(), z, create_graph=True)
