"""GPU parity of the norms of a linear-attention block against the float64 oracle.

Tolerances (derived, elementwise |x - ref| <= tol |ref| + tol max|ref|): 16-bit outputs are rounded once, half a step
(bf16 2^-8, fp16 2^-11).  float32: a mean over W values of one sign is within 8 roundings (eight in a thread, then a
tree), the factors of an element within a dozen more, 20 * 2^-24 = 1.2e-6, the second term of a gradient as much
again: 5e-6.  Column sums over T rows with random signs add up T roundings of 2^-24, relative to a sum of size
sqrt(T): 5e-6 + sqrt(T) 2^-24.
dx = r (dn - x r^2 mean(dn x)) is a difference: for one feature a group the two terms r dn and r dn x^2 / (x^2 + eps)
cancel down to r dn eps / (x^2 + eps), for two often by much, and each is within 5e-6 of itself: dx is compared next to
its largest term r dn."""
import math

import numpy as np
import pytest
import torch

from bc_mamba_b200 import interface as itf
from helpers import assert_close, assert_exact
from oracle import block_norm as orc

pytestmark = pytest.mark.gpu
dev = "cuda"
F32 = 5e-6
TOL = {torch.float32: F32, torch.bfloat16: 2.0 ** -8 + F32, torch.float16: 2.0 ** -11 + F32}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _sums(rows):
    return F32 + math.sqrt(rows) * 2.0 ** -24


def _rn(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def _close_dx(got, ref, x, z, w, d, groups, eps, tol, what):
    x, z, w, d = (_np(t) for t in (x, z, w, d))
    parts = x.reshape(x.shape[0], groups, -1)
    r = np.repeat(1 / np.sqrt((parts ** 2).mean(-1) + eps), parts.shape[-1], axis=-1)
    terms = np.abs(r * d * w * z / (1 + np.exp(-z))).max()
    err = np.abs(_np(got) - ref)
    assert (err <= tol * (np.abs(ref) + np.abs(ref).max() + terms)).all(), (what, err.max(), np.abs(ref).max(), terms)


SHAPES = [(1, 1, 1), (3, 8, 1), (5, 24, 3), (7, 64, 1), (300, 65, 1), (33, 256, 4), (9, 255, 1), (21, 1000, 8), (12, 1001, 1), (4, 2048, 1),
          (3, 2049, 1), (2, 4096, 1), (5, 8192, 1), (2, 4097, 1), (2, 8191, 1), (2, 8192, 512), (4000, 40, 5), (0, 16, 2)]


@pytest.mark.parametrize("T,D,groups", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_norm(T, D, groups, dtype):
    x, z, d = (_rn(T, D, seed=n, dtype=dtype).requires_grad_(n < 2) for n in range(3))
    w = (1 + 0.3 * _rn(D, seed=3)).requires_grad_(True)
    out = itf.gated_norm(x, z, w, groups=groups, eps=1e-5)
    grads = torch.autograd.grad(out, [x, z, w], d)
    if T == 0:
        assert (grads[2] == 0).all() and out.shape == x.shape
        return
    want = orc.gated(_np(x), _np(z), _np(w), groups, 1e-5, _np(d))
    assert out.dtype == dtype and grads[2].dtype == torch.float32
    assert_close(out, want[0], TOL[dtype], "out")
    _close_dx(grads[0], want[1], x, z, w, d, groups, 1e-5, TOL[dtype], "dx")
    assert_close(grads[1], want[2], TOL[dtype], "dgate")
    assert_close(grads[2], want[3], _sums(T), "dweight")


@pytest.mark.parametrize("T,D", [s[:2] for s in SHAPES])
@pytest.mark.parametrize("dtype,wide", [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, False), (torch.float16, True)])
@pytest.mark.parametrize("scaled", [False, True])
def test_add_norm(T, D, dtype, wide, scaled):
    rt = torch.float32 if wide else dtype
    r, b = _rn(T, D, seed=0, dtype=rt).requires_grad_(True), _rn(T, D, seed=1, dtype=dtype).requires_grad_(True)
    dr, d = _rn(T, D, seed=2, dtype=rt), _rn(T, D, seed=4, dtype=dtype)
    w = (1 + 0.3 * _rn(D, seed=3)).requires_grad_(True)
    s = (0.5 + 0.3 * _rn(D, seed=5)).requires_grad_(True) if scaled else None
    v, out = itf.add_norm(r, b, w, scale=s, eps=1e-5)
    leaves = [r, b, w] + ([s] if scaled else [])
    grads = torch.autograd.grad([v, out], leaves, [dr, d])
    if T == 0:
        assert all((g == 0).all() for g in grads[2:]) and v.shape == r.shape
        return
    want = orc.add(_np(r), _np(b), _np(w), _np(s), 1e-5, _np(dr), _np(d))
    assert v.dtype == rt and out.dtype == dtype
    for got, ref, what, t in zip((v, out, *grads[:2]), want, ("v", "out", "dresidual", "dbranch"), (rt, dtype, rt, dtype)):
        assert_close(got, ref, TOL[t], what)
    for got, ref, what in zip(grads[2:], want[4:], ("dweight", "dscale")):
        assert_close(got, ref, _sums(T), what)


@pytest.mark.parametrize("scaled", [False, True])
def test_one_upstream_gradient(scaled):
    r, b, w = _rn(40, 100, seed=0).requires_grad_(True), _rn(40, 100, seed=1).requires_grad_(True), _rn(100, seed=2).requires_grad_(True)
    s = _rn(100, seed=3).requires_grad_(True) if scaled else None
    d = _rn(40, 100, seed=4)
    for which in (0, 1):
        outs = itf.add_norm(r, b, w, scale=s)
        grads = torch.autograd.grad(outs[which], [r, b, w], d)
        want = orc.add(_np(r), _np(b), _np(w), _np(s), 1e-6, _np(d) if which == 0 else None, _np(d) if which else None)
        for got, ref, what in zip(grads, want[2:5], ("dresidual", "dbranch", "dweight")):
            assert_close(got, ref, _sums(40), what)


def test_many_rows_and_groups():
    """More rows than blocks stay for, and more groups than there are blocks."""
    x, z, d = (_rn(30000, 40, seed=n).requires_grad_(n < 2) for n in range(3))
    w = _rn(40, seed=3).requires_grad_(True)
    out = itf.gated_norm(x, z, w, groups=5)
    want = orc.gated(_np(x), _np(z), _np(w), 5, 1e-6, _np(d))
    grads = torch.autograd.grad(out, [x, z, w], d)
    assert_close(grads[0], want[1], F32, "dx")
    assert_close(grads[2], want[3], _sums(30000), "dweight")
    x, z, d = (_rn(6, 6000, seed=n).requires_grad_(n < 2) for n in range(3))
    w = _rn(6000, seed=3).requires_grad_(True)
    out = itf.gated_norm(x, z, w, groups=3000)
    want = orc.gated(_np(x), _np(z), _np(w), 3000, 1e-6, _np(d))
    grads = torch.autograd.grad(out, [x, z, w], d)
    _close_dx(grads[0], want[1], x, z, w, d, 3000, 1e-6, F32, "dx of pairs")
    for got, ref in zip((out, *grads[1:]), (want[0], *want[2:])):
        assert_close(got, ref, F32, "pairs")


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    """Rows of a wider buffer on and off 16 bytes, leading dimensions that do not merge, strided features."""
    wide = _rn(3, 7, 301, seed=0, dtype=dtype)
    w = _rn(96, seed=1)
    for x, z in [(wide[..., :96], wide[..., 96:192]), (wide[..., 1:97], wide[..., 200:296]), (wide[:, 1:4, 8:104], wide[:, 3:6, 104:200]),
                 (wide.transpose(0, 1)[..., :96], wide.transpose(0, 1)[..., 96:192]), (wide[..., :192:2], wide[..., 1:192:2])]:
        a = itf.gated_norm(x, z, w, groups=3)
        b = itf.gated_norm(x.contiguous(), z.contiguous(), w, groups=3)
        assert_close(a, _np(b), TOL[dtype], "gated")
        for got, want in zip(itf.add_norm(x, z, w), itf.add_norm(x.contiguous(), z.contiguous(), w)):
            assert_close(got, _np(want), TOL[dtype], "add")
        leaves, plain = [x.detach().requires_grad_(True), z.detach().requires_grad_(True)], [x.contiguous().requires_grad_(True), z.contiguous().requires_grad_(True)]
        d = torch.ones_like(a)
        for got, want in zip(torch.autograd.grad(itf.gated_norm(*leaves, w, groups=3), leaves, d.expand(d.shape)),
                             torch.autograd.grad(itf.gated_norm(*plain, w, groups=3), plain, d)):
            assert_close(got, _np(want), TOL[dtype], "gradient")


def test_zero_rows_and_what_is_not_finite():
    x, z, w = torch.zeros(3, 64, device=dev), _rn(3, 64, seed=0), _rn(64, seed=1)
    assert (itf.gated_norm(x, z, w, groups=2) == 0).all()
    v, out = itf.add_norm(x, x, w)
    assert (v == 0).all() and (out == 0).all()
    x = _rn(3, 64, seed=2)
    x[1, 3] = math.nan
    out = itf.gated_norm(x, z, w, groups=2)
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all() and torch.isfinite(out[1, 32:]).all()
    assert torch.isnan(out[1, :32]).all()


def test_same_from_run_to_run_streams_and_graphs():
    x, z, d = (_rn(5000, 300, seed=n, dtype=torch.bfloat16).requires_grad_(n < 2) for n in range(3))
    w, s = _rn(300, seed=4).requires_grad_(True), _rn(300, seed=5).requires_grad_(True)

    def call():
        a = itf.gated_norm(x, z, w, groups=3)
        b = itf.add_norm(x, z, w, scale=s)
        return (a.detach(), *(t.detach() for t in b), *torch.autograd.grad(a, [x, z, w], d), *torch.autograd.grad(b, [x, z, w, s], [d, d]))

    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = call()
    torch.cuda.current_stream().wait_stream(side)
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, held):
        assert_exact(a, b, "stream")
        assert_exact(a, c, "graph")


def test_refusals():
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, device=dev, dtype=dtype)
    x, w = z(4, 12), z(12)
    for call, why in [(lambda: itf.gated_norm(x, x, w, groups=5), "multiple of the groups"), (lambda: itf.gated_norm(x, x, w, groups=0), "multiple"),
                      (lambda: itf.gated_norm(x, x[:3], w), "gate has the wrong shape"), (lambda: itf.gated_norm(x, x.half(), w), "gate has the wrong device or dtype"),
                      (lambda: itf.gated_norm(x, x, w.half()), "weight must be a float32"), (lambda: itf.gated_norm(x, x, w, eps=0.0), "eps"),
                      (lambda: itf.gated_norm(x, x, w, eps=math.nan), "eps"), (lambda: itf.gated_norm(z(2, 8193), z(2, 8193), z(8193)), "more than 8192"),
                      (lambda: itf.gated_norm(x.cpu(), x, w), "CUDA"), (lambda: itf.add_norm(x, x, w, eps=-1.0), "eps"),
                      (lambda: itf.add_norm(x.half(), x, w), "dtype of branch or be float32"), (lambda: itf.add_norm(x[:3], x, w), "residual has the wrong shape"),
                      (lambda: itf.add_norm(x, x, w, scale=w[:3]), "scale has the wrong shape"), (lambda: itf.add_norm(x, x.double(), w), "float32, float16"),
                      (lambda: itf.add_norm(z(2, 8193), z(2, 8193), z(8193)), "more than 8192")]:
        with pytest.raises(RuntimeError, match=why):
            call()
    y = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(itf.gated_norm(y, x, w).sum(), y, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(itf.add_norm(y, x, w)[1].sum(), y, create_graph=True)
