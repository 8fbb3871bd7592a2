"""GPU parity of the linear attention with a decay for each head (forward, backward, packed sequences, one-token step)
against the float64 oracle.

Tolerances (derived, elementwise |x - ref| <= tol |ref| + tol max|ref|): an output in 16 bits is rounded once, half a
step (bf16 2^-8, fp16 2^-11).  float32 outputs: sums of up to 64 + 128 products, each with a rounding of 2^-24 and a
decay within 2^-22, whose magnitudes add up to at most sqrt(192) = 14 times the result of random signs: 14 * (2^-22 +
sqrt(192) 2^-24) = 1.5e-5 at worst; with 16-bit inputs each product carries a piece's rounding of 2^-18, which
enters with random signs like the result itself, 4e-6: 2e-5 bounds both, and is added to the 16-bit outputs'."""
import math

import numpy as np
import pytest
import torch

from bc_mamba_b200 import interface as itf
from helpers import assert_close, assert_exact
from oracle import decay_attn as orc

pytestmark = pytest.mark.gpu
dev = "cuda"
F32 = 2e-5
TOL = {torch.float32: F32, torch.bfloat16: 2.0 ** -8 + F32, torch.float16: 2.0 ** -11 + F32}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(rows, n, heads, hk, dk, dv, dtype, seed, strong=False):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    t = dict(q=rn(rows, hk, dk) * dk ** -0.5, k=rn(rows, hk, dk), v=rn(rows, heads, dv), dy=rn(rows, heads, dv))
    t = {k: v.to(dtype).to(dev) for k, v in t.items()}
    decay = torch.rand(rows, heads, generator=g)
    t["g"] = (-(20.0 * decay ** 4) if strong else -0.2 * decay).to(dev)
    t["h0"], t["dh"] = rn(n, heads, dk, dv).to(dev), rn(n, heads, dk, dv).to(dev)
    return t


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _check(t, cu, shape, with_h0=True, with_dy=True, with_dh=True, fixed=False):
    """Forward and backward on `shape` ((B, L) dense, None packed), every output against the oracle."""
    cu = [int(c) for c in cu]
    dtype, rows = t["v"].dtype, t["v"].shape[0]
    view = (lambda x: x.reshape(*shape, *x.shape[1:])) if shape else (lambda x: x)
    flat = lambda x: x.reshape(rows, *x.shape[2:]) if shape else x
    names = ["q", "k", "v"]
    leaves = {k: view(t[k]).detach().clone().requires_grad_(True) for k in names}
    g = t["g"]
    if fixed:
        g = t["g"][0].expand_as(t["g"])
        leaves["g"] = t["g"][0].clone().requires_grad_(True)
    else:
        leaves["g"] = view(t["g"]).clone().requires_grad_(True)
    if with_h0:
        leaves["h0"] = t["h0"].clone().requires_grad_(True)
    cu_t = None if shape else torch.tensor(cu, dtype=torch.int32, device=dev)
    y, h_last = itf.decay_attention(leaves["q"], leaves["k"], leaves["v"], leaves["g"], h0=leaves.get("h0"), cu_seqlens=cu_t)
    assert y.dtype == dtype and y.shape == leaves["v"].shape and h_last.dtype == torch.float32
    a = [_np(t[k]) for k in names] + [_np(g)]
    h0 = _np(t["h0"]) if with_h0 else None
    ry, rh = orc.fwd(*a, h0, cu)
    assert_close(flat(y), ry, TOL[dtype], "y")
    assert_close(h_last, rh, F32, "h_last")
    outs = ([y] if with_dy else []) + ([h_last] if with_dh else [])
    ups = ([view(t["dy"])] if with_dy else []) + ([t["dh"]] if with_dh else [])
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), ups)))
    ref = dict(zip(("q", "k", "v", "g", "h0"), orc.bwd(*a, h0, cu, _np(t["dy"]) if with_dy else None, _np(t["dh"]) if with_dh else None)))
    for k in leaves:
        got, want = grads[k], ref[k]
        if k == "g" and fixed:
            # a sum over the rows whose signs may cancel: the roundings of each add up like sqrt(rows)
            assert_close(got, want.sum(0), F32 * math.sqrt(rows), "dg")
            continue
        if k != "h0":
            got = flat(got)
        # exp(-100) = 2^-144 lies below float32's least normal number, 2^-126, and the exponentials flush such values:
        # a gradient that is smaller as a whole counts as 0
        want = np.where(np.abs(want) < 2.0 ** -126, 0.0, want)
        assert_close(got, want, TOL[dtype] if k in names else F32, "d" + k)


@pytest.mark.parametrize("B,L,H,Hk,N,P", [(1, 1, 1, 1, 1, 1), (2, 3, 2, 1, 5, 7), (1, 63, 3, 3, 16, 32), (2, 64, 2, 2, 17, 33), (1, 65, 4, 2, 32, 64),
                                          (2, 129, 2, 1, 64, 65), (1, 200, 3, 1, 128, 64), (1, 193, 2, 2, 127, 130), (2, 128, 1, 1, 8, 300),
                                          (1, 1000, 2, 2, 48, 80), (40, 7, 9, 3, 12, 20)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_dense(B, L, H, Hk, N, P, dtype):
    _check(_inputs(B * L, B, H, Hk, N, P, dtype, seed=B + L + N), range(0, B * L + 1, L), (B, L))


@pytest.mark.parametrize("cu", [(0, 1), (0, 0, 1, 1), (0, 5, 5, 5, 200), (0, 64, 128, 192, 193), (0, 127, 129, 129, 700), tuple(range(0, 71))])
@pytest.mark.parametrize("N,P,dtype", [(5, 9, torch.float32), (64, 64, torch.bfloat16), (16, 40, torch.float16)])
def test_packed(cu, N, P, dtype):
    _check(_inputs(cu[-1], len(cu) - 1, 4, 2, N, P, dtype, seed=len(cu) + N), cu, None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sequences_in_items(dtype):
    """Few heads and long sequences are cut into items of 256 tokens and more, their states joined; packed sequences
    that begin at an item's first token, end at its last, and span several."""
    _check(_inputs(2 * 1500, 2, 2, 1, 16, 24, dtype, seed=1), (0, 1500, 3000), (2, 1500))
    for cu in ((0, 256, 512, 512, 1100, 2500), (0, 1, 255, 256, 2499, 2500), (0, 2500), (0, 0, 2500, 2500)):
        _check(_inputs(2500, len(cu) - 1, 2, 2, 20, 33, dtype, seed=len(cu)), cu, None)
    t = _inputs(2500, 3, 2, 2, 20, 33, dtype, seed=9)
    _check(t, (0, 600, 1280, 2500), None, False, True, False)
    _check(t, (0, 600, 1280, 2500), None, True, False, True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_partial_gradients(dtype):
    t = _inputs(2 * 100, 2, 4, 2, 24, 40, dtype, seed=5)
    for h0, dy, dh in ((False, True, False), (True, True, False), (True, False, True)):
        _check(t, (0, 100, 200), (2, 100), h0, dy, dh)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_decay_for_each_head(dtype):
    _check(_inputs(2 * 150, 2, 4, 2, 24, 40, dtype, seed=6), (0, 150, 300), (2, 150), fixed=True)
    _check(_inputs(300, 3, 300, 150, 4, 3, dtype, seed=7), (0, 150, 150, 300), None, fixed=True)
    _check(_inputs(300, 3, 3, 1, 8, 90, dtype, seed=8), (0, 150, 150, 300), None, fixed=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strong_decays(dtype):
    _check(_inputs(2 * 200, 2, 2, 1, 16, 24, dtype, seed=3, strong=True), (0, 200, 400), (2, 200))


def test_gradient_of_a_strong_decay_keeps_its_digits():
    """dg_t is proportional to a_t: with every decay between exp(-30) and exp(-10) each value agrees relative to
    itself (the sums of up to 64 terms that the token's own dominate, 32 times a rounding of 2^-22 with cancellation)."""
    t = _inputs(200, 1, 2, 2, 8, 8, torch.float32, seed=4)
    t["g"] = -10 - 20 * torch.rand(200, 2, generator=torch.Generator().manual_seed(0)).to(dev)
    leaf = t["g"][None].clone().requires_grad_(True)
    y, h = itf.decay_attention(t["q"][None], t["k"][None], t["v"][None], leaf, h0=t["h0"])
    got = torch.autograd.grad([y, h], leaf, [t["dy"][None], t["dh"]])[0][0]
    a = [_np(t[k]) for k in ("q", "k", "v", "g")]
    want = orc.bwd(*a, _np(t["h0"]), (0, 200), _np(t["dy"]), _np(t["dh"]))[3]
    size = np.exp(a[3]) * np.sqrt(8 * 8)           # of a product of two 8 x 8 matrices of such entries
    assert (np.abs(_np(got) - want) <= 1e-4 * np.abs(want) + 1e-5 * size).all()


@pytest.mark.parametrize("drop", [-math.inf, -3.4028234663852886e38, -1e4, -100.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_dropped_state(drop, dtype):
    """A log-decay of -inf, of the type's lowest value or merely large: what follows depends on nothing before, and
    the decays after it keep their precision."""
    t = _inputs(300, 1, 2, 1, 16, 24, dtype, seed=11)
    for at in (0, 1, 63, 64, 100, 101, 299):
        t["g"][at] = drop
    _check(t, (0, 300), (1, 300))
    y, h = itf.decay_attention(*(t[k][None] for k in ("q", "k", "v", "g")), h0=t["h0"])
    y2, h2 = itf.decay_attention(*(t[k][None, 101:] for k in ("q", "k", "v", "g")), h0=None)
    assert_close(y[:, 101:], _np(y2), TOL[dtype], "y after the drop")
    assert_close(h, _np(h2), F32, "h after the drop")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_finite_reaches_no_token_before_it(dtype, bad):
    t = _inputs(300, 2, 2, 1, 16, 40, dtype, seed=12)
    cu = torch.tensor([0, 180, 300], dtype=torch.int32, device=dev)
    clean, _ = itf.decay_attention(t["q"], t["k"], t["v"], t["g"], h0=t["h0"], cu_seqlens=cu)
    for name in ("q", "k", "v", "g"):
        if name == "g" and bad == math.inf:
            continue
        x = {k: t[k].clone() for k in ("q", "k", "v", "g")}
        x[name][100, 0] = bad
        y, h = itf.decay_attention(x["q"], x["k"], x["v"], x["g"], h0=t["h0"], cu_seqlens=cu)
        assert_exact(y[:64], clean[:64], "chunks before " + name)
        assert_close(y[64:100], _np(clean[64:100]), 2 * TOL[dtype], "tokens before " + name)
        assert_exact(y[180:], clean[180:], "the other sequence " + name)
        assert not torch.isfinite(y[100:180, 0]).all() and torch.isfinite(h[1]).all()
        ry, rh = orc.fwd(*(_np(x[k]) for k in ("q", "k", "v", "g")), _np(t["h0"]), (0, 180, 300))
        assert (np.isfinite(ry) == torch.isfinite(y).cpu().numpy()).all(), name
        assert (np.isfinite(rh) == torch.isfinite(h).cpu().numpy()).all(), name


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_a_chunk_with_nan(dtype):
    """A NaN in dy reaches the gradients of its own and earlier tokens alone; one in v those of q behind it, of k at it
    and of the decays that it meets.  What the oracle says is finite is finite and equal."""
    for name in ("dy", "v", "q", "k", "h0"):
        t = _inputs(150, 1, 2, 1, 8, 40, dtype, seed=13)
        (t[name][0, 1, 2] if name == "h0" else t[name][100, 0])[3] = math.nan
        leaves = {k: t[k][None].clone().requires_grad_(True) for k in ("q", "k", "v", "g")}
        h0 = t["h0"].clone().requires_grad_(True)
        y, h = itf.decay_attention(leaves["q"], leaves["k"], leaves["v"], leaves["g"], h0=h0)
        grads = torch.autograd.grad([y, h], [*leaves.values(), h0], [t["dy"][None], t["dh"]])
        ref = orc.bwd(*(_np(t[k]) for k in ("q", "k", "v", "g")), _np(t["h0"]), (0, 150), _np(t["dy"]), _np(t["dh"]))
        for which, got, want in zip(("dq", "dk", "dv", "dg", "dh0"), grads, ref):
            got = _np(got if which == "dh0" else got[0])
            fine = np.isfinite(want)
            assert np.isfinite(got[fine]).all(), (name, which)
            if fine.any():
                tol = TOL[dtype] if which in ("dq", "dk", "dv") else F32
                assert (np.abs(got - want)[fine] <= tol * (np.abs(want[fine]) + np.abs(want[fine]).max())).all(), (name, which)


def test_rows_behind_the_last_sequence_are_zero():
    t = _inputs(700, 2, 2, 1, 16, 72, torch.bfloat16, seed=14)
    cu = torch.tensor([0, 100, 130], dtype=torch.int32, device=dev)
    for k in ("q", "k", "v", "g"):
        t[k][130:] = math.nan
    leaves = {k: t[k].clone().requires_grad_(True) for k in ("q", "k", "v", "g")}
    y, h = itf.decay_attention(*leaves.values(), h0=t["h0"], cu_seqlens=cu)
    grads = torch.autograd.grad([y, h], list(leaves.values()), [t["dy"], t["dh"]])
    for x in (y, *grads):
        assert (x[130:] == 0).all() and torch.isfinite(x[:130]).all()


def test_bad_offsets_stay_in_range():
    """Offsets that leave the rows or are not ascending: undefined values, but every access in range and every sum
    ended (bounded by a table of the rows that exist)."""
    t = _inputs(300, 4, 2, 1, 16, 24, torch.float32, seed=15)
    for cu in ((0, 500, 200, 300, 300), (-5, 100, 90, 2000, 10), (300, 0, 300, 0, 300)):
        c = torch.tensor(cu, dtype=torch.int32, device=dev)
        y, h = itf.decay_attention(t["q"], t["k"], t["v"], t["g"], h0=t["h0"], cu_seqlens=c)
        assert y.shape == t["v"].shape
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """Slices of one projection, heads before tokens, batch rows apart, rows off 16 bytes: as contiguous copies."""
    B, L, H, N, P = 2, 150, 4, 16, 32
    t = _inputs(B * L, B, H, H, N, P, dtype, seed=16)
    q, k, v, g = (t[x].reshape(B, L, *t[x].shape[1:]) for x in ("q", "k", "v", "g"))
    want = itf.decay_attention(q, k, v, g, h0=t["h0"])
    wide = torch.zeros(B, L + 3, H * (2 * N + P) + 1, device=dev, dtype=dtype)[:, 2:L + 2, 1:]
    wide[..., :H * N], wide[..., H * N:2 * H * N], wide[..., 2 * H * N:] = q.flatten(2), k.flatten(2), v.flatten(2)
    a, b, c = wide.split([H * N, H * N, H * P], -1)
    layouts = [(a.unflatten(-1, (H, N)), b.unflatten(-1, (H, N)), c.unflatten(-1, (H, P)), g.transpose(1, 2).contiguous().transpose(1, 2)),
               tuple(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, g)),
               tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, g)),
               (q.transpose(-1, -2).contiguous().transpose(-1, -2), k, v, g)]
    for x in layouts:
        leaves = [y.detach().requires_grad_(True) for y in x]
        got = itf.decay_attention(*leaves, h0=t["h0"])
        assert_exact(got[0], want[0], "y")
        assert_exact(got[1], want[1], "h_last")
        dy = t["dy"].reshape(B, L, H, P)
        one = torch.autograd.grad(got, leaves, [dy, t["dh"]])
        plain = [y.detach().clone().requires_grad_(True) for y in (q, k, v, g)]
        two = torch.autograd.grad(itf.decay_attention(*plain, h0=t["h0"]), plain,
                                  [dy.transpose(1, 2).contiguous().transpose(1, 2), t["dh"]])
        for m, n in zip(one, two):
            assert_exact(m, n, "gradient")


def test_gradient_equals_differences():
    """Central differences of the forward in float32: step 1e-2 on values of order one, truncation 1e-4 of the third
    derivative and 2e-5 / 1e-2 of rounding in sums of 40 outputs."""
    t = _inputs(40, 1, 1, 1, 4, 4, torch.float32, seed=17)
    x = [t[k][None].clone().requires_grad_(True) for k in ("q", "k", "v", "g")]
    w = t["dy"][None]
    loss = lambda *a: (itf.decay_attention(*a, h0=t["h0"])[0].double() * w.double()).sum()
    grads = torch.autograd.grad(loss(*x), x)
    gen = torch.Generator().manual_seed(1)
    for n, leaf in enumerate(x):
        d = torch.randn(leaf.shape, generator=gen).to(dev)
        d = d / d.norm()
        up = [a.detach() + (1e-2 * d if m == n else 0) for m, a in enumerate(x)]
        down = [a.detach() - (1e-2 * d if m == n else 0) for m, a in enumerate(x)]
        num = (loss(*up) - loss(*down)).item() / 2e-2
        assert abs(num - (grads[n] * d).sum().item()) <= 5e-3 * (1 + abs(num)) * grads[n].norm().item() ** 0.5 + 5e-3, n


@pytest.mark.parametrize("B,H,Hk,N,P", [(1, 1, 1, 1, 1), (1, 4, 1, 16, 64), (3, 6, 2, 17, 33), (2, 2, 2, 128, 256), (5, 3, 3, 64, 60), (70, 3, 1, 8, 4)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_step(B, H, Hk, N, P, dtype):
    t = _inputs(B, B, H, Hk, N, P, dtype, seed=B + N)
    h = t["h0"].clone()
    y = itf.decay_attention_step(t["q"], t["k"], t["v"], t["g"], h)
    ry, rh = orc.fwd(*(_np(t[k]) for k in ("q", "k", "v", "g")), _np(t["h0"]), range(B + 1))
    assert_close(y, ry, TOL[dtype], "y")
    assert_close(h, rh, 1e-6, "h")
    h = t["h0"].clone()
    itf.decay_attention_step(t["q"], t["k"], t["v"], t["g"][0], h)
    _, rh = orc.fwd(*(_np(t[k]) for k in ("q", "k", "v")), _np(t["g"][:1].expand(B, H)), _np(t["h0"]), range(B + 1))
    assert_close(h, rh, 1e-6, "h of one decay for each head")


def test_steps_continue_a_prefill():
    t = _inputs(2 * 90, 2, 4, 2, 16, 24, torch.bfloat16, seed=20)
    q, k, v, g = (t[x].reshape(2, 90, *t[x].shape[1:]) for x in ("q", "k", "v", "g"))
    y, h_all = itf.decay_attention(q, k, v, g, h0=t["h0"])
    _, h = itf.decay_attention(q[:, :70], k[:, :70], v[:, :70], g[:, :70], h0=t["h0"])
    for s in range(70, 90):
        out = itf.decay_attention_step(q[:, s], k[:, s], v[:, s], g[:, s], h)
        assert_close(out, _np(y[:, s]), 2 * TOL[torch.bfloat16], "step")
    assert_close(h, _np(h_all), F32, "h")


def test_same_from_run_to_run_streams_and_graphs():
    t = _inputs(900, 3, 4, 2, 32, 72, torch.bfloat16, seed=21)
    cu = torch.tensor([0, 400, 400, 900], dtype=torch.int32, device=dev)
    leaves = [t[k].clone().requires_grad_(True) for k in ("q", "k", "v", "g")]

    def call():
        out = itf.decay_attention(*leaves, h0=t["h0"], cu_seqlens=cu)
        return (*(o.detach() for o in out), *torch.autograd.grad(out, leaves, [t["dy"], t["dh"]]))

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
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, held):
        assert_exact(a, b, "stream")
        assert_exact(a, c, "graph")


def test_no_tokens_and_no_sequences():
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, device=dev, dtype=dtype)
    h0 = torch.randn(2, 3, 4, 5, device=dev)
    leaf = z(2, 0, 3, 5).requires_grad_(True)
    y, h = itf.decay_attention(z(2, 0, 1, 4), z(2, 0, 1, 4), leaf, z(3), h0=h0)
    assert y.shape == (2, 0, 3, 5) and torch.equal(h, h0)
    assert torch.autograd.grad(h.sum(), leaf)[0].shape == leaf.shape
    y, h = itf.decay_attention(z(0, 7, 1, 4), z(0, 7, 1, 4), z(0, 7, 3, 5), z(0, 7, 3))
    assert y.shape == (0, 7, 3, 5) and h.shape == (0, 3, 4, 5)
    y, h = itf.decay_attention(z(0, 1, 4), z(0, 1, 4), z(0, 3, 5), z(0, 3), cu_seqlens=z(3, dtype=torch.int32), h0=h0)
    assert torch.equal(h, h0)
    assert itf.decay_attention_step(z(0, 1, 4), z(0, 1, 4), z(0, 3, 5), z(0, 3), z(0, 3, 4, 5)).shape == (0, 3, 5)


def test_refusals():
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, device=dev, dtype=dtype)
    q, v, g = z(2, 5, 2, 8), z(2, 5, 4, 6), z(2, 5, 4)
    for bad, why in [((q, q, v, z(2, 5, 3)), "log_decay has the wrong shape"), ((q, q, v, g.double()), "log_decay must be a float32"),
                     ((q, q[:, :4], v, g), "one shape"), ((q, q, v[0], g), "must be"), ((q.half(), q, v, g), "device and dtype"),
                     ((z(2, 5, 3, 8), z(2, 5, 3, 8), v, g), "multiple"), ((q.double(), q.double(), v.double(), g), "float32, float16 or bfloat16"),
                     ((z(2, 5, 2, 129), z(2, 5, 2, 129), v, g), "more than 128"), ((q, q, v.cpu(), g), "CUDA")]:
        with pytest.raises(RuntimeError, match=why):
            itf.decay_attention(*bad)
    with pytest.raises(RuntimeError, match="h0 has the wrong shape"):
        itf.decay_attention(q, q, v, g, h0=z(2, 4, 6, 8))
    with pytest.raises(RuntimeError, match="cu_seqlens"):
        itf.decay_attention(q[0], q[0], v[0], g[0], cu_seqlens=z(3, dtype=torch.int64))
    h = z(2, 4, 8, 6)
    with pytest.raises(RuntimeError, match="contiguous"):
        itf.decay_attention_step(q[:, 0], q[:, 0], v[:, 0], g[:, 0], h.transpose(2, 3))
    with pytest.raises(RuntimeError, match="no gradient passes"):
        itf.decay_attention_step(q[:, 0], q[:, 0], v[:, 0].clone().requires_grad_(True), g[:, 0], h)
    leaf = h.clone().requires_grad_(True)
    saved = (leaf * 2) * 1
    keep = saved * saved
    with torch.no_grad():
        itf.decay_attention_step(q[:, 0], q[:, 0], v[:, 0], g[:, 0], saved)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        keep.sum().backward()
    x = v.clone().requires_grad_(True)
    y, _ = itf.decay_attention(q, q, x, g)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [1, 2, 7, 8, 9])
@pytest.mark.parametrize("N,P,H,Hk", [(5, 9, 2, 1), (64, 64, 3, 3), (128, 132, 2, 2)])
@pytest.mark.parametrize("entering", [False, True])
def test_few_tokens_without_a_gradient(L, dtype, N, P, H, Hk, entering):
    """Calls that record no gradient give what calls that do give: float32 sums of at most N products for the former, two
    bfloat16 pieces of 2^-18 for the latter, so 2 half steps of the output's type and 2^-16 apart next to the largest."""
    g = torch.Generator(device=dev).manual_seed(L)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev)
    q, k, v = (rn(3, L, Hk, N) * N ** -0.5).to(dtype), rn(3, L, Hk, N).to(dtype), rn(3, L, H, P).to(dtype)
    log_decay, h0 = -torch.rand(3, L, H, generator=g, device=dev), rn(3, H, N, P) if entering else None
    y, h = itf.decay_attention(q, k, v, log_decay, h0=h0)
    y2, h2 = itf.decay_attention(q.requires_grad_(True), k, v, log_decay, h0=h0)
    tol = torch.finfo(dtype).eps + 2.0 ** -16
    assert ((y - y2).abs() <= tol * (y2.abs() + y2.abs().max())).all()
    assert ((h - h2).abs() <= 2.0 ** -16 * (h2.abs() + h2.abs().max())).all()
