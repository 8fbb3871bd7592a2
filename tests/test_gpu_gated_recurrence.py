"""GPU parity of the gated linear recurrence (forward, backward, packed
sequences, one-token step) against the float64 oracle.

Tolerances (derived, elementwise |x - ref| <= tol |ref| + tol max|ref|):
fp32 values carry a few roundings per token, each fading with the decay, 1e-5;
16-bit values are rounded once, half an ulp of bf16 (2^-9) or fp16 (2^-12),
doubled, on top of 1e-5; dlam adds N signed terms per feature, each within
1e-6, whose sum may cancel to 1/sqrt(N) of their magnitudes: 1e-5 + 1e-6 sqrt(N)."""
import math

import numpy as np
import pytest
import torch

from bc_mamba_b200 import interface as itf
from helpers import assert_close, assert_exact
from oracle import gated_rec as orc

pytestmark = pytest.mark.gpu
dev = "cuda"
TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11 + 1e-5}


def _inputs(rows, d, n, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    t = dict(x=rn(rows, d), r=spread * rn(rows, d), i=spread * rn(rows, d), dy=rn(rows, d))
    t = {k: v.to(dtype).to(dev) for k, v in t.items()}
    decay = 0.9 + 0.099 * torch.rand(d, generator=g)
    t["lam"] = torch.log(torch.expm1(-0.25 * torch.log(decay))).to(dev)
    t["h0"], t["dh"] = rn(n, d).to(dev), rn(n, d).to(dev)
    return t


def _np(t):
    return t.detach().double().cpu().numpy()


def _check(t, cu, shape, with_h0=True, with_dy=True, with_dh=True, c=8.0):
    """Runs forward and backward on `shape` ((B, L) dense, None packed) and compares every output."""
    cu_np = [int(v) for v in cu]
    dtype, d, n = t["x"].dtype, t["x"].shape[-1], len(cu_np) - 1
    view = (lambda v: v.reshape(*shape, d)) if shape else (lambda v: v)
    flat = lambda v: v.reshape(-1, d)
    leaves = {k: view(t[k]).detach().clone().requires_grad_(True) for k in ("x", "r", "i")}
    leaves["lam"] = t["lam"].clone().requires_grad_(True)
    if with_h0:
        leaves["h0"] = t["h0"].clone().requires_grad_(True)
    cu_t = None if shape else torch.tensor(cu_np, dtype=torch.int32, device=dev)
    y, h_last = itf.gated_recurrence(leaves["x"], leaves["r"], leaves["i"], leaves["lam"], h0=leaves.get("h0"),
                                     cu_seqlens=cu_t, decay_scale=c)
    assert y.dtype == dtype and h_last.dtype == torch.float32
    a = [_np(t[k]) for k in ("x", "r", "i")]
    lam, h0 = _np(t["lam"]), _np(t["h0"]) if with_h0 else None
    ry, rh = orc.fwd(*a, lam, h0, cu_np, c)
    assert_close(flat(y), ry, TOL[dtype], "y")
    assert_close(h_last, rh, 1e-5, "h_last")
    outs, ups = [], []
    if with_dy:
        outs, ups = outs + [y], ups + [view(t["dy"])]
    if with_dh:
        outs, ups = outs + [h_last], ups + [t["dh"]]
    grads = torch.autograd.grad(outs, list(leaves.values()), ups)
    rx, rr, ri, rl, r0 = orc.bwd(*a, lam, h0, cu_np, _np(t["dy"]) if with_dy else None, _np(t["dh"]) if with_dh else None, c)
    ref = dict(x=rx, r=rr, i=ri, lam=rl, h0=r0)
    rows = t["x"].shape[0]
    for k, gk in zip(leaves, grads):
        tol = TOL[dtype] if k in "xri" else 1e-5 + 1e-6 * math.sqrt(rows) if k == "lam" else 1e-5
        assert_close(flat(gk) if k in "xri" else gk, ref[k], tol, "d" + k)


@pytest.mark.parametrize("B,L,D", [(1, 1, 1), (2, 3, 5), (3, 8, 32), (1, 9, 33), (2, 63, 64), (2, 64, 65), (1, 129, 200),
                                   (5, 257, 31), (2, 1000, 96), (1, 4097, 66), (70, 17, 130), (1, 2049, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dense(B, L, D, dtype):
    _check(_inputs(B * L, D, B, dtype, seed=B + L + D), range(0, B * L + 1, L), (B, L))


@pytest.mark.parametrize("B,L,D", [(3000, 1, 65), (700, 2, 64), (333, 7, 96), (90, 64, 33), (41, 65, 10), (9, 255, 6), (2, 256, 64),
                                   (1, 20000, 4)])
def test_many_short_and_one_long(B, L, D):
    _check(_inputs(B * L, D, B, torch.float32, seed=B + L), range(0, B * L + 1, L), (B, L))


@pytest.mark.parametrize("D", [63, 66, 129, 1001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_off_16_bytes(D, dtype):
    _check(_inputs(3 * 300, D, 3, dtype, seed=D), (0, 300, 600, 900), (3, 300))
    _check(_inputs(300, D, 4, dtype, seed=D), (0, 7, 7, 200, 300), None)
    _check(_inputs(40 * 7, D, 40, dtype, seed=D), range(0, 281, 7), (40, 7))


def test_half():
    _check(_inputs(2 * 300, 70, 2, torch.float16, seed=3), (0, 300, 600), (2, 300))


@pytest.mark.parametrize("cu", [(0, 1), (0, 0, 1, 1), (0, 5, 5, 5, 200), (0, 64, 128, 192, 193), (0, 127, 129, 129, 1000, 1300),
                                tuple(range(0, 301, 1)), (0, 0, 0, 2500, 2500)])
@pytest.mark.parametrize("D,dtype", [(5, torch.float32), (64, torch.bfloat16), (130, torch.float32)])
def test_packed(cu, D, dtype):
    _check(_inputs(cu[-1], D, len(cu) - 1, dtype, seed=len(cu) + D), cu, None)


@pytest.mark.parametrize("B,L,D,dtype", [(1800, 9, 30, torch.float32), (900, 70, 130, torch.bfloat16), (2000, 3, 7, torch.float16), (5000, 8, 64, torch.float32),
                                         (600, 33, 161, torch.float32), (20000, 1, 6, torch.float32)])
def test_a_warp_for_each_sequence(B, L, D, dtype):
    _check(_inputs(B * L, D, B, dtype, seed=B + L), range(0, B * L + 1, L), (B, L))
    if B == 1800:
        for h0, dy, dh in ((False, True, False), (True, False, True)):
            _check(_inputs(B * L, D, B, dtype, seed=3), range(0, B * L + 1, L), (B, L), h0, dy, dh)
        t = _inputs(B * L, 3 * D, B, dtype, seed=4)        # sequences apart from one another, rows off 16 bytes
        wide = [torch.zeros(B, L + 2, 3 * D + 1, device=dev)[:, 1:L + 1, 1:] for _ in range(3)]
        for v, k in zip(wide, ("x", "r", "i")):
            v.copy_(t[k].reshape(B, L, 3 * D))
        y, h = itf.gated_recurrence(*wide, t["lam"], h0=t["h0"])
        want = itf.gated_recurrence(*(v.contiguous() for v in wide), t["lam"], h0=t["h0"])
        assert_exact(y, want[0], "y")
        assert_exact(h, want[1], "h_last")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_sequences_in_segments(dtype):
    """Few features and long sequences: segments of the tokens with their states joined, dense and packed; sequences
    that start at a segment's first token, end at its last, and span several."""
    _check(_inputs(2 * 9000, 70, 2, dtype, seed=1), (0, 9000, 18000), (2, 9000))
    _check(_inputs(8191, 3, 1, dtype, seed=2), (0, 8191), (1, 8191))
    for cu in ((0, 2048, 4096, 4096, 9000, 20000), (0, 1, 2047, 2048, 19999, 20000), (0, 20000), (0, 0, 20000, 20000)):
        _check(_inputs(20000, 5, len(cu) - 1, dtype, seed=len(cu)), cu, None)
    t = _inputs(20000, 5, 3, dtype, seed=9)
    _check(t, (0, 6000, 12288, 20000), None, False, True, False)
    _check(t, (0, 6000, 12288, 20000), None, True, False, True)


def test_nan_stays_in_its_sequence_across_segments():
    cu = torch.tensor([0, 4096, 9000, 20000], dtype=torch.int32, device=dev)
    t = _inputs(20000, 6, 3, torch.float32, seed=12)
    clean, _ = itf.gated_recurrence(t["x"], t["r"], t["i"], t["lam"], h0=t["h0"], cu_seqlens=cu)
    x = t["x"].clone()
    x[4097, 2] = math.nan
    y, h = itf.gated_recurrence(x, t["r"], t["i"], t["lam"], h0=t["h0"], cu_seqlens=cu)
    bad = torch.zeros(20000, 6, dtype=torch.bool, device=dev)
    bad[4097:9000, 2] = True
    assert_exact(torch.isnan(y), bad, "NaN region")
    assert_exact(y[~bad], clean[~bad], "clean region")
    assert torch.isnan(h).sum() == 1 and torch.isnan(h[1, 2])


@pytest.mark.parametrize("seed,n,T,D", [(0, 9, 700, 40), (1, 64, 5000, 6), (2, 200, 9000, 70), (3, 1500, 3000, 3), (4, 40, 20000, 2)])
def test_packed_runs(seed, n, T, D):
    """Many sequences of uneven length, cut at random (some empty), and one that takes nearly every token."""
    rng = np.random.default_rng(seed)
    cu = [0, *np.sort(rng.integers(0, T + 1, n - 1)).tolist(), T]
    _check(_inputs(T, D, n, torch.float32, seed), cu, None)
    cu = [0] * (n // 2) + [5] * (n // 4) + [T] * (n + 1 - n // 2 - n // 4)
    _check(_inputs(T, D, n, torch.bfloat16, seed), cu, None)


@pytest.mark.parametrize("h0,dy,dh", [(False, True, False), (True, False, True), (False, True, True)])
def test_optional_parts(h0, dy, dh):
    _check(_inputs(2 * 150, 40, 2, torch.float32, seed=1), (0, 150, 300), (2, 150), h0, dy, dh)
    _check(_inputs(300, 40, 3, torch.float32, seed=2), (0, 100, 100, 300), None, h0, dy, dh)


@pytest.mark.parametrize("c", [0.0, 0.5, 50.0])
def test_decay_scale(c):
    """c = 0 keeps every state (a = 1, nothing enters); a large c forgets at once."""
    _check(_inputs(200, 33, 2, torch.float32, seed=5), (0, 100, 200), (2, 100), c=c)


def test_strided_views():
    """The three inputs as slices of one projection, the upstream gradient transposed."""
    B, L, D = 3, 70, 48
    t = _inputs(B * L, D, B, torch.float32, seed=9)
    proj = torch.stack([t[k].reshape(B, L, D) for k in ("x", "r", "i")], 2).reshape(B, L, 3 * D).requires_grad_(True)
    x, r, i = proj.split(D, -1)
    y, _ = itf.gated_recurrence(x, r, i, t["lam"])
    up = t["dy"].reshape(B, L, D).permute(2, 0, 1).contiguous().permute(1, 2, 0)
    g, = torch.autograd.grad(y, proj, up)
    y2, _ = itf.gated_recurrence(*(v.contiguous() for v in (x, r, i)), t["lam"])
    assert_exact(y, y2, "y")
    ref = orc.bwd(*(_np(t[k]) for k in ("x", "r", "i")), _np(t["lam"]), None, range(0, B * L + 1, L), _np(t["dy"]), None)
    for k, want in enumerate(ref[:3]):
        assert_close(g[..., k * D:(k + 1) * D].reshape(-1, D), want, 1e-5, "d" + "xri"[k])
    odd = torch.randn(2, 40, 3 * 21 + 1, device=dev).to(torch.bfloat16)[..., 1:]     # rows that start at odd elements
    a = odd.split(21, -1)
    lam = t["lam"][:21].contiguous()
    assert_exact(itf.gated_recurrence(*a, lam)[0], itf.gated_recurrence(*(v.contiguous() for v in a), lam)[0], "odd rows")


def test_broadcast_gradient():
    """A gate shared by every sequence (zero stride) gets the sum of its gradients."""
    t = _inputs(4 * 30, 16, 4, torch.float32, seed=4)
    gate = t["r"][:30].clone().requires_grad_(True)
    x, i = t["x"].reshape(4, 30, 16), t["i"].reshape(4, 30, 16)
    y, _ = itf.gated_recurrence(x, gate[None].expand(4, 30, 16), i, t["lam"])
    g, = torch.autograd.grad(y, gate, t["dy"].reshape(4, 30, 16))
    full = _np(gate[None].expand(4, 30, 16).reshape(-1, 16))
    _, rr, _, _, _ = orc.bwd(_np(t["x"]), full, _np(t["i"]), _np(t["lam"]), None, range(0, 121, 30), _np(t["dy"]), None)
    assert_close(g, rr.reshape(4, 30, 16).sum(0), 4e-5, "shared gate")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_closed_and_extreme_gates(dtype):
    """Gates at +-infinity and at the type's lowest value, lam from never to at once: a closed decay
    gate keeps the state exactly, gradients stay finite and match."""
    t = _inputs(160, 40, 2, dtype, seed=7)
    big = torch.finfo(dtype).max
    for k, v in enumerate((math.inf, -math.inf, -big, big, 60.0, -60.0, 100.0, -100.0)):
        t["r"][k * 5:k * 5 + 3, k::8] = v
        t["i"][80 + k * 5:80 + k * 5 + 3, k::8] = v
    t["lam"][:6] = torch.tensor([-100.0, -30.0, 0.0, 19.9, 20.1, 60.0])
    _check(t, (0, 80, 160), (2, 80))
    closed = torch.full((1, 50, 8), -math.inf, device=dev)
    h0 = torch.randn(1, 8, device=dev)
    y, h = itf.gated_recurrence(torch.randn(1, 50, 8, device=dev), closed, closed, torch.zeros(8, device=dev), h0=h0)
    assert_exact(h, h0, "kept state")
    assert_exact(y, h0[:, None].expand(1, 50, 8), "kept output")


def test_nan_stays_in_its_sequence():
    """A NaN poisons its feature from its token to its sequence's end, and nothing else."""
    cu = (0, 40, 40, 90, 300)
    t = _inputs(300, 20, 4, torch.float32, seed=11)
    clean, _ = itf.gated_recurrence(t["x"], t["r"], t["i"], t["lam"], h0=t["h0"],
                                    cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev))
    x = t["x"].clone().requires_grad_(True)
    with torch.no_grad():
        x[50, 3] = math.nan
    y, h = itf.gated_recurrence(x, t["r"], t["i"], t["lam"], h0=t["h0"], cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev))
    bad = torch.zeros(300, 20, dtype=torch.bool, device=dev)
    bad[50:90, 3] = True
    assert_exact(torch.isnan(y), bad, "NaN region")
    assert_exact(y[~bad], clean[~bad], "clean region")
    assert torch.isnan(h).sum() == 1 and torch.isnan(h[2, 3])
    dy = t["dy"].clone()
    dy[200, 5] = math.inf
    gx, = torch.autograd.grad(y, x, dy)
    assert torch.isfinite(gx[:90]).all() and not torch.isfinite(gx[200, 5])


def test_no_tokens_and_no_sequences():
    lam = torch.zeros(4, device=dev, requires_grad=True)
    h0 = torch.randn(3, 4, device=dev, requires_grad=True)
    x = torch.zeros(3, 0, 4, device=dev, requires_grad=True)
    y, h = itf.gated_recurrence(x, x, x, lam, h0=h0)
    assert y.shape == (3, 0, 4)
    assert_exact(h, h0, "state of empty sequences")
    g = torch.autograd.grad(h, [h0, lam], torch.ones_like(h))
    assert_exact(g[0], torch.ones_like(h), "dh0")
    assert_exact(g[1], torch.zeros(4), "dlam")
    e = torch.zeros(0, 5, 4, device=dev)
    y, h = itf.gated_recurrence(e, e, e, lam)
    assert y.shape == (0, 5, 4) and h.shape == (0, 4)
    p = torch.zeros(0, 4, device=dev)
    y, h = itf.gated_recurrence(p, p, p, lam, h0=h0, cu_seqlens=torch.zeros(4, dtype=torch.int32, device=dev))
    assert_exact(h, h0, "state of empty packed sequences")


def test_gradient_against_differences():
    """The kernel's gradient along a direction equals the difference quotient of the float64 oracle."""
    t = _inputs(2 * 90, 24, 2, torch.float32, seed=13)
    cu = (0, 90, 180)
    leaves = {k: (t[k].reshape(2, 90, 24) if k in "xri" else t[k]).clone().requires_grad_(True) for k in ("x", "r", "i", "lam", "h0")}
    y, h = itf.gated_recurrence(*(leaves[k] for k in ("x", "r", "i", "lam")), h0=leaves["h0"])
    grads = torch.autograd.grad([y, h], list(leaves.values()), [t["dy"].reshape(2, 90, 24), t["dh"]])
    rng = np.random.default_rng(0)
    base = {k: _np(t[k]) for k in leaves}

    def loss(v):
        yy, hh = orc.fwd(v["x"], v["r"], v["i"], v["lam"], v["h0"], cu)
        return (yy * _np(t["dy"])).sum() + (hh * _np(t["dh"])).sum()

    for k, g in zip(leaves, grads):
        direction = rng.standard_normal(base[k].shape)
        eps = 1e-5
        up, down = dict(base), dict(base)
        up[k], down[k] = base[k] + eps * direction, base[k] - eps * direction
        want = (loss(up) - loss(down)) / (2 * eps)
        g = _np(g).reshape(direction.shape)
        # fp32 gradients within 1e-5 of their largest entry, added up along the direction
        assert abs((g * direction).sum() - want) <= 1e-5 * np.abs(g).max() * np.abs(direction).sum() ** 0.5 * 10 + 1e-6


def test_gradients_repeat_bit_for_bit():
    t = _inputs(4 * 700, 96, 4, torch.float32, seed=17)

    def once():
        a = [t[k].reshape(4, 700, 96).clone().requires_grad_(True) for k in ("x", "r", "i")] + [t["lam"].clone().requires_grad_(True)]
        y, h = itf.gated_recurrence(*a)
        return torch.autograd.grad([y, h], a, [t["dy"].reshape(4, 700, 96), t["dh"]])

    for a, b in zip(once(), once()):
        assert_exact(a, b, "gradient")


def test_continues_in_pieces_and_by_steps():
    """A sequence in one call, in three calls with carried states, and token by token."""
    t = _inputs(300, 64, 1, torch.float32, seed=19)
    a = [t[k].reshape(1, 300, 64) for k in ("x", "r", "i")]
    y, h = itf.gated_recurrence(*a, t["lam"], h0=t["h0"])
    parts, state = [], t["h0"]
    for lo, hi in ((0, 1), (1, 130), (130, 300)):
        yy, state = itf.gated_recurrence(*(v[:, lo:hi] for v in a), t["lam"], h0=state)
        parts.append(yy)
    assert_close(torch.cat(parts, 1), _np(y), 1e-5, "pieces")
    state = t["h0"].clone()
    steps = [itf.gated_recurrence_step(*(v[:, k] for v in a), t["lam"], state) for k in range(300)]
    assert_close(torch.stack(steps, 1), _np(y), 1e-5, "steps")
    assert_close(state, _np(h), 1e-5, "state")


@pytest.mark.parametrize("B,D", [(1, 1), (3, 33), (64, 256), (257, 1000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_step(B, D, dtype):
    t = _inputs(B, D, B, dtype, seed=B + D)
    h = t["h0"].clone()
    y = itf.gated_recurrence_step(t["x"], t["r"], t["i"], t["lam"], h)
    ry, rh = orc.fwd(*(_np(t[k]) for k in ("x", "r", "i", "lam", "h0")), range(B + 1))
    assert_close(y, ry, TOL[dtype], "y")
    assert_close(h, rh, 1e-5, "h")
    proj = torch.cat([t["x"], t["r"], t["i"]], 1)
    h2 = t["h0"].clone()
    assert_exact(itf.gated_recurrence_step(*proj.split(D, 1), t["lam"], h2), y, "slices of a projection")


def test_other_stream():
    """Work goes to the current stream, in order with it."""
    t = _inputs(4 * 2000, 128, 4, torch.float32, seed=23)
    a = [t[k].reshape(4, 2000, 128) for k in ("x", "r", "i")]
    want, _ = itf.gated_recurrence(*a, t["lam"])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = [torch.zeros_like(v) for v in a]
        torch.cuda._sleep(20_000_000)
        for dst, src in zip(b, a):
            dst.copy_(src)
        got, _ = itf.gated_recurrence(*b, t["lam"])
    s.synchronize()
    assert_exact(got, want, "on another stream")


def test_offsets_past_32_bits():
    """Rows more than 2^31 elements apart."""
    D, gap = 64, (1 << 31) // 20 + 64
    big = torch.empty(21 * gap, dtype=torch.bfloat16, device=dev)
    x = torch.as_strided(big, (1, 21, D), (0, gap, 1))
    t = _inputs(21, D, 1, torch.bfloat16, seed=29)
    x.copy_(t["x"][None])
    y, _ = itf.gated_recurrence(x, t["r"][None], t["i"][None], t["lam"])
    want, _ = itf.gated_recurrence(t["x"][None], t["r"][None], t["i"][None], t["lam"])
    assert_exact(y, want, "far rows")
    xb = torch.as_strided(big, (2, 10, D), (11 * gap, gap, 1))
    xb.copy_(t["x"][:20].reshape(2, 10, D))
    y, _ = itf.gated_recurrence(xb, t["r"][:20].reshape(2, 10, D), t["i"][:20].reshape(2, 10, D), t["lam"])
    want, _ = itf.gated_recurrence(*(t[k][:20].reshape(2, 10, D) for k in ("x", "r", "i")), t["lam"])
    assert_exact(y, want, "far sequences")


def test_refusals():
    x, lam = torch.zeros(2, 3, 4, device=dev), torch.zeros(4, device=dev)
    cu = torch.tensor([0, 3, 6], dtype=torch.int32, device=dev)
    ok = dict(x=x, r=x, i=x, lam=lam)
    for bad, match in [(dict(r=x[:, :2]), "shape of x"), (dict(i=x.half()), "dtype of x"), (dict(lam=lam.half()), "lam"),
                       (dict(lam=lam[:3]), "lam has the wrong shape"), (dict(h0=torch.zeros(3, 4, device=dev)), "h0 has the wrong shape"),
                       (dict(cu_seqlens=cu), "with cu_seqlens"), (dict(r=x.cpu()), "device of x"),
                       (dict(x=x.double(), r=x.double(), i=x.double()), "float32, float16 or bfloat16"),
                       (dict(decay_scale=-1.0), "decay_scale"), (dict(decay_scale=math.nan), "decay_scale"),
                       (dict(x=x[0], r=x[0], i=x[0]), "must be \\(B, L, D\\)"),
                       (dict(x=x[0], r=x[0], i=x[0], cu_seqlens=cu.long()), "int32")]:
        with pytest.raises(RuntimeError, match=match):
            itf.gated_recurrence(**{**ok, **bad})
    h = torch.zeros(2, 4, device=dev)
    for bad, match in [(dict(h=h.half()), "h must be"), (dict(h=h[:1]), "h has the wrong shape"), (dict(x=x), "\\(B, D\\)")]:
        with pytest.raises(RuntimeError, match=match):
            itf.gated_recurrence_step(**{**dict(x=x[:, 0], r=x[:, 0], i=x[:, 0], lam=lam, h=h), **bad})


def test_second_derivatives_are_refused_and_unused_outputs_cost_nothing():
    x = torch.randn(1, 5, 4, device=dev, requires_grad=True)
    lam = torch.zeros(4, device=dev)
    y, h = itf.gated_recurrence(x, x.detach(), x.detach(), lam)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    y, h = itf.gated_recurrence(x, x.detach(), x.detach(), lam)
    g, = torch.autograd.grad(h.sum(), x)                   # y takes no part
    assert torch.isfinite(g).all() and not itf.gated_recurrence(x.detach(), x.detach(), x.detach(), lam)[0].requires_grad
    with torch.no_grad():
        assert not itf.gated_recurrence(x, x, x, lam)[0].requires_grad
    z = torch.randn(1, 5, 4, device=dev, requires_grad=True)
    y, _ = itf.gated_recurrence(z * 1, x.detach(), x.detach(), lam)
    w = y.detach()
    y.sum().backward()
    assert z.grad is not None and w.shape == y.shape
