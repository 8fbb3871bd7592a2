"""The linear attention over the layouts that its smallest cases do not reach: keys of more than 64 features in sequences that
are cut or packed, values of several slices, values that are not finite in every one of them, and the precision of float32
results.  Tolerances as derived in test_gpu_decay_attention.py unless a test says otherwise."""
import math

import numpy as np
import pytest
import torch

from bc_mamba_b200 import interface as itf
from bc_mamba_b200 import recurrent_lm as lm
from helpers import assert_close, assert_exact
from oracle import decay_attn as orc
from test_gpu_decay_attention import DTYPES, F32, TOL, _check, _inputs, _np

gpu = pytest.mark.gpu
dev = "cuda"


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,P", [(72, 40), (100, 65), (128, 64), (128, 130)])
def test_many_features_cut_and_packed(N, P, dtype):
    _check(_inputs(2 * 700, 2, 2, 1, N, P, dtype, seed=N + P), (0, 700, 1400), (2, 700))
    _check(_inputs(1300, 5, 4, 2, N, P, dtype, seed=N), (0, 0, 3, 520, 584, 1300), None)
    _check(_inputs(900, 2, 3, 3, N, P, dtype, seed=P), (0, 899, 900), None, True, False, True, fixed=True)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,P", [(72, 72), (96, 24), (65, 9)])
def test_many_features_with_strides(N, P, dtype):
    """Slices of one projection on and off 16 bytes, heads before tokens: as contiguous copies, in every output."""
    B, L, H = 2, 300, 2
    t = _inputs(B * L, B, H, H, N, P, dtype, seed=41)
    q, k, v, g = (t[x].reshape(B, L, *t[x].shape[1:]) for x in ("q", "k", "v", "g"))
    dy = t["dy"].reshape(B, L, H, P)

    def both(x, up):
        leaves = [y.detach().requires_grad_(True) for y in (*x, t["h0"])]
        out = itf.decay_attention(*leaves[:4], h0=leaves[4])
        return (*out, *torch.autograd.grad(out, leaves, [up, t["dh"]]))

    want = both((q, k, v, g), dy)
    for off in (0, 1):
        wide = torch.zeros(B, L + 3, H * (2 * N + P) + 8, device=dev, dtype=dtype)[:, 2:L + 2, off:off + H * (2 * N + P)]
        wide[..., :H * N], wide[..., H * N:2 * H * N], wide[..., 2 * H * N:] = q.flatten(2), k.flatten(2), v.flatten(2)
        a, b, c = wide.split([H * N, H * N, H * P], -1)
        for got, ref in zip(both((a.unflatten(-1, (H, N)), b.unflatten(-1, (H, N)), c.unflatten(-1, (H, P)), g), dy), want):
            assert_exact(got, ref, f"slices off by {off}")
    turned = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)
    for got, ref in zip(both([turned(x) for x in (q, k, v, g)], turned(dy)), want):
        assert_exact(got, ref, "heads before tokens")


NAMES = ["q", "k", "v", "g", "dy", "h0", "dh"]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,P", [(33, 40), (64, 130), (128, 72)])
@pytest.mark.parametrize("name", NAMES)
def test_what_is_not_finite_in_a_cut_sequence(name, N, P, dtype):
    """One NaN (q, g, h0, dh) or infinity (k, v, dy) in an early, a middle or the last item of a sequence cut into four: every
    output is finite where the oracle's is, and equal there."""
    rows = 900
    t = _inputs(rows, 1, 2, 1, N, P, dtype, seed=51)
    bad = math.inf if name in ("k", "v", "dy") else math.nan
    at = (100, 440, rows - 3)[(NAMES.index(name) + N) % 3]
    if name in ("h0", "dh"):
        t[name][0, 1, N - 1, 3] = bad
    elif name == "g":
        t[name][at, 1] = bad
    else:
        t[name][at, 0, (3, P - 1)[at % 2] if name in ("v", "dy") else N - 1] = bad
    leaves = [t[k][None].clone().requires_grad_(True) for k in ("q", "k", "v", "g")] + [t["h0"].clone().requires_grad_(True)]
    y, h = itf.decay_attention(*leaves[:4], h0=leaves[4])
    grads = torch.autograd.grad([y, h], leaves, [t["dy"][None], t["dh"]])
    with np.errstate(invalid="ignore", over="ignore"):
        a = [_np(t[k]) for k in ("q", "k", "v", "g", "h0")]
        ref = orc.fwd(*a, (0, rows)) + orc.bwd(*a, (0, rows), _np(t["dy"]), _np(t["dh"]))
    for what, got, want in zip(("y", "h", "dq", "dk", "dv", "dg", "dh0"), (y, h, *grads), ref):
        got = _np(got).reshape(want.shape)
        fine = np.isfinite(want)
        assert (np.isfinite(got) == fine).all(), what
        if fine.any():
            tol = TOL[dtype] if what in ("y", "dq", "dk", "dv") else F32
            assert (np.abs(got[fine] - want[fine]) <= tol * (np.abs(want[fine]) + np.abs(want[fine]).max())).all(), what


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [1, 2, 4, 5])
def test_few_tokens_against_the_oracle(L, dtype):
    """Calls without a gradient: one decay for each head, and dropped states."""
    t = _inputs(3 * L, 3, 4, 2, 24, 40, dtype, seed=61)
    view = lambda x: x.reshape(3, L, *x.shape[1:])
    a = [_np(t[k]) for k in ("q", "k", "v")]
    cu = range(0, 3 * L + 1, L)
    for decay in (t["g"], t["g"][0], torch.where(torch.rand_like(t["g"]) < 0.4, -math.inf, t["g"])):
        g = decay if decay.dim() == 1 else view(decay)
        with torch.no_grad():
            y, h = itf.decay_attention(view(t["q"]), view(t["k"]), view(t["v"]), g, h0=t["h0"])
        ry, rh = orc.fwd(*a, _np(decay.expand(3 * L, 4)), _np(t["h0"]), cu)
        assert_close(y.reshape(ry.shape), ry, TOL[dtype], "y")
        assert_close(h, rh, F32, "h_last")


@gpu
def test_bad_offsets_stay_in_range_backward():
    """The backward reads the table that the forward reads: bounded and ascending."""
    for dtype, N in ((torch.float32, 16), (torch.float16, 72)):
        t = _inputs(300, 4, 2, 1, N, 24, dtype, seed=15)
        for cu in ((0, 500, 200, 300, 300), (-5, 100, 90, 2000, 10), (300, 0, 300, 0, 300), (7, 7, 7, 7, 7)):
            c = torch.tensor(cu, dtype=torch.int32, device=dev)
            leaves = [t[k].clone().requires_grad_(True) for k in ("q", "k", "v", "g", "h0")]
            out = itf.decay_attention(*leaves[:4], h0=leaves[4], cu_seqlens=c)
            grads = torch.autograd.grad(out, leaves, [t["dy"], t["dh"]])
            assert all(x.shape == y.shape for x, y in zip(grads, leaves))
        torch.cuda.synchronize()


# Relative size (of the root mean squares) of what float32 results may be off by.  Each is a sum of products of three-piece
# operands, whose missing piece products lie below 2^-24; a term's decay is within 2^-22 (2 units of ex2, uniform: 2^-22 /
# sqrt(3) = 1.4e-7 rms); the tensor cores cut the sum off at each of up to 12 steps of 16 (128 features, then 64 tokens), by
# half a unit of 2^-23 on average of a partial sum of about two thirds: 12 * 2^-24 * 0.67 = 4.8e-7; together 6e-7, and as
# much again for what a second product makes of the first's would be the worst of all signs.  An operand of two pieces is off
# by 2.45e-6 (the next test), two of them by 3.5e-6.
EXACT32 = 1.2e-6


def _rms(x):
    return float(np.sqrt((np.asarray(x, np.float64) ** 2).mean()))


def _pieces(x, n):
    """The sum of n bf16 pieces of float32 numbers, each the rounding of what is left."""
    out, left = np.zeros(x.shape), x.astype(np.float32)
    for _ in range(n):
        u = left.view(np.uint32)
        p = ((u + 0x7fff + ((u >> 16) & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)
        out, left = out + p, left - p
    return out


def test_the_bound_tells_two_pieces_from_three():
    rng = np.random.default_rng(0)
    for k in (16, 64, 128):
        a, b = (rng.standard_normal(s).astype(np.float32) for s in ((400, k), (k, 300)))
        exact = a.astype(np.float64) @ b
        assert _rms(_pieces(a, 2) @ _pieces(b, 3) - exact) > 1.9 * EXACT32 * _rms(exact)
        assert _rms(_pieces(a, 3) @ _pieces(b, 3) - exact) < 0.01 * EXACT32 * _rms(exact)


@gpu
@pytest.mark.parametrize("N", [16, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_float32_results_have_float32_precision(N, dtype):
    """y, both states and all gradients of float32 inputs; the states' and the decays' of 16-bit ones."""
    t = _inputs(1000, 1, 2, 1, N, 64, dtype, seed=71)
    leaves = [t[k][None].clone().requires_grad_(True) for k in ("q", "k", "v", "g")] + [t["h0"].clone().requires_grad_(True)]
    y, h = itf.decay_attention(*leaves[:4], h0=leaves[4])
    grads = torch.autograd.grad([y, h], leaves, [t["dy"][None], t["dh"]])
    a = [_np(t[k]) for k in ("q", "k", "v", "g", "h0")]
    ref = orc.fwd(*a, (0, 1000)) + orc.bwd(*a, (0, 1000), _np(t["dy"]), _np(t["dh"]))
    for what, got, want in zip(("y", "h", "dq", "dk", "dv", "dg", "dh0"), (y, h, *grads), ref):
        if dtype == torch.float32 or what in ("h", "dg", "dh0"):
            err = _rms(_np(got).reshape(want.shape) - want) / _rms(want)
            print(dtype, N, what, err)
            assert err <= EXACT32, (what, err)


@gpu
def test_decode_equals_prefill_in_float32():
    """Two layers in float32: each operator and product within F32 of its largest value, four of them a layer, and the same
    again for what the next makes of it: 16 F32."""
    model = lm.AttentionLM(300, 32, 40, 2, dev, torch.float32, seed=4, heads=2, features=12)
    seq = torch.randint(0, 300, (3, 90), generator=torch.Generator().manual_seed(1)).to(dev)
    with torch.no_grad():
        dense, states = model.logits(seq)
        _, some = model.logits(seq[:, :70])
        for t in range(70, 90):
            assert_close(model.step_logits(seq[:, t], some), _np(dense[:, t]), 16 * F32, "logits")
        packed, packed_states = model.logits(seq.reshape(-1), cu_seqlens=torch.tensor([0, 90, 180, 270], dtype=torch.int32, device=dev))
    assert_close(packed.reshape(3, 90, -1), _np(dense), 16 * F32, "packed")
    for a, b, c in zip(states, some, packed_states):
        assert_close(b, _np(a), 16 * F32, "stepped states")
        assert_close(c, _np(a), 16 * F32, "packed states")


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_an_infinite_gradient_does_not_slow_every_token_down(dtype):
    """An overflow is an ordinary event of training with a loss scale.  The chunk that has it goes token by token, some 1.4 ms;
    32 of them in a row would take 43 ms, where a clean backward takes 0.3 ms: 20 ms tell the two apart."""
    t = _inputs(19 * 2048, 19, 8, 8, 64, 64, dtype, seed=81)
    leaves = [t[k].reshape(19, 2048, *t[k].shape[1:]).requires_grad_(True) for k in ("q", "k", "v", "g")]
    dy = t["dy"].reshape(19, 2048, 8, 64).clone()
    dy[:, -1, :, 0] = math.inf
    y, h = itf.decay_attention(*leaves)
    took = []
    for _ in range(3):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        grads = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        end.record()
        torch.cuda.synchronize()
        took.append(begin.elapsed_time(end))
    assert min(took) < 20, took
    dq, dk, dv, dg = grads
    assert not torch.isfinite(dq[:, -1]).any() and torch.isfinite(dq[:, :-1]).all() and torch.isfinite(dv[..., 1:]).all()
    assert not torch.isfinite(dk).any() and not torch.isfinite(dv[..., 0]).any() and not torch.isfinite(dg[:, 1:]).any()
