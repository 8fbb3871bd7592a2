"""The linear attention at the edges of its contract, against the float64 oracle.  Tolerances as derived in
test_gpu_decay_attention.py unless a test says otherwise."""
import math

import pytest
import torch

from bc_mamba_b200 import interface as itf
from helpers import assert_close
from oracle import decay_attn as orc
from test_gpu_decay_attention import DTYPES, F32, TOL, _check, _inputs, _np

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_sequences_without_a_token(dtype):
    """The state passes through, and so does its gradient, whatever form the decays have."""
    z = lambda *s, dtype=dtype: torch.zeros(*s, device=dev, dtype=dtype)
    for shape, cu in (((2, 0), None), ((0,), z(3, dtype=torch.int32))):
        for decay in ((*shape, 3), (3,)):
            leaves = [z(*shape, 1, 4), z(*shape, 1, 4), z(*shape, 3, 5), z(*decay, dtype=torch.float32), torch.randn(2, 3, 4, 5, device=dev)]
            leaves = [x.requires_grad_(True) for x in leaves]
            y, h = itf.decay_attention(*leaves[:4], h0=leaves[4], cu_seqlens=cu)
            dh = torch.randn_like(h)
            grads = torch.autograd.grad([y, h], leaves, [torch.zeros_like(y), dh])
            assert torch.equal(grads[4], dh) and (grads[3] == 0).all()
            assert all(g.shape == x.shape for g, x in zip(grads, leaves))


@pytest.mark.parametrize("rows", [100, 1500])
@pytest.mark.parametrize("which", ["v", "k", "q", "h0", "dh", "dy"])
def test_values_next_to_the_largest_float(rows, which):
    """3.4e38 is finite, but its nearest bf16 number is not: alone, and in a sequence that is cut into items."""
    t = _inputs(rows, 1, 2, 1, 16, 24, torch.float32, seed=31)
    for name in ("q", "k", "v", "dy", "h0", "dh"):
        t[name] *= 0.05
    for at in ((0, 1, 2, 3),) if which in ("h0", "dh") else ((rows // 3, 0, 3), (rows - 30, 0, 5)):
        t[which][at] = 3.4e38
    _check(t, (0, rows), (1, rows))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 100, 1500])
def test_states_next_to_the_largest_float(rows, dtype):
    t = _inputs(rows, 1, 2, 1, 16, 24, dtype, seed=32)
    t["q"].zero_()
    t["g"] *= 1e-6
    t["h0"][0, 1, 2, 3] = -3.4e38
    y, h = itf.decay_attention(*(t[k][None] for k in ("q", "k", "v", "g")), h0=t["h0"])
    assert (y == 0).all() and torch.isfinite(h).all()
    assert_close(h, orc.fwd(*(_np(t[k]) for k in ("q", "k", "v", "g")), _np(t["h0"]), (0, rows))[1], F32, "h_last")


@pytest.mark.parametrize("cu", [None, (0, 5, 2147479550 - 1000, 2147479550)])
def test_close_to_two_to_the_31_tokens(cu):
    """The last item of a sequence ends before its span would, which passes 2^31.  One token expanded to all of them:
    y_t = sum of a^s over s <= t, which is constant from the hundredth token on."""
    rows = 2147479550
    one = torch.ones(1, 1, device=dev, dtype=torch.bfloat16)
    x = one.expand(rows, 1, 1) if cu else one.expand(1, rows, 1, 1)
    g = torch.full((1,), -0.5, device=dev)
    with torch.no_grad():
        y, h = itf.decay_attention(x, x, x, g, cu_seqlens=None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev))
    y = y.reshape(-1)
    want = 1 / (1 - math.exp(-0.5))
    starts = cu or (0, rows)
    for a, b in zip(starts, starts[1:]):
        n = min(100, b - a)
        first = torch.tensor([want * (1 - math.exp(-0.5 * (t + 1))) for t in range(n)], device=dev)
        assert ((y[a:a + n].float() - first).abs() <= TOL[torch.bfloat16] * want).all()
        for lo in range(a + n, b, 1 << 28):
            part = y[lo:min(b, lo + (1 << 28))]
            assert abs(part.min().item() - want) <= TOL[torch.bfloat16] * want and abs(part.max().item() - want) <= TOL[torch.bfloat16] * want
    assert abs(h[-1].item() - want) <= F32 * want


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_captured_step_goes_on_with_every_replay(dtype):
    """A graph of one step, its inputs rewritten between the replays: what steps without a graph give, states at an offset of
    4 bytes among others."""
    B, H, N, P = 3, 4, 24, 40
    t = _inputs(5 * B, B, H, 2, N, P, dtype, seed=91)
    q, k, v, g = (t[x].reshape(5, B, *t[x].shape[1:]) for x in ("q", "k", "v", "g"))
    for off in (0, 1):
        room = torch.zeros(t["h0"].numel() + 4, device=dev)
        h = room[off:off + t["h0"].numel()].view_as(t["h0"]).copy_(t["h0"])
        plain = t["h0"].clone()
        held = [x[0].clone() for x in (q, k, v, g)]
        itf.decay_attention_step(*held, h.clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = itf.decay_attention_step(*held, h)
        for s in range(5):
            for to, x in zip(held, (q, k, v, g)):
                to.copy_(x[s])
            graph.replay()
            want = itf.decay_attention_step(q[s], k[s], v[s], g[s], plain)
            assert_close(out, _np(want), TOL[dtype], "y")
        assert_close(h, _np(plain), F32, "h")
        assert (room[:off] == 0).all() and (room[off + h.numel():] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 100, 900])
@pytest.mark.parametrize("N", [24, 72])
def test_a_query_that_is_not_finite_without_a_gradient_of_y(rows, N, dtype):
    """No gradient of y is no contribution, not zero times the query: whole sequences and cut ones alike."""
    t = _inputs(rows, 1, 2, 1, N, 40, dtype, seed=95)
    a = [_np(t[k]) for k in ("q", "k", "v", "g", "h0")]
    want = orc.bwd(*a, (0, rows), None, _np(t["dh"]))
    t["q"][rows // 3, 0, 5], t["q"][max(0, rows - 2), 0, 7] = math.nan, math.inf
    leaves = [t[k][None].clone().requires_grad_(True) for k in ("q", "k", "v", "g")] + [t["h0"].clone().requires_grad_(True)]
    _, h = itf.decay_attention(*leaves[:4], h0=leaves[4])
    grads = torch.autograd.grad(h, leaves, t["dh"])
    assert (grads[0] == 0).all()
    for what, got, ref in zip(("dk", "dv", "dg", "dh0"), grads[1:], want[1:]):
        assert_close(got.reshape(ref.shape), ref, TOL[dtype] if what in ("dk", "dv") else F32, what)
