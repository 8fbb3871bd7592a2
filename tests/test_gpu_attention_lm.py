"""The linear attention, the gated norm, the residual norm, the distillation loss and the sampler together, as the small
language model uses them."""
import pytest
import torch

from bc_mamba_b200 import interface as itf
from bc_mamba_b200 import recurrent_lm as lm

pytestmark = pytest.mark.gpu
dev = "cuda"


def test_a_training_step_has_gradients():
    """Every parameter gets a gradient, equal to the difference of the loss along it: central differences in float32 with
    a step of 1e-2 in a direction of unit length, truncation 1e-4 of the third derivative, rounding 1e-6 / 1e-2."""
    model = lm.AttentionLM(200, 32, 48, 2, dev, torch.float32, seed=1, heads=3, features=8)
    tokens = torch.randint(0, 200, (150,), generator=torch.Generator().manual_seed(0)).to(dev)
    cu = torch.tensor([0, 90, 90, 91, 150], dtype=torch.int32, device=dev)
    w = torch.randn(150, 200, generator=torch.Generator().manual_seed(1)).to(dev) / 150
    loss = lambda: (model.logits(tokens, cu_seqlens=cu)[0].double() * w.double()).sum()
    params = model.parameters()
    grads = torch.autograd.grad(loss(), params)
    gen = torch.Generator().manual_seed(2)
    for p, g in zip(params, grads):
        assert torch.isfinite(g).all()
        d = torch.randn(p.shape, generator=gen).to(dev)
        d /= d.norm()
        with torch.no_grad():
            p += 1e-2 * d
            up = loss()
            p -= 2e-2 * d
            down = loss()
            p += 1e-2 * d
        assert abs((up - down).item() / 2e-2 - (g * d).sum().item()) <= 2e-3 * (1 + g.norm().item())


def test_distill_step_and_generate():
    model = lm.AttentionLM(300, 32, 64, 2, dev, torch.bfloat16, seed=3)
    opt = torch.optim.AdamW(model.parameters(), lr=1e-3)
    tokens = torch.randint(0, 300, (200,), generator=torch.Generator().manual_seed(0)).to(dev)
    cu = torch.tensor([0, 150, 150, 200], dtype=torch.int32, device=dev)
    with torch.no_grad():
        top, ids = model.logits(tokens, cu_seqlens=cu)[0].float().topk(8, -1)
    loss = lm.distill_step(model, opt, tokens, cu, top, ids, torch.ones(200, device=dev))
    assert torch.isfinite(loss) and all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    out, logp = lm.generate(model, tokens[:40].view(2, 20), torch.rand(2, 5, device=dev), temperature=0.8, top_k=20)
    assert out.shape == (2, 5) and ((out >= 0) & (out < 300)).all() and torch.isfinite(logp).all()


def test_decode_gives_what_prefill_gives():
    model = lm.AttentionLM(300, 32, 40, 2, dev, torch.float32, seed=4, heads=2, features=12)
    seq = torch.randint(0, 300, (3, 90), generator=torch.Generator().manual_seed(1)).to(dev)
    with torch.no_grad():
        dense, states = model.logits(seq)
        _, some = model.logits(seq[:, :70])
        for t in range(70, 90):
            step = model.step_logits(seq[:, t], some)
            assert torch.allclose(step, dense[:, t], rtol=1e-3, atol=1e-3)
        packed, packed_states = model.logits(seq.reshape(-1), cu_seqlens=torch.tensor([0, 90, 180, 270], dtype=torch.int32, device=dev))
    assert torch.allclose(packed.reshape(3, 90, -1), dense, rtol=1e-3, atol=1e-3)
    for a, b, c in zip(states, some, packed_states):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4) and torch.allclose(a, c, rtol=1e-4, atol=1e-4)


def test_stages():
    model = lm.AttentionLM(50, 16, 16, 1, dev, torch.float32, seed=5, heads=2, features=8)
    with itf.stage_timing() as log:
        y, states = model.logits(torch.zeros(2, 9, dtype=torch.int64, device=dev))
        y.sum().backward()
        model.step_logits(torch.zeros(2, dtype=torch.int64, device=dev), states)
    torch.cuda.synchronize()
    assert [name for name, _, _ in log] == ["decay_attention_forward", "gated_norm_forward", "add_norm_forward", "add_norm_backward",
                                            "gated_norm_backward", "decay_attention_backward", "decay_attention_step",
                                            "gated_norm_forward", "add_norm_forward"]
    assert all(start.elapsed_time(end) > 0 for _, start, end in log)


def test_a_second_gradient_is_refused():
    q = torch.randn(1, 5, 2, 8, device=dev, requires_grad=True)
    w = torch.ones(8, device=dev)
    for y in (itf.decay_attention(q, q, q, torch.zeros(2, device=dev))[0], itf.gated_norm(q, q, w), itf.add_norm(q, q, w)[1]):
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(y.sum(), q, create_graph=True)


def test_two_streams_at_once_give_what_one_gives():
    """Calls that overlap share no workspace, and their blocks wait for tensor memory without holding each other up."""
    g = torch.Generator(device=dev).manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev)
    calls = [[rn(1, 6000, 2, n) / 8, rn(1, 6000, 2, n), rn(1, 6000, 4, 64), -0.1 * torch.rand(1, 6000, 4, generator=g, device=dev)] for n in (16, 64, 128)]
    for dtype in (torch.float32, torch.bfloat16):
        args = [[t.to(dtype) for t in c[:3]] + [c[3]] for c in calls]
        alone = [itf.decay_attention(*c) for c in args]
        streams = [torch.cuda.Stream() for _ in args]
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        got = []
        for _ in range(5):
            for c, s in zip(args, streams):
                with torch.cuda.stream(s):
                    got.append(itf.decay_attention(*c))
        torch.cuda.synchronize()
        for n, (y, h) in enumerate(got):
            assert torch.equal(y, alone[n % 3][0]) and torch.equal(h, alone[n % 3][1])
