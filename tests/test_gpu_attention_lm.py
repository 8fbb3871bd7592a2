"""The linear attention, the gated norm, the residual norm, the distillation loss and the sampler together, as the small
language model uses them."""
import pytest
import torch

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
