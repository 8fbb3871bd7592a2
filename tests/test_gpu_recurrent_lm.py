"""The recurrence, the distillation loss and the sampler together, as the small
language model uses them."""
import pytest
import torch

from bc_mamba_b200 import recurrent_lm as lm

pytestmark = pytest.mark.gpu
dev = "cuda"


def test_distillation_lowers_the_loss():
    teacher = lm.RecurrentLM(500, 32, 48, 2, dev, torch.float32, seed=1)
    student = lm.RecurrentLM(500, 32, 48, 2, dev, torch.float32, seed=2)
    opt = torch.optim.AdamW(student.parameters(), lr=3e-3)
    tokens = torch.randint(0, 500, (400,), generator=torch.Generator().manual_seed(0)).to(dev)
    cu = torch.tensor([0, 150, 150, 151, 400], dtype=torch.int32, device=dev)
    weight = torch.ones(400, device=dev)
    weight[380:] = 0
    with torch.no_grad():
        top, ids = teacher.logits(tokens, cu_seqlens=cu)[0].topk(12, -1)
    losses = [float(lm.distill_step(student, opt, tokens, cu, top, ids, weight)) for _ in range(40)]
    assert losses[-1] < 0.7 * losses[0]
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in student.parameters())


def test_decode_gives_what_prefill_gives():
    """Greedy tokens from prefill + steps equal those of prefills of ever longer prompts, and a packed
    pass equals its documents one by one."""
    model = lm.RecurrentLM(300, 32, 40, 2, dev, torch.float32, seed=3)
    prompts = torch.randint(0, 300, (3, 17), generator=torch.Generator().manual_seed(1)).to(dev)
    u = torch.full((3, 9), 0.5, device=dev)
    got, logp = lm.generate(model, prompts, u, temperature=0.0)
    seq = prompts
    with torch.no_grad():
        for _ in range(9):
            seq = torch.cat([seq, model.logits(seq)[0][:, -1].argmax(-1, keepdim=True)], 1)
        assert got.tolist() == seq[:, 17:].tolist() and (logp == 0).all()
        cu = torch.tensor([0, 26, 52, 78], dtype=torch.int32, device=dev)
        packed, states = model.logits(seq.reshape(-1), cu_seqlens=cu)
        dense, dense_states = model.logits(seq)
    assert torch.allclose(packed.reshape(3, 26, -1), dense, rtol=1e-4, atol=1e-4)
    for a, b in zip(states, dense_states):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)
