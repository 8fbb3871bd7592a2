"""Every launch of the language-model operators is a stage that stage_timing() reports, the backward passes too."""
import pytest
import torch

from bc_mamba_b200 import interface as itf

pytestmark = pytest.mark.gpu
dev = "cuda"


def _train():
    g = torch.Generator().manual_seed(0)
    x, r, i = (torch.randn(2, 40, 16, generator=g).to(dev).requires_grad_(True) for _ in range(3))
    lam = torch.zeros(16, device=dev, requires_grad=True)
    y, h = itf.gated_recurrence(x, r, i, lam)
    loss = itf.distill_topk(y.reshape(80, 16), torch.zeros(80, 2, device=dev), torch.tensor([[1, 3]], device=dev).expand(80, 2))
    loss.sum().backward()
    with torch.no_grad():
        itf.gated_recurrence_step(x[:, 0], r[:, 0], i[:, 0], lam, h)
    itf.sample_tokens(y.detach()[:, -1], torch.zeros(2, device=dev))
    return x.grad


def test_stages_of_a_training_step():
    with itf.stage_timing() as log:
        first = _train()
    torch.cuda.synchronize()
    assert [name for name, _, _ in log] == ["gated_recurrence_forward", "distill_forward", "distill_backward",
                                            "gated_recurrence_backward", "gated_recurrence_step", "sample_tokens"]
    assert all(start.elapsed_time(end) > 0 for _, start, end in log)
    n = len(log)
    assert torch.equal(_train(), first) and len(log) == n             # closed: nothing more is recorded
    with itf.stage_timing() as outer:
        with itf.stage_timing() as inner:
            _train()
        _train()
    assert len(inner) == n and len(outer) == n


def test_a_backward_that_is_refused_leaves_no_stage_open():
    z = torch.randn(3, 50, device=dev, requires_grad=True)
    with itf.stage_timing() as log:
        loss = itf.distill_topk(z, torch.zeros(3, 2, device=dev), torch.zeros(3, 2, dtype=torch.int64, device=dev))
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(loss.sum(), z, create_graph=True)
        torch.autograd.grad(itf.distill_topk(z, torch.zeros(3, 2, device=dev), torch.zeros(3, 2, dtype=torch.int64, device=dev)).sum(), z)
    assert [name for name, _, _ in log] == ["distill_forward", "distill_forward", "distill_backward"]
