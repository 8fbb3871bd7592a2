"""The one-token step writes its state in place: autograd learns of it, and
inputs that would need gradients are refused."""
import pytest
import torch

from bc_mamba_b200 import interface as itf
from bc_mamba_b200 import recurrent_lm as lm

pytestmark = pytest.mark.gpu
dev = "cuda"


def _rows(*shape):
    g = torch.Generator().manual_seed(1)
    return [torch.randn(*shape, generator=g).to(dev) for _ in range(3)]


def test_a_state_saved_for_backward_cannot_be_stepped_unnoticed():
    x, r, i = _rows(2, 5, 8)
    lam, state = torch.zeros(8, device=dev), torch.randn(2, 8, device=dev)
    x.requires_grad_(True)
    y, _ = itf.gated_recurrence(x, r, i, lam, h0=state)
    before = state._version
    with torch.no_grad():
        itf.gated_recurrence_step(r[:, 0], r[:, 0], i[:, 0], lam, state)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("which", ["x", "r", "i", "lam", "h"])
def test_inputs_that_need_gradients_are_refused(which):
    x, r, i = _rows(2, 8)
    t = dict(x=x, r=r, i=i, lam=torch.zeros(8, device=dev), h=torch.randn(2, 8, device=dev))
    want_h = t["h"].clone()
    want = itf.gated_recurrence_step(x, r, i, t["lam"], want_h)
    t[which].requires_grad_(True)
    kept = t["h"].detach().clone()
    with pytest.raises(RuntimeError, match="no gradient"):
        itf.gated_recurrence_step(**t)
    assert torch.equal(t["h"], kept)
    with torch.no_grad():                                 # without gradients to record, the same call runs
        y = itf.gated_recurrence_step(**t)
    assert torch.equal(y, want) and torch.equal(t["h"], want_h) and not y.requires_grad


def test_inference_tensors():
    with torch.inference_mode():
        x, r, i = _rows(2, 8)
        h = torch.zeros(2, 8, device=dev)
        lam = torch.zeros(8, device=dev)
        a = itf.gated_recurrence_step(x, r, i, lam, h)
    with torch.no_grad():
        b = itf.gated_recurrence_step(x, r, i, lam, torch.zeros(2, 8, device=dev))
        itf.gated_recurrence_step(x, r, i, lam, h)
    assert torch.equal(a, b)


def test_decode_of_the_model_records_nothing():
    """Outside no_grad, with parameters that require gradients."""
    model = lm.RecurrentLM(50, 16, 24, 1, dev, torch.float32, seed=1)
    states = [torch.zeros(3, 24, device=dev)]
    logits = model.step_logits(torch.tensor([1, 2, 3], device=dev), states)
    assert not logits.requires_grad and torch.isfinite(logits).all() and states[0].abs().max() > 0
