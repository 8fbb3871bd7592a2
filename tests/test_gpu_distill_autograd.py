"""What a caller may do with the tensors around the distillation loss's backward."""
import torch
import pytest

from bc_mamba_b200 import interface as itf
from helpers import assert_exact
from test_gpu_distill import _inputs

pytestmark = pytest.mark.gpu


def test_stats_lie_on_any_float():
    """The forward's stats handed to the backward at an address that is no multiple of 8."""
    z, q, ids, w, up = _inputs(5, 700, 9, torch.float32, seed=30)
    w[2] = 0
    ops = itf.load_ops()
    loss, stats = ops.distill_fwd(z, q, ids, w, 2.0, False)
    want = ops.distill_bwd(z, q, ids, w, 2.0, loss, stats, up)
    odd = torch.empty(11, device="cuda")[1:].view(5, 2)
    odd.copy_(stats)
    assert odd.data_ptr() % 8 == 4
    assert_exact(ops.distill_bwd(z, q, ids, w, 2.0, loss, odd, up), want, "gradient")


def test_the_loss_may_be_changed_in_place():
    """The backward reads nothing of the loss: masking it in place is a caller's right."""
    z, q, ids, w, up = _inputs(5, 700, 9, torch.float32, seed=31)
    mask = torch.tensor([1.0, 0.0, 1.0, 0.5, 1.0], device="cuda")
    leaf = z.clone().requires_grad_(True)
    want, = torch.autograd.grad(itf.distill_topk(leaf, q, ids, weight=w), leaf, mask)
    loss = itf.distill_topk(leaf, q, ids, weight=w)
    loss *= mask
    got, = torch.autograd.grad(loss.sum(), leaf)
    assert_exact(got, want, "gradient")
