"""The distillation loss does not depend on an offset common to a row's
logits, nor on how low the teacher's finite logits are.

Tolerance (derived): differences within a row are taken before anything else
and are exact to 2^-24 of their size (below 40 here), so the loss stays within
the 1e-5 of max(1, loss) that it has without an offset, w and tau included.
The oracle sees the offset logits as the type holds them."""
import numpy as np
import pytest
import torch

from bc_mamba_b200 import interface as itf
from oracle import distill as orc
from test_gpu_distill import _check, _inputs, _np

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("student,teacher", [(1e3, 0.0), (1e4, 0.0), (-1e4, 0.0), (1e5, 0.0), (0.0, 1e4), (0.0, -1e5), (1e4, 1e4)])
@pytest.mark.parametrize("tau", [0.7, 1.0, 3.0])
def test_offsets(student, teacher, tau):
    z, q, ids, w, up = _inputs(9, 2000, 16, torch.float32, seed=21)
    _check(z + student, q + teacher, ids, w, tau, up)


def test_offset_over_a_cluster():
    z, q, ids, w, up = _inputs(2, 60001, 16, torch.float32, seed=22)
    _check(z + 1e4, q - 1e4, ids, w, 1.3, up)


@pytest.mark.parametrize("tau", [0.5, 1.0, 2.0])
def test_finite_teacher_logits_are_never_absent(tau):
    """Logits at the type's lowest value, finite, whatever the temperature makes of them: alone, or beside larger ones."""
    z, q, ids, w, up = _inputs(4, 500, 6, torch.float32, seed=23)
    low = torch.finfo(torch.float32).min
    q[0] = low
    q[1, 2:] = low
    q[2] = low * 0.75
    loss, dz = itf.distill_topk_with_grad(z, q, ids, weight=w, temperature=tau)
    want, dwant = orc.loss_and_grad(_np(z), _np(q), ids.cpu().numpy(), _np(w), tau)
    assert (np.abs(_np(loss) - want) <= 1e-5 * np.maximum(1.0, np.abs(want)) * max(1.0, tau * tau)).all()
    assert np.abs(_np(dz) - dwant).max() <= 1e-5 * np.abs(dwant).max()
    assert (want != 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tau", [0.25, 0.5])
def test_a_target_masked_by_the_lowest_value(dtype, tau):
    """The loss is as large as the mask times tau, which the type of the loss holds: no step on the way is larger."""
    z, q, ids, w, up = _inputs(4, 700, 6, dtype, seed=24)
    z.scatter_(1, ids[:, :1], torch.finfo(dtype).min)
    w.clamp_(max=1.0)
    assert torch.isfinite(itf.distill_topk(z, q, ids, weight=w, temperature=tau)).all()
    _check(z, q, ids, w, tau, up)
