"""The norms of a linear-attention block at the edges of their contract, against the float64 oracle.  Tolerances as
derived in test_gpu_block_norm.py unless a test says otherwise."""
import pytest
import torch

from bc_mamba_b200 import interface as itf
from helpers import assert_close
from oracle import block_norm as orc
from test_gpu_block_norm import F32, TOL, _np, _rn

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.mark.parametrize("eps", [1e-37, 1e-39, 1e-42])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [24, 8192])
def test_rows_of_zeros_with_a_tiny_eps(eps, dtype, D):
    """eps only has to be positive: (mean x^2 + eps)^(-1/2) is 1e21 at most, its square is infinite in float32.  eps itself
    is rounded to float32 (steps of 1.4e-45 there), so the oracle gets the rounded one."""
    eps32 = torch.tensor(eps, dtype=torch.float32).double().item()
    x = torch.zeros(4, D, device=dev, dtype=dtype)
    x[2] = _rn(D, seed=1, dtype=dtype)
    x.requires_grad_(True)
    z, d, w = (_rn(*s, seed=n, dtype=t) for n, (s, t) in enumerate((((4, D), dtype), ((4, D), dtype), ((D,), torch.float32)), 2))
    none = torch.zeros_like(x)
    out = itf.gated_norm(x, z, w, groups=3 if D == 24 else 1, eps=eps)
    got = torch.autograd.grad(out, x, d)[0]
    want = orc.gated(_np(x), _np(z), _np(w), 3 if D == 24 else 1, eps32, _np(d))
    v, normed = itf.add_norm(x, none, w, eps=eps)
    got2 = torch.autograd.grad(normed, x, d)[0]
    want2 = orc.add(_np(x), _np(none), _np(w), None, eps32, None, _np(d))
    for rows in ((0, 1, 3), (2,)):                 # (the gradients at zero are 1e20 times those elsewhere)
        rows = list(rows)
        assert_close(got[rows], want[1][rows], TOL[dtype], "gated_norm")
        assert_close(got2[rows], want2[2][rows], TOL[dtype], "add_norm")
