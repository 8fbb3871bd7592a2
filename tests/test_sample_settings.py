"""Settings of one per row: every integer and floating type, values past the 32 bits that the sampler takes."""
import math

import pytest
import torch

from bc_mamba_b200 import interface as itf

MOST = 2 ** 31 - 1


@pytest.mark.parametrize("dtype,values,want", [
    (torch.int8, [-3, 0, 5, 127], [0, 0, 5, 127]), (torch.uint8, [0, 1, 50, 255], [0, 1, 50, 255]),
    (torch.int16, [-9, 0, 50, 32767], [0, 0, 50, 32767]), (torch.int64, [-1, 0, 50, 2 ** 40], [0, 0, 50, MOST]),
    (torch.float32, [-1.0, 0.0, 50.0, 3e9], [0, 0, 50, MOST]), (torch.float64, [7.0, 1e300, math.inf, math.nan], [7, MOST, MOST, 0]),
    (torch.float16, [1.0, 50.0, math.inf, -math.inf], [1, 50, MOST, 0]), (torch.bfloat16, [1.0, 3.0, 2.0 ** 40, math.nan], [1, 3, MOST, 0]),
    (torch.float32, [-3e38, math.inf, -math.inf, math.nan], [0, MOST, 0, 0])])
def test_top_k_of_any_type(dtype, values, want):
    number, got = itf._per_row(torch.tensor(values, dtype=dtype), 0, torch.int32)
    assert number == 0 and got.dtype == torch.int32 and got.tolist() == want


def test_settings_in_their_own_type_pass_unchanged():
    k, p = torch.tensor([-3, 5, 50], dtype=torch.int32), torch.tensor([0.5, math.nan])
    assert itf._per_row(k, 0, torch.int32)[1] is k and itf._per_row(p, 1.0, torch.float32)[1] is p
    assert itf._per_row(None, 1.0, torch.float32) == (1.0, None) and itf._per_row(0.3, 1.0, torch.float32) == (0.3, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int64, torch.float16, torch.float32, torch.float64])
def test_top_k_of_any_type_on_a_gpu(dtype):
    g = torch.Generator().manual_seed(1)
    x, u, k = torch.randn(4, 3000, generator=g).cuda(), torch.rand(4, generator=g).cuda(), [0, 1, 7, 100]
    want = itf.sample_tokens(x, u, top_k=torch.tensor(k, dtype=torch.int32).cuda())
    got = itf.sample_tokens(x, u, top_k=torch.tensor(k, dtype=dtype).cuda())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
