"""cuda_stage as a context and as a decorator, without a GPU and with a fake of torch's NVTX calls."""
import pytest
import torch

from bc_mamba_b200 import interface as itf


def test_decorates_functions_that_call_themselves(monkeypatch):
    calls = []
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda.nvtx, "range_push", lambda name: calls.append(name))
    monkeypatch.setattr(torch.cuda.nvtx, "range_pop", lambda: calls.append("pop"))

    @itf.cuda_stage("stage")
    def down(n):
        return n if n == 0 else down(n - 1) + 1

    assert down(2) == 2 and calls == ["stage"] * 3 + ["pop"] * 3
    calls.clear()
    with pytest.raises(ValueError):
        with itf.cuda_stage("failing"):
            raise ValueError
    assert calls == ["failing", "pop"]


def test_without_a_gpu():
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is here")
    with itf.cuda_stage("nothing"):
        pass
    assert itf.cuda_stage("nothing")(lambda: 3)() == 3
