"""A wait for the tensor cores that runs out of time: every wait of the linear attention has a limit of about a second,
after which the block ends and leaves NaN, never rows that look like results.  Built here from the kernels' own header; what
is awaited is a barrier that nothing arrives at."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from bc_mamba_b200 import build

pytestmark = pytest.mark.gpu


def test_waits_end_and_are_told_of(tmp_path):
    lib = tmp_path / "wait_runs_out.so"
    subprocess.run([build.NVCC, *build.ARCH, *build.NVCC_FLAGS, "-shared", "-o", str(lib), str(Path(__file__).with_name("wait_runs_out.cu"))], check=True)
    run = ctypes.CDLL(str(lib)).run_wait
    run.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p]
    for arrive in (1, 0):
        out, told = torch.ones(40, 10, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        assert run(arrive, out.data_ptr() + 4 * 2, 10, 30, 7, told.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        end.record()
        torch.cuda.synchronize()
        assert told.item() == (0 if arrive else 256)
        nan = torch.zeros(40, 10, dtype=torch.bool, device="cuda")
        nan[:30, 2:9] = nan[0, 1] = not arrive
        assert torch.equal(torch.isnan(out), nan) and (out[~nan] == 1).all()
        assert begin.elapsed_time(end) < (100 if arrive else 10000)
