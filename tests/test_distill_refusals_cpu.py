"""Arguments that the distillation entry points refuse before anything reaches a GPU."""
import ctypes

import pytest

import bc_mamba_b200


class Args(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int64), ("vocab", ctypes.c_int64), ("k", ctypes.c_int64), ("dtype", ctypes.c_int),
                ("teacher_dtype", ctypes.c_int), ("ids_are_int64", ctypes.c_int), ("temperature", ctypes.c_float),
                ("logits", ctypes.c_void_p), ("logits_stride", ctypes.c_int64), ("teacher_logits", ctypes.c_void_p),
                ("teacher_ids", ctypes.c_void_p), ("weight", ctypes.c_void_p), ("loss", ctypes.c_void_p), ("stats", ctypes.c_void_p),
                ("dloss", ctypes.c_void_p), ("dlogits", ctypes.c_void_p)]


def _call(name, **kw):
    lib = bc_mamba_b200.load_library()
    lib.bcm_last_error.restype = ctypes.c_char_p
    f = getattr(lib, name)
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]
    args = Args(rows=0, vocab=10, k=2, temperature=1.0)
    for k, v in kw.items():
        setattr(args, k, v)
    return f(ctypes.byref(args), None), lib.bcm_last_error()


@pytest.mark.parametrize("name", ["bcm_distill_fwd", "bcm_distill_bwd", "bcm_distill_fwd_grad"])
def test_temperatures(name):
    """Of one whose reciprocal is no finite number, every exponent would be 0 times infinity."""
    for tau in (1e-40, 1e-44, 4e-39, 0.0, -1.0, float("inf"), float("nan")):
        status, why = _call(name, temperature=tau)
        assert status == 1 and b"temperature" in why, tau
    for tau in (1e-38, 0.5, 1e18):
        assert _call(name, temperature=tau) == (0, b"")
