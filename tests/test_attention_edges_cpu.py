"""CPU tests of what the linear attention's C entries accept and refuse at the edges of their contract, before any kernel
runs: a call that passes the checks ends with a CUDA error here, where there is no GPU."""
import ctypes

import pytest

from test_attention_operators_cpu import Attn, _call


def _some(n=4):
    """n addresses that no check may look behind."""
    return [ctypes.c_void_p(256 * (1 + k)) for k in range(n)]


@pytest.mark.parametrize("heads,qk_heads", [(1, 1), (4, 2)])
def test_sequences_without_a_token_need_no_decays_gradient(heads, qk_heads):
    """Per-token decays of no token: their gradient is empty, and an empty tensor has no address."""
    dh0, ws = _some(2)
    status, text = _call("bcm_decay_attn_bwd", Attn(batch=2, seqlen=0, heads=heads, qk_heads=qk_heads, dim_k=8, dim_v=8, dh0=dh0, workspace=ws,
                                                    workspace_bytes=1 << 20))
    assert b"null pointer" not in text, text
    # one decay for each head has a gradient all the same, and a token's decay too
    for more in (dict(fixed_decay=1), dict(seqlen=1, ckpt_bytes=1 << 20, **{n: _some(1)[0] for n in ("q", "k", "v", "g", "dq", "dk", "dv", "ckpt")})):
        a = Attn(**{**dict(batch=2, seqlen=0, heads=heads, qk_heads=qk_heads, dim_k=8, dim_v=8, dh0=dh0, workspace=ws, workspace_bytes=1 << 20), **more})
        assert _call("bcm_decay_attn_bwd", a) == (1, b"decay_attn_bwd: null pointer")


@pytest.mark.parametrize("name,more", [("bcm_decay_attn_fwd", ()), ("bcm_decay_attn_bwd", ()), ("bcm_decay_attn_step", (None,))])
@pytest.mark.parametrize("buffer", ["ckpt", "workspace"])
@pytest.mark.parametrize("off", [4, 8, 12])
def test_buffers_off_16_bytes_are_refused(name, more, buffer, off):
    """Both are read 16 bytes at a time."""
    a = Attn(batch=0, seqlen=1, heads=4, qk_heads=2, dim_k=8, dim_v=8, **{buffer: ctypes.c_void_p(4096 + off)})
    assert _call(name, a, *more) == (1, f"{name[4:]}: ckpt and workspace must be aligned to 16 bytes".encode())
    setattr(a, buffer, 4096 + 16)
    assert _call(name, a, *more) == (0, b"")
