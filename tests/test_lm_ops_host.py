"""The host side of the language model's operators without a GPU: refusals and sizes of the C entry points, what the
public calls say of bad arguments."""

import ctypes

import pytest
import torch

import llattn_b200
from llattn_b200 import _lib


def refused(rc, msg):
    assert rc != 0
    assert msg in _lib.lib().llattn_last_error().decode(), _lib.lib().llattn_last_error().decode()


# --- gated feed-forward block ---------------------------------------------------

def gated_args(**kw):
    base = dict(tokens=10, d=64, ff=96, d_out=40, dtype=_lib.BF16, activation=_lib.ACT_SILU, x=1 << 20, ldx=64, w_gate=2 << 20,
                ldg=64, w_up=3 << 20, ldu=64, w_down=4 << 20, ldd=96, y=5 << 20, kept=6 << 20, dy=7 << 20, lddy=40, dx=8 << 20,
                dw_gate=9 << 20, dw_up=10 << 20, dw_down=11 << 20, workspace=None, workspace_bytes=0)
    base.update(kw)
    return _lib.GatedArgs(*base.values())


@pytest.mark.parametrize("bad,msg", [
    (dict(tokens=0), ">= 1"), (dict(d=0), ">= 1"), (dict(ff=-1), ">= 1"), (dict(d_out=0), ">= 1"), (dict(dtype=5), "dtype"),
    (dict(activation=2), "activation"), (dict(ldx=63), "row strides"), (dict(ldg=1), "row strides"),
    (dict(ldu=0), "row strides"), (dict(ldd=95), "row strides"), (dict(ff=1 << 21, ldd=1 << 21), "too large"),
    (dict(tokens=1 << 27), "too large"), (dict(x=None), "NULL"), (dict(w_up=None), "NULL"), (dict(y=None), "NULL"),
    (dict(), "workspace of"),
])
def test_gated_refusals(bad, msg):
    refused(_lib.lib().llattn_gated_fwd(ctypes.byref(gated_args(**bad)), None), msg)


@pytest.mark.parametrize("bad,msg", [
    (dict(lddy=39), "row strides"), (dict(dy=None), "NULL"), (dict(kept=None), "NULL"),
    (dict(dx=None, dw_gate=None, dw_up=None, dw_down=None), "no output"), (dict(), "workspace of"),
    (dict(workspace=1 << 30), "workspace of"), (dict(workspace=(1 << 30) + 64, workspace_bytes=1 << 40), "aligned"),
    (dict(workspace=1 << 30, workspace_bytes=1 << 40, kept=(6 << 20) + 128), "aligned"),
])
def test_gated_backward_refusals(bad, msg):
    refused(_lib.lib().llattn_gated_bwd(ctypes.byref(gated_args(**bad)), None), msg)


def test_gated_null_args_and_sizes():
    L = _lib.lib()
    assert L.llattn_gated_fwd(None, None) == 1 and L.llattn_gated_bwd(None, None) == 1
    assert L.llattn_gated_workspace_bytes(ctypes.byref(gated_args(d=0)), 0) == 0
    assert L.llattn_gated_kept_bytes(ctypes.byref(gated_args(ff=0))) == 0
    size = lambda b, **kw: L.llattn_gated_workspace_bytes(ctypes.byref(gated_args(**kw)), b)
    aligned = size(0)
    # an unaligned operand is packed: its rows and no more (256-byte steps)
    assert size(0, w_gate=(2 << 20) + 2) - aligned == 96 * 64 * 2
    assert size(0, ldx=65) - aligned == -(-10 * 64 * 2 // 256) * 256
    # the backward holds what its outputs need
    assert size(1, dx=None, dw_gate=None, dw_up=None) < size(1, dw_down=None) < size(1)
    # what is kept: 4 bytes an inner column and token and 2 a block of 32, or 8 bytes
    from llattn_b200 import lm_ops
    for n, ff in ((1, 1), (10, 96), (33, 97), (4095, 3749)):
        for code, dt in ((_lib.BF16, torch.bfloat16), (_lib.F32, torch.float32)):
            got = L.llattn_gated_kept_bytes(ctypes.byref(gated_args(tokens=n, ff=ff, ldd=ff, dtype=code)))
            assert got == lm_ops._kept_bytes(n, ff, dt)
            assert got >= n * ff * (4 if dt == torch.bfloat16 else 8)


def test_gated_mlp_on_the_cpu_is_refused():
    x, w = torch.randn(3, 8), torch.randn(8, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        llattn_b200.gated_mlp(x, w, w, w)
    with pytest.raises(RuntimeError, match="activation"):
        llattn_b200.gated_mlp(x, w, w, w, activation="tanh")
