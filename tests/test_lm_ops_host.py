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


# --- token embedding ------------------------------------------------------------------

def embed_args(**kw):
    base = dict(batch=3, length=5, d=16, dtype=_lib.F32, ids_wide=1, position_rows=8, vocab=100, padding=-1, scale=1.0, ids=1 << 20,
                w=2 << 20, ldw=16, positions=3 << 20, ldp=16, out=4 << 20, dout=5 << 20, dw=6 << 20, dpositions=7 << 20,
                workspace=None, workspace_bytes=0)
    base.update(kw)
    return _lib.EmbedArgs(*base.values())


@pytest.mark.parametrize("bad,msg", [
    (dict(batch=0), ">= 1"), (dict(length=0), ">= 1"), (dict(d=0), ">= 1"), (dict(vocab=0), ">= 1"), (dict(dtype=3), "dtype"),
    (dict(batch=1 << 20, length=1 << 11, position_rows=1 << 11), "too large"), (dict(vocab=(1 << 24) + 1), "too large"),
    (dict(padding=100), "padding"), (dict(position_rows=4), "position rows"),
])
def test_embed_refusals(bad, msg):
    L = _lib.lib()
    refused(L.llattn_embed_fwd(ctypes.byref(embed_args(**bad)), None), msg)
    refused(L.llattn_embed_bwd(ctypes.byref(embed_args(**bad)), None), msg)
    assert L.llattn_embed_workspace_bytes(ctypes.byref(embed_args(**bad))) == 0


@pytest.mark.parametrize("bad,msg", [(dict(ids=None), "NULL"), (dict(w=None), "NULL"), (dict(out=None), "NULL"),
                                     (dict(ldw=15), "row strides"), (dict(ldp=15), "row strides")])
def test_embed_forward_refusals(bad, msg):
    refused(_lib.lib().llattn_embed_fwd(ctypes.byref(embed_args(**bad)), None), msg)


@pytest.mark.parametrize("bad,msg", [(dict(dout=None), "NULL"), (dict(ids=None), "NULL"), (dict(dw=None, dpositions=None), "no output"),
                                     (dict(), "workspace of"),
                                     (dict(workspace=(1 << 30) + 8, workspace_bytes=1 << 40), "aligned")])
def test_embed_backward_refusals(bad, msg):
    refused(_lib.lib().llattn_embed_bwd(ctypes.byref(embed_args(**bad)), None), msg)


# --- norm and clipping ----------------------------------------------------------------

def clip_args(ptrs, lens, codes, **kw):
    n = len(ptrs)
    base = dict(count=n, norm_type=_lib.NORM_2, scale=1, tensors=(ctypes.c_void_p * n)(*ptrs), sizes=(ctypes.c_int64 * n)(*lens),
                dtypes=(ctypes.c_int32 * n)(*codes), max_norm=1.0, norm=1 << 20, workspace=None, workspace_bytes=0)
    base.update(kw)
    return _lib.ClipArgs(*base.values())


@pytest.mark.parametrize("lists,kw,msg", [
    (([4096], [4], [_lib.F32]), dict(count=-1), "count"), (([4096], [4], [_lib.F32]), dict(norm_type=2), "norm"),
    (([4096], [4], [_lib.F32]), dict(max_norm=-0.5), "max_norm"), (([4096], [4], [_lib.F32]), dict(max_norm=float("nan")), "max_norm"),
    (([4096], [4], [5]), {}, "dtype"), (([4096], [-1], [0]), {}, "elements"), (([None], [4], [0]), {}, "NULL"),
    (([4098], [4], [0]), {}, "aligned"), (([4097], [4], [1]), {}, "aligned"), (([4096], [4], [0]), dict(norm=None), "NULL"),
    (([4096], [4], [0]), dict(tensors=None), "NULL"), (([4096, 4104], [4, 4], [0, 0]), {}, "tensors 0 and 1 share"),
    (([8192, 4096, 8190], [4, 100, 2], [1, 1, 1]), {}, "tensors 0 and 2 share"), (([4096, 4112], [4, 4], [0, 0]), {}, "workspace of"),
    (([4096, 4096], [4, 0], [0, 0]), {}, "workspace of"), (([4096, 4096], [4, 4], [0, 0]), dict(scale=0), "workspace of"),
    (([4096], [4], [0]), dict(workspace=(1 << 30) + 8, workspace_bytes=1 << 40), "aligned"),
])
def test_clip_refusals(lists, kw, msg):
    refused(_lib.lib().llattn_clip(ctypes.byref(clip_args(*lists, **kw)), None), msg)


def test_clip_workspace_counts_what_holds_something():
    size = lambda lens: _lib.lib().llattn_clip_workspace_bytes(
        ctypes.byref(clip_args([4096 * (i + 1) for i in range(len(lens))], lens, [_lib.F32] * len(lens))))
    one = size([])
    assert one > 0 and size([0] * 5000) == one
    for n, launches in ((1, 1), (96, 1), (97, 1), (1299, 1), (1300, 1), (1301, 2), (2600, 2), (2601, 3), (3900, 3)):
        for before, after in ((0, 0), (0, 1), (7, 2000), (1300, 1300)):
            assert size([0] * before + [5] * n + [0] * after) == launches * one, (n, before, after)


@pytest.mark.parametrize("code,off", [(_lib.BF16, 1), (_lib.F32, 1), (_lib.F32, 2)])
def test_tensors_that_start_inside_an_element(code, off):
    """A pointer that no element starts at would fault in the kernels' single-element loads and stores."""
    L, size = _lib.lib(), dict(workspace=1 << 30, workspace_bytes=1 << 40)
    for name in ("x", "w_gate", "w_up", "w_down", "y"):
        bad = gated_args(dtype=code, **size)
        setattr(bad, name, getattr(bad, name) + off)
        refused(L.llattn_gated_fwd(ctypes.byref(bad), None), "aligned to its elements")
    for name in ("x", "w_gate", "w_up", "w_down", "dy", "dx", "dw_gate", "dw_up", "dw_down"):
        bad = gated_args(dtype=code, **size)
        setattr(bad, name, getattr(bad, name) + off)
        refused(L.llattn_gated_bwd(ctypes.byref(bad), None), "aligned to its elements")
    for f, names in ((L.llattn_embed_fwd, ("w", "positions", "out", "ids")), (L.llattn_embed_bwd, ("dout", "dw", "dpositions", "ids"))):
        for name in names:
            bad = embed_args(dtype=code, **size)
            setattr(bad, name, getattr(bad, name) + off)
            refused(f(ctypes.byref(bad), None), "aligned to its elements")
    for wide, step in ((1, 4), (0, 2)):
        bad = embed_args(ids_wide=wide, ids=(1 << 20) + step, **size)
        refused(L.llattn_embed_fwd(ctypes.byref(bad), None), "aligned to its elements")
        refused(L.llattn_embed_bwd(ctypes.byref(bad), None), "aligned to its elements")
    bad = clip_args([4096], [4], [code], norm=(1 << 20) + off, **size)
    refused(L.llattn_clip(ctypes.byref(bad), None), "norm is not aligned")


def test_lm_ops_on_the_cpu_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        llattn_b200.token_embedding(torch.zeros(2, 3, dtype=torch.long), torch.randn(4, 8))
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="CUDA"):
        llattn_b200.clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        llattn_b200.total_norm([p])


def test_dense_layouts():
    from llattn_b200.lm_ops import _dense
    t = torch.zeros(4, 5, 6)
    assert _dense(t) and _dense(t.permute(2, 0, 1)) and _dense(t[1:3]) and _dense(t[:, :, :1][:, :1]) is False
    assert not _dense(t[:, 1:3]) and not _dense(torch.zeros(1).expand(3)) and _dense(torch.zeros(3, 1).expand(3, 1))
    assert _dense(torch.zeros(0, 3)) and not _dense(t[..., ::2])
