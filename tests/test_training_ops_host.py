"""The training operators' host side without a GPU: what the backward of
linear_cross_entropy hands to the C calls, with stand-ins for them."""

import contextlib
import ctypes
import gc
import math
import random

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils.checkpoint import checkpoint

import llattn_b200
from llattn_b200 import _lib, training_ops

KEPT = 4096


class StandIn:
    """llattn_xent by its arguments alone: records the addresses that each call
    is given, and at the gradients' which of them belong to a live tensor."""

    def __init__(self):
        self.calls = []

    def llattn_xent_workspace_bytes(self, ref):
        return 256 if ref._obj.stage == _lib.XENT_GRADS else KEPT

    def llattn_xent(self, ref, stream):
        a = ref._obj
        if a.stage == _lib.XENT_LOSS:
            ctypes.memset(a.loss, 0, 4)
            self.calls.append(("loss", a.workspace))
        else:
            assert a.stage == _lib.XENT_GRADS
            live = {t.data_ptr() for t in gc.get_objects() if type(t) in (torch.Tensor, torch.nn.Parameter)}
            self.calls.append(("grads", a.kept, a.kept in live, a.w in live, a.targets in live, a.w))
            for p, n in ((a.dx, a.tokens * a.d), (a.dw, a.vocab * a.d)):
                if p:
                    ctypes.memset(p, 0, 4 * n)
        return 0


@pytest.fixture
def calls(monkeypatch):
    fake = StandIn()
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    monkeypatch.setattr(training_ops, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(training_ops, "_stream", lambda t: 0)
    monkeypatch.setattr(training_ops, "_check_xent", lambda *a: None)
    return fake.calls


def copying_hooks():
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), lambda t: t)


def case():
    x = torch.randn(6, 16, requires_grad=True)
    w = torch.nn.Parameter(torch.randn(10, 16))
    return x, w, torch.arange(6)


@pytest.mark.parametrize("how", ["plain", "hooks", "checkpoint"])
def test_backward_reads_live_memory_only(calls, how):
    """The kept workspace belongs to the graph's saved tensors, which hooks (an
    offload, a checkpoint) may replace: the backward takes it from there."""
    x, w, t = case()
    f = lambda x, w: llattn_b200.linear_cross_entropy(x, w, t)
    if how == "hooks":
        with copying_hooks():
            loss = f(x, w)
    elif how == "checkpoint":
        loss = checkpoint(f, x, w, use_reentrant=False)
    else:
        loss = f(x, w)
    gc.collect()
    loss.backward()
    grads = [c for c in calls if c[0] == "grads"]
    assert len(grads) == 1 and grads[0][2:5] == (True, True, True), calls
    if how == "checkpoint":  # computed again, and taken from there
        assert [c[0] for c in calls] == ["loss", "loss", "grads"] and grads[0][1] == calls[1][1]


def test_backward_follows_the_weight_to_its_new_memory(calls):
    """A weight whose memory is given up between forward and backward and gathered
    again elsewhere (sharded parameters) is read where it is then."""
    x, w, t = case()
    loss = llattn_b200.linear_cross_entropy(x, w, t)
    other = torch.randn(10, 16)
    old = w.data_ptr()
    w.data = other
    assert w.data_ptr() != old
    loss.backward()
    assert calls[-1][0] == "grads" and calls[-1][5] == other.data_ptr(), calls


def test_backward_computes_again_what_does_not_fit_its_inputs(calls, monkeypatch):
    """A saved weight that comes back in another layout than it was kept for
    (its packed copy is, or is not, part of the workspace): a loss of its own."""
    x, w, t = case()
    loss = llattn_b200.linear_cross_entropy(x, w, t)
    monkeypatch.setattr(StandIn, "llattn_xent_workspace_bytes",
                        lambda self, ref: 256 if ref._obj.stage == _lib.XENT_GRADS else 2 * KEPT)
    loss.backward()
    assert [c[0] for c in calls] == ["loss", "loss", "grads"] and calls[2][1] == calls[1][1] and calls[2][2]


# --- who watches -----------------------------------------------------------------

def fake_case(grads=False):
    f = lambda *s: torch.empty(*s, device="cuda", dtype=torch.bfloat16, requires_grad=grads)
    return f(6, 16), f(10, 16), torch.empty(6, dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_fake_tensors_go_through_the_custom_ops(reduction):
    with FakeTensorMode():
        x, w, t = fake_case()
        out = llattn_b200.linear_cross_entropy(x, w, t, reduction=reduction)
        assert out.shape == ((6,) if reduction == "none" else ()) and out.dtype == torch.float32
        x, w, t = fake_case(True)
        out = llattn_b200.linear_cross_entropy(x, w, t, reduction=reduction)
        assert out.requires_grad
        g = llattn_b200.newton_schulz(fake_case()[0].float())
        assert g.shape == (6, 16) and g.dtype == torch.bfloat16
        for o, shape in zip(llattn_b200.newton_schulz([x, w, x]), ((6, 16), (10, 16), (6, 16))):
            assert o.shape == shape and o.dtype == torch.bfloat16


# --- workspaces, from the host --------------------------------------------------

def sizes(n, d, v, dtype=_lib.BF16, stage=_lib.XENT_GRADS):
    outs = dict(loss=None, dx=1 << 21, dw=1 << 22, kept=1 << 23) if stage == _lib.XENT_GRADS else dict(dx=1 << 21, dw=1 << 22)
    a = _lib.XentArgs(n, d, v, dtype, _lib.XENT_MEAN, -100, 1 << 24, d, 1 << 25, d, 1 << 26, None, None)
    for k, val in {**outs, "stage": stage}.items():
        setattr(a, k, val)
    return _lib.lib().llattn_xent_workspace_bytes(ctypes.byref(a))


@pytest.mark.parametrize("dtype", [_lib.BF16, _lib.F32])
def test_small_calls_take_small_workspaces(dtype):
    """Nothing is reserved for sums that no product of these sizes splits."""
    assert sizes(1, 64, 97, dtype) <= 256 and sizes(512, 128, 128, dtype) <= 256
    assert sizes(1, 64, 97, dtype, _lib.XENT_ALL) <= 1 << 18
    assert sizes(512, 128, 128, dtype, _lib.XENT_ALL) <= 3 << 20  # 512 x 128 of x in planes, exponentials, G


SHAPES = {0: (128, 32), 1: (128, 128), 2: (256, 256), 3: (256, 512), 4: (128, 64)}


def split_bytes(m, n, k, shape, sms=148):
    """Partial sums of the product's last wave (mm_plan's rule)."""
    bm, bn = SHAPES[shape]
    units = sms // 2 if shape in (2, 3) else sms
    total, steps = -(-m // bm) * -(-n // bn), -(-k // 64)
    tail = total % units
    block = 205 * (bm * bn // 1024) // 64
    best, cost = 1, None
    for s in range(1, 33):
        if s > 1 and (steps < 8 * s or tail * s > 4 * units):
            break
        c = 1024 * -(-tail * s // units) * (-(-steps // s) + 6) + (block * tail * s if s > 1 else 0)
        if cost is None or c < cost:
            best, cost = s, c
    return 4 * bm * bn * tail * best if best > 1 else 0


def test_workspace_holds_every_split():
    """Whatever the shape that a product runs in and however few tokens count (the
    device cuts dx's rows and dw's sums to them)."""
    rng = random.Random(0)
    for _ in range(300):
        n, d, v = (int(math.exp(rng.uniform(math.log(a), math.log(b)))) for a, b in ((1, 8000), (1, 5000), (1, 32000)))
        have = sizes(n, d, v)
        for counted in {0, 1, n, n // 2, rng.randint(0, n), rng.randint(0, n)}:
            for shape in SHAPES:
                assert split_bytes(counted, d, v, shape) <= have, (n, d, v, counted, shape)
                assert split_bytes(v, d, counted, shape) <= have, (n, d, v, counted, shape)


@pytest.mark.skipif(torch.cuda.is_available(), reason="a device whose clusters fit")
@pytest.mark.parametrize("rows,cols", [(8, 8), (64, 300), (64, 1536), (3000, 48)])
def test_matrices_without_a_cluster_get_the_general_kernels(rows, cols):
    """Where a matrix's cluster of CTAs does not fit the device (here there is
    none), the call is planned for the kernels that need no cluster."""
    for dtype in (_lib.BF16, _lib.F32):
        ptrs = (ctypes.c_void_p * 1)(1 << 20)
        a = _lib.OrthArgs(rows, cols, 1, 5, dtype, 3.4, -4.7, 2.0, 1e-7, ptrs, 1 << 21, None, 0)
        up = (cols + 7) // 8 * 8
        assert _lib.lib().llattn_orth_workspace_bytes(ctypes.byref(a)) >= 3 * 2 * rows * up


def test_stage_loss_refuses_row_gradients():
    """grad_rows goes with reduction none, which has no stages: given to a stage's
    loss it would weight the exponentials that are kept."""
    a = _lib.XentArgs(10, 64, 100, _lib.BF16, _lib.XENT_MEAN, -100, 1 << 20, 64, 2 << 20, 64, 3 << 20, 1 << 22, None, 4 << 20)
    a.stage = _lib.XENT_LOSS
    L = _lib.lib()
    assert L.llattn_xent(ctypes.byref(a), None) != 0
    assert "grad_rows" in L.llattn_last_error().decode()
