"""The training operators as training programs use them: saved-tensor hooks,
checkpoints, storage that comes and goes."""

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.checkpoint import checkpoint

from llattn_b200 import linear_cross_entropy, newton_schulz
from llattn_b200.lm import LocalLatentLM, ModelConfig
from test_training_ops_gpu import BF, FP, make

pytestmark = pytest.mark.gpu


def gradients(loss, *inputs):
    return loss.detach(), *torch.autograd.grad(loss, inputs)


def churn():
    """Fills the allocator's free blocks, of every size up to 64 MB, with other values."""
    torch.cuda.synchronize()
    held = [torch.full((1 << k,), 0x7f, dtype=torch.uint8, device="cuda") for k in range(9, 27) for _ in range(4)]
    torch.cuda.synchronize()
    return held


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("how", ["save_on_cpu", "hooks", "checkpoint"])
def test_saved_tensors_that_move(how, dtype):
    """The backward of a head whose saved tensors were offloaded, copied or thrown
    away and computed again: the same bits as the plain call's."""
    n, d, v = 300, 136, 1003  # (rows of w that are copied where they are, and rows that are packed)
    for cut in (d, d - 5):
        x, w, t = make(n, d, v, dtype, ignored=0.1)
        x, w = x[:, :cut].requires_grad_(True), w[:, :cut].requires_grad_(True)
        want = gradients(linear_cross_entropy(x, w, t) * 0.7, x, w)
        f = lambda x, w: linear_cross_entropy(x, w, t)
        if how == "checkpoint":
            loss = checkpoint(f, x, w, use_reentrant=False)
        elif how == "save_on_cpu":
            with torch.autograd.graph.save_on_cpu():
                loss = f(x, w)
        else:
            with torch.autograd.graph.saved_tensors_hooks(lambda s: s.detach().clone(), lambda s: s):
                loss = f(x, w)
        held = churn()
        got = gradients(loss * 0.7, x, w)
        del held
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_weight_gathered_again_elsewhere(dtype):
    """A weight whose storage is freed after the forward and filled again before
    the backward, as sharded parameters are."""
    x, w, t = make(200, 64, 700, dtype)
    x, w = x.requires_grad_(True), torch.nn.Parameter(w)
    want = gradients(linear_cross_entropy(x, w, t), x, w)
    loss = linear_cross_entropy(x, w, t)
    values, store = w.detach().clone(), w.untyped_storage()
    size = store.size()
    torch.cuda.synchronize()
    store.resize_(0)
    held = churn()
    store.resize_(size)
    with torch.no_grad():
        w.data.copy_(values)
    got = gradients(loss, x, w)
    del held
    for a, b in zip(got, want):
        assert torch.equal(a, b)


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_dispatch_modes_see_the_operators(reduction):
    """Counters and tracers see a custom op, forward and backward; results as without them (fp32: an upstream
    gradient of 1 rounds nowhere)."""
    x, w, t = make(90, 64, 256, FP, ignored=0.1)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    f = lambda: gradients(linear_cross_entropy(x, w, t, reduction=reduction).sum(), x, w)
    want = f()
    with Seen() as seen:
        got = f()
    ours = [n for n in seen.names if n.startswith("llattn_b200.")]
    assert any(n.startswith("llattn_b200.linear_xent") for n in ours) and (reduction == "mean" or len(ours) == 2)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    g = torch.randn(48, 80, device="cuda")
    with Seen() as seen:
        outs = newton_schulz([g, g])
    assert any(n.startswith("llattn_b200.newton_schulz") for n in seen.names)
    assert torch.equal(outs[1], newton_schulz(g))


def test_fake_and_traced_gradients():
    with FakeTensorMode():
        x = torch.empty(6, 16, device="cuda", requires_grad=True)
        w = torch.empty(10, 16, device="cuda", requires_grad=True)
        t = torch.empty(6, dtype=torch.int64, device="cuda")
        for reduction in ("mean", "none"):
            dx, dw = torch.autograd.grad(linear_cross_entropy(x, w, t, reduction=reduction).sum(), (x, w))
            assert dx.shape == x.shape and dw.shape == w.shape
    x, w, t = make(20, 16, 40, FP)
    f = lambda x, w: linear_cross_entropy(x, w, t)
    graph = make_fx(f)(x, w)
    assert "llattn_b200.linear_xent" in graph.code and torch.equal(graph(x, w), f(x, w))


def test_autocast_in_fp16_takes_fp32():
    x, w, t = make(90, 64, 256, FP, ignored=0.1)
    xh, wr = x.half().requires_grad_(True), w.half().float().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.float16):
        loss = linear_cross_entropy(xh, wr, t)
    dx, dw = torch.autograd.grad(loss, (xh, wr))
    full = gradients(linear_cross_entropy(xf := xh.detach().float().requires_grad_(True), wr, t), xf, wr)
    assert torch.equal(loss, full[0]) and torch.equal(dw, full[2]) and torch.equal(dx, full[1].half())


def test_fused_loss_under_fp16_autocast_follows_the_plain_head():
    """The LM's head with a gradient scaler's autocast: fp16 logits in the plain head
    (2^-11 of logits below 8: 4e-3 of the loss at most)."""
    torch.manual_seed(0)
    m = LocalLatentLM(ModelConfig(vocab_size=512, max_seq_len=128, d_model=256, n_heads=2, n_layers=1, d_ff=512, local_window=64,
                                  latent_tokens=8, latent_d_model=64, latent_heads=2)).cuda()
    h, t = torch.randn(2, 64, 256, device="cuda"), torch.randint(0, 512, (2, 64), device="cuda")
    got = {}
    for fused in (False, True):
        m.fused_loss = fused
        with torch.autocast("cuda", dtype=torch.float16):
            got[fused] = m.loss_head(h, t).item()
    assert abs(got[True] - got[False]) <= 4e-3 * got[False]
