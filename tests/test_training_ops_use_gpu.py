"""The training operators as training programs use them: saved-tensor hooks,
checkpoints, storage that comes and goes."""

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.checkpoint import checkpoint

from llattn_b200 import _lib, linear_cross_entropy, newton_schulz
from llattn_b200.lm import LocalLatentLM, ModelConfig
from test_training_ops_gpu import BF, FP, make, plain, rel, spectrum

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


# --- gradients that are made with the loss and scaled in the backward -------------

# bf16: G's rounding, the stored gradient's and the scaled one's, each 2^-9 at most
THREE = 3 * 2**-9
PIECES = {BF: (8500, 65, 32771), FP: (1700, 65, 32771)}  # tokens past what is held at a time; V d odd


def pieces_case(dtype):
    n, d, v = PIECES[dtype]
    x, w, t = make(n, d, v, dtype, ignored=0.1)
    return x.requires_grad_(True), w.requires_grad_(True), t


@pytest.mark.parametrize("dtype", [BF, FP])
def test_several_pieces_with_an_upstream_gradient(dtype):
    x, w, t = pieces_case(dtype)
    _, rdx, rdw = plain(x, w, t)
    tol = THREE if dtype == BF else 1e-5
    for factor in (-1.7, 0.0, 1.0):
        dx, dw = torch.autograd.grad(linear_cross_entropy(x, w, t) * factor, (x, w))
        if factor == 0.0:
            assert not dx.any() and not dw.any()
            continue
        assert rel(dx, rdx * factor) <= tol and rel(dw, rdw * factor) <= tol
        assert not dx[t == -100].any()
    # (the last one's: factor 1) only one of them wanted
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, w.detach(), t), x)[0], dx)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x.detach(), w, t), w)[0], dw)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_several_pieces_twice_through_a_retained_graph(dtype):
    x, w, t = pieces_case(dtype)
    loss = linear_cross_entropy(x, w, t)
    first = [g.clone() for g in torch.autograd.grad(loss * -1.7, (x, w), retain_graph=True)]
    again = [g.clone() for g in torch.autograd.grad(loss * -1.7, (x, w), retain_graph=True)]
    other = torch.autograd.grad(loss * 0.5, (x, w))
    plain_ones = torch.autograd.grad(linear_cross_entropy(x, w, t), (x, w))
    for a, b, c, p in zip(first, again, other, plain_ones):
        assert torch.equal(a, b) and torch.equal(c, p * 0.5)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_several_pieces_under_hooks_and_checkpoints(dtype):
    x, w, t = pieces_case(dtype)
    f = lambda x, w: linear_cross_entropy(x, w, t)
    want = gradients(f(x, w) * 0.7, x, w)
    with torch.autograd.graph.save_on_cpu():
        offloaded = f(x, w)
    for loss in (offloaded, checkpoint(f, x, w, use_reentrant=False)):
        held = churn()
        for a, b in zip(gradients(loss * 0.7, x, w), want):
            assert torch.equal(a, b)
        del held


def test_bad_target_in_a_later_piece():
    x, w, t = pieces_case(BF)
    t[8400] = 32771
    loss = linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert math.isnan(loss.item()) and dx[8400].isnan().all() and dw.isnan().any()
    ok = torch.arange(8500, device="cuda") != 8400
    assert torch.isfinite(dx[ok]).all()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_compiled_gradients_with_an_upstream_gradient(dtype):
    x, w, t = make(90, 64, 256, dtype, ignored=0.1)
    _, rdx, rdw = plain(x, w, t)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    step = torch.compile(lambda x, w: linear_cross_entropy(x, w, t) * -1.7, backend="aot_eager", fullgraph=True)
    dx, dw = torch.autograd.grad(step(x, w), (x, w))
    tol = THREE if dtype == BF else 1e-5
    assert rel(dx, rdx * -1.7) <= tol and rel(dw, rdw * -1.7) <= tol


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("na,nb,off", [(1, 0, 0), (7, 3, 0), (4096, 5, 0), (100003, 77, 0), (1000, 999, 1), (100003, 100003, 3)])
def test_scale(dtype, na, nb, off):
    """llattn_scale: whole chunks and tails, bases without 16-byte alignment, a factor of 1; the elements around stay."""
    code = _lib.BF16 if dtype == BF else _lib.F32
    for factor in (-1.7, 0.0, 1.0):
        a, b = (torch.randn(off + m + 9, device="cuda").to(dtype) for m in (na, nb))
        f = torch.tensor(factor, device="cuda")
        want = [v.clone() for v in (a, b)]
        for v, m in zip(want, (na, nb)):
            v[off:off + m] = (v[off:off + m].float() * f).to(dtype)
        s = torch.cuda.current_stream().cuda_stream
        _lib.check(_lib.lib().llattn_scale(a[off:].data_ptr(), na, b[off:].data_ptr(), nb, code, f.data_ptr(), s), "llattn_scale")
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])


# --- CUDA graphs -------------------------------------------------------------------

def replayed(f):
    """f in a CUDA graph: what it returns, filled by each replay."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            f()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = f()
    return graph, outs


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n,d,v", [(40, 64, 256), (500, 264, 5003)])
def test_loss_in_a_cuda_graph(n, d, v, dtype):
    x, w, t = make(n, d, v, dtype, ignored=0.1)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    per = lambda: linear_cross_entropy(x.detach(), w.detach(), t, reduction="none")
    step = lambda: (*gradients(linear_cross_entropy(x, w, t) * 0.7, x, w), per())
    graph, outs = replayed(step)
    for seed in (1, 2):
        nx, nw, nt = make(n, d, v, dtype, seed=seed, ignored=0.3 * seed)
        with torch.no_grad():
            x.copy_(nx), w.copy_(nw), t.copy_(nt)
        graph.replay()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("m,n,count", [(64, 1536, 2), (256, 256, 4), (300, 777, 1)])
def test_newton_schulz_in_a_cuda_graph(m, n, count):
    gs = [spectrum(m, n, 0.5, FP, i) for i in range(count)]
    graph, outs = replayed(lambda: newton_schulz(gs))
    for g in gs:
        g.copy_(spectrum(m, n, 0.2, FP, 9) * 3)
    graph.replay()
    for o, want in zip(outs, newton_schulz(gs)):
        assert torch.equal(o, want)
