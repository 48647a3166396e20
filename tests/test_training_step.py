"""The training step with linear_cross_entropy and Muon: the LM's switches, their
agreement with the plain step, and the C entry points' refusals (no GPU)."""

import ctypes
import importlib.util
import os

import pytest
import torch

import llattn_b200
from llattn_b200 import _lib
from llattn_b200.lm import LocalLatentLM, ModelConfig, build_optimizer, train_step

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def small_cfg(**kw):
    base = dict(vocab_size=512, max_seq_len=256, d_model=256, n_heads=2, n_layers=2, d_ff=512, local_window=64,
                latent_tokens=8, latent_d_model=64, latent_heads=2)
    return ModelConfig(**{**base, **kw})


# --- host side ---------------------------------------------------------------

def test_optimizer_for_hidden_matrices():
    m = LocalLatentLM(small_cfg())
    opt = build_optimizer(m, lr=2e-3, hidden="muon")
    muon, adamw = opt.optimizers
    inside = {id(p) for g in muon.param_groups for p in g["params"]}
    for name, p in m.named_parameters():
        assert (id(p) in inside) == ("blocks." in name and p.dim() == 2 and min(p.shape) > 1), name
    outside = [id(p) for g in adamw.param_groups for p in g["params"]]
    assert not inside & set(outside) and len(inside) + len(outside) == len(list(m.parameters()))
    assert all(g["lr"] == 2e-3 for g in opt.param_groups)
    with pytest.raises(ValueError, match="hidden"):
        build_optimizer(m, hidden="sgd")


def test_muon_refusals():
    p = torch.nn.Parameter(torch.zeros(4, 4))
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(steps=0)):
        with pytest.raises(ValueError, match="hyper-parameters"):
            llattn_b200.Muon([p], **kw)
    with pytest.raises(ValueError, match="matrices"):
        llattn_b200.Muon([torch.nn.Parameter(torch.zeros(4))])


def xent_args(**kw):
    base = dict(tokens=10, d=64, vocab=100, dtype=_lib.BF16, reduction=_lib.XENT_MEAN, ignore_index=-100, x=1 << 20, ldx=64,
                w=2 << 20, ldw=64, targets=3 << 20, grad_rows=None, losses=None, loss=4 << 20, dx=None, dw=None,
                workspace=None, workspace_bytes=0)
    base.update(kw)
    return _lib.XentArgs(*base.values())


@pytest.mark.parametrize("bad,msg", [
    (dict(tokens=0), "tokens"), (dict(d=0), ">= 1"), (dict(vocab=0), ">= 1"), (dict(dtype=7), "dtype"),
    (dict(reduction=9), "reduction"), (dict(ldx=63), "row strides"), (dict(ldw=10), "row strides"),
    (dict(vocab=1 << 22), "too large"), (dict(x=None), "NULL"), (dict(targets=None), "NULL"), (dict(loss=None), "no output"),
    (dict(reduction=_lib.XENT_NONE), "scalar loss"), (dict(dx=1 << 21, losses=1 << 22), "without gradients"),
    (dict(dx=1 << 21, grad_rows=1 << 22), "grad_rows"), (dict(), "workspace"),
    (dict(workspace=257, workspace_bytes=1 << 40), "256-byte"),
])
def test_xent_refusals_on_the_host(bad, msg):
    L = _lib.lib()
    assert L.llattn_xent(ctypes.byref(xent_args(**bad)), None) != 0
    assert msg in L.llattn_last_error().decode()


@pytest.mark.parametrize("bad,msg", [
    (dict(stage=3), "unknown stage"), (dict(stage=-1), "unknown stage"),
    (dict(stage=_lib.XENT_LOSS, reduction=_lib.XENT_NONE), "mean and sum"),
    (dict(stage=_lib.XENT_LOSS, dx=1 << 21), "loss only"), (dict(stage=_lib.XENT_LOSS, losses=1 << 22), "loss only"),
    (dict(stage=_lib.XENT_GRADS, dx=1 << 21, kept=1 << 23), "kept workspace"),
    (dict(stage=_lib.XENT_GRADS, loss=None, kept=1 << 23), "kept workspace"),
    (dict(stage=_lib.XENT_GRADS, loss=None, dx=1 << 21), "kept workspace"),
    (dict(stage=_lib.XENT_GRADS, loss=None, dx=1 << 21, kept=1), "kept workspace"),
    (dict(factor=1 << 23), "go with stage grads"), (dict(stage=_lib.XENT_LOSS, kept=1 << 23), "go with stage grads"),
    (dict(stage=_lib.XENT_LOSS, tokens=100000, vocab=1 << 20), "one piece"),
    (dict(stage=_lib.XENT_LOSS), "workspace of"), (dict(stage=_lib.XENT_GRADS, loss=None, dw=1 << 21, kept=1 << 23), "workspace of"),
])
def test_xent_stage_refusals_on_the_host(bad, msg):
    L = _lib.lib()
    args = xent_args(**{k: v for k, v in bad.items() if k not in ("stage", "factor", "kept")})
    args.stage, args.factor, args.kept = bad.get("stage", _lib.XENT_ALL), bad.get("factor"), bad.get("kept")
    assert L.llattn_xent(ctypes.byref(args), None) != 0
    assert msg in L.llattn_last_error().decode()


def test_xent_workspace_is_bounded():
    """Half a GiB of exponentials whatever the number of tokens; what grows
    with them is their packed rows and a few words each."""
    L = _lib.lib()
    size = lambda n, **kw: L.llattn_xent_workspace_bytes(ctypes.byref(xent_args(
        tokens=n, d=1536, vocab=32000, ldx=1536, ldw=1536, dx=1 << 20, dw=1 << 21, **kw)))
    a, b = size(32768), size(65536)
    assert a < 2 << 30 and b - a <= 32768 * (2 * 1536 + 32)
    assert size(0) == 0 and size(100, dtype=9) == 0


@pytest.mark.parametrize("bad,msg", [
    (dict(rows=0), ">= 1"), (dict(count=0), ">= 1"), (dict(steps=0), "steps"), (dict(steps=65), "steps"), (dict(dtype=3), "dtype"),
    (dict(a=17.0), "coefficients"), (dict(b=float("nan")), "coefficients"), (dict(eps=-1.0), "eps"), (dict(out=None), "NULL"),
    (dict(), "workspace"), (dict(rows=1 << 21), "too large"),
])
def test_orth_refusals_on_the_host(bad, msg):
    ptrs = (ctypes.c_void_p * 2)(1 << 20, 2 << 20)
    base = dict(rows=256, cols=512, count=2, steps=5, dtype=_lib.BF16, a=3.4, b=-4.7, c=2.0, eps=1e-7, g=ptrs, out=3 << 20,
                workspace=None, workspace_bytes=0)
    base.update(bad)
    L = _lib.lib()
    assert L.llattn_orth(ctypes.byref(_lib.OrthArgs(*base.values())), None) != 0
    assert msg in L.llattn_last_error().decode()


def test_orth_null_matrix_and_scale_refusals():
    ptrs = (ctypes.c_void_p * 2)(1 << 20, None)
    L = _lib.lib()
    assert L.llattn_orth(ctypes.byref(_lib.OrthArgs(8, 8, 2, 5, _lib.F32, 3.4, -4.7, 2.0, 1e-7, ptrs, 1 << 21, None, 0)), None) != 0
    assert "matrix 1" in L.llattn_last_error().decode()
    assert L.llattn_scale(None, 4, None, 0, _lib.F32, 1 << 20, None) != 0
    assert L.llattn_scale(1 << 20, 4, None, 0, 9, 1 << 21, None) != 0


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        llattn_b200.linear_cross_entropy(torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        llattn_b200.newton_schulz(torch.zeros(4, 8))


# --- on the GPU ----------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("autocast", [True, False])
def test_fused_loss_and_its_gradients_match_the_plain_head(autocast):
    """The same model, tokens and weights through both heads. fp32: 1e-4 of
    every gradient's norm (the attention block's own fp32 tolerance); bf16
    autocast: 2e-2, the two heads round G and the logits at different places."""
    torch.manual_seed(0)
    m = LocalLatentLM(small_cfg()).cuda()
    gen = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 512, (2, 129), generator=gen).cuda()
    got = {}
    for fused in (False, True):
        m.fused_loss = fused
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            loss = m(ids[:, :-1], ids[:, 1:])
        loss.backward()
        got[fused] = loss.item(), {n: p.grad.clone() for n, p in m.named_parameters()}
    tol = 2e-2 if autocast else 1e-4
    assert abs(got[True][0] - got[False][0]) <= tol * got[False][0]
    for n, g in got[False][1].items():
        assert (got[True][1][n] - g).norm() <= tol * g.norm() + 1e-12, n


@pytest.mark.gpu
def test_training_step_with_both_operators_learns():
    torch.manual_seed(0)
    m = LocalLatentLM(small_cfg()).cuda()
    m.fused_loss = True
    opt = build_optimizer(m, lr=1e-3, hidden="muon")
    gen = torch.Generator().manual_seed(0)
    start = torch.randint(0, 512, (4, 1), generator=gen)
    seq = ((start + torch.arange(129)) % 512).cuda()
    losses = [train_step(m, opt, seq[:, :-1], seq[:, 1:]).item() for _ in range(30)]
    assert all(map(lambda v: v == v, losses)) and losses[-1] < 0.5 * losses[0], losses
    # saved and loaded, the optimisers continue the same run
    state = opt.state_dict()
    opt2 = build_optimizer(m, lr=1e-3, hidden="muon")
    opt2.load_state_dict(state)
    for a, b in zip(opt.param_groups, opt2.param_groups):
        assert a["lr"] == b["lr"] and len(a["params"]) == len(b["params"])


@pytest.mark.gpu
def test_compiled_loss_head_matches_eager():
    torch.manual_seed(0)
    m = LocalLatentLM(small_cfg()).cuda()
    m.fused_loss = True
    x = torch.randn(2, 64, 256, device="cuda")
    t = torch.randint(0, 512, (2, 64), device="cuda")
    got = []
    for head in (m.loss_head, torch.compile(m.loss_head, backend="aot_eager", fullgraph=True)):
        m.zero_grad(set_to_none=True)
        xr = x.clone().requires_grad_(True)
        loss = head(xr, t)
        loss.backward()
        got.append((loss.detach(), xr.grad, m.lm_head.weight.grad.clone()))
    for a, b in zip(*got):
        assert (a - b).norm() <= 1e-5 * b.norm()


@pytest.mark.gpu
def test_example_runs():
    spec = importlib.util.spec_from_file_location("train_lm_example", os.path.join(ROOT, "examples", "train_lm.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses = mod.main(["--steps", "6", "--layers", "1"])
    assert len(losses) == 6 and losses[-1] < losses[0]
