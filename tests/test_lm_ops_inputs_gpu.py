"""What the training step's operators do with inputs that carry more than their values."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from llattn_b200 import clip_grad_norm_, gated_mlp, linear_cross_entropy, token_embedding, total_norm

pytestmark = pytest.mark.gpu


def randn(*shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda").to(dtype)


def calls(dtype):
    n, d, ff, v = 5, 16, 24, 50
    x, ws = randn(n, d, dtype=dtype), [randn(ff, d, dtype=dtype), randn(ff, d, dtype=dtype), randn(d, ff, dtype=dtype)]
    table, pos, ids = randn(v, d, dtype=dtype), randn(7, d, dtype=dtype), torch.randint(0, v, (2, 7), device="cuda")
    targets = torch.randint(0, ff, (n,), device="cuda")
    return {
        "gated x": (lambda t: gated_mlp(t, *ws), x), "gated w_gate": (lambda t: gated_mlp(x, t, *ws[1:]), ws[0]),
        "gated w_up": (lambda t: gated_mlp(x, ws[0], t, ws[2]), ws[1]), "gated w_down": (lambda t: gated_mlp(x, *ws[:2], t), ws[2]),
        "gated in 3 dimensions": (lambda t: gated_mlp(t, *ws), x[None]),
        "embedding": (lambda t: token_embedding(ids, t), table),
        "embedding with positions": (lambda t: token_embedding(ids, t, positions=pos), table),
        "positions": (lambda t: token_embedding(ids, table, positions=t), pos),
        "loss x": (lambda t: linear_cross_entropy(t, ws[0], targets), x),
        "loss weight": (lambda t: linear_cross_entropy(x, t, targets, reduction="sum"), ws[0]),
        "losses": (lambda t: linear_cross_entropy(t, ws[0], targets, reduction="none"), x),
    }


NAMES = ["gated x", "gated w_gate", "gated w_up", "gated w_down", "gated in 3 dimensions", "embedding", "embedding with positions",
         "positions", "loss x", "loss weight", "losses"]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_dual_tensors_are_refused(name, grad):
    f, t = calls(torch.float32)[name]
    t = t.clone().requires_grad_(grad)
    want = f(t)
    with fwAD.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError), match="forward-mode|forward mode|jvp"):
            f(fwAD.make_dual(t, torch.ones_like(t)))
        assert torch.equal(f(t), want)  # (without a tangent, inside the level)
    assert torch.equal(f(t), want)


@pytest.mark.parametrize("name", NAMES)
def test_dual_upstream_gradients_are_refused(name):
    f, t = calls(torch.bfloat16)[name]
    t = t.clone().requires_grad_(True)
    out = f(t)
    up = torch.randn_like(out)
    (want,) = torch.autograd.grad(f(t), t, up)
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, t, fwAD.make_dual(up, torch.ones_like(up)), retain_graph=True)
        assert torch.equal(torch.autograd.grad(out, t, up)[0], want)


def test_dual_gradients_are_not_clipped():
    p = torch.nn.Parameter(randn(9))
    with fwAD.dual_level():
        p.grad = fwAD.make_dual(randn(9), randn(9))
        before = fwAD.unpack_dual(p.grad).primal.clone()
        with pytest.raises(RuntimeError, match="forward-mode"):
            clip_grad_norm_([p], 0.1)
        assert torch.equal(fwAD.unpack_dual(p.grad).primal, before)
        assert abs(total_norm([p.grad]).item() / before.norm().item() - 1) < 1e-6  # (not differentiable)


def test_autocast_casts_what_it_casts_for_a_linear_layer():
    ins = randn(5, 16), randn(24, 16), randn(24, 16), randn(16, 24)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want = gated_mlp(*ins)
        assert torch.equal(gated_mlp(*(t.bfloat16() for t in ins)), want) and want.dtype == torch.bfloat16
        assert gated_mlp(*(t.half() for t in ins)).dtype == torch.bfloat16
        for k in range(4):
            for dt in (torch.float64, torch.long):
                own = [t.to(dt) if i == k else t for i, t in enumerate(ins)]
                with pytest.raises(RuntimeError, match="dtype"):
                    gated_mlp(*own)
        with pytest.raises(RuntimeError, match="dtype"):
            gated_mlp(*(t.double() for t in ins))


def pending(t):
    """-t as a view that has its sign still to be applied: what imag of a conjugate is."""
    return torch._neg_view(t)


def test_signs_that_are_still_to_be_applied():
    one, z = torch.ones(1, 1, device="cuda"), torch.complex(*torch.full((2, 1, 1), 2.0, device="cuda")).conj().imag
    assert z.is_neg() and z.item() == -2.0
    assert torch.equal(gated_mlp(z, one, one, one), gated_mlp(z.clone(), one, one, one))
    ins = [randn(5, 16), randn(24, 16), randn(24, 16), randn(16, 24)]
    for k in range(4):
        got = []
        for f in (pending, torch.neg):
            leaves = [t.clone().requires_grad_(True) for t in ins]
            y = gated_mlp(*(f(t) if i == k else t for i, t in enumerate(leaves)))
            dy = torch.ones_like(y)
            grads = torch.autograd.grad(y, leaves, f(dy))
            with torch.no_grad():
                got.append((y, gated_mlp(*(f(t) if i == k else t for i, t in enumerate(ins))), *grads))
        assert all(torch.equal(a, b) for a, b in zip(*got))
    table, pos, ids = randn(50, 16), randn(7, 16), torch.randint(0, 50, (2, 7), device="cuda")
    got = []
    for f in (pending, torch.neg):
        leaves = [t.clone().requires_grad_(True) for t in (table, pos)]
        out = token_embedding(ids, f(leaves[0]), positions=f(leaves[1]))
        got.append((out, *torch.autograd.grad(out, leaves, f(torch.ones_like(out)))))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    p = torch.nn.Parameter(randn(9))
    p.grad = pending(randn(9) * 3)
    before = p.grad.clone()
    norm = clip_grad_norm_([p], 0.5)
    assert abs(norm.item() / before.norm().item() - 1) < 1e-6
    assert torch.allclose(p.grad, before * (0.5 / before.norm()), rtol=1e-5)
