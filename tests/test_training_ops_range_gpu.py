"""Entry by entry: small gradients beside large ones. Norms over a whole matrix
do not see them, an optimiser that divides each entry by its own size does."""

import math

import pytest
import torch

from llattn_b200 import linear_cross_entropy
from test_training_ops_gpu import BF, FP, make, plain, rel, run

pytestmark = pytest.mark.gpu


def parts(x, w, t, scale=None):
    """dx, dw in 64 bits and what each of their entries sums in magnitude: |G| |w|, |G|^T |x|."""
    xd, wd = x.detach().double(), w.detach().double()
    g = torch.softmax(xd @ wd.T, 1)
    g[torch.arange(len(t), device=x.device), t] -= 1
    g = g * (1 / len(t) if scale is None else scale.double()[:, None])
    return g @ wd, g.T @ xd, g.abs() @ wd.abs(), g.abs().T @ xd.abs()


def worst(got, want, size):
    return ((got.double() - want).abs() / size).max().item()


def test_rows_of_improbable_words_keep_fp32():
    """dw of words whose probability falls from 1 to e^-60. A probability is off by
    its logit's absolute error, logits of at most 60: their sum's, their
    difference's and their exponent's rounding, 3 x 60 x 2^-24 = 1.1e-5, and three
    times that for what the tensor cores' sums drop: 3.3e-5 of an entry."""
    n, d, v = 200, 64, 1000
    gen = torch.Generator(device="cuda").manual_seed(0)
    x, w = torch.randn(n, d, generator=gen, device="cuda"), torch.randn(v, d, generator=gen, device="cuda") * 0.05
    x[:, 0] = 1.0
    w[:, 0] = -torch.linspace(0, 60, v, device="cuda")
    t = torch.randint(0, 20, (n,), generator=gen, device="cuda")
    _, dx, dw = run(x, w, t)
    rdx, rdw, sdx, sdw = parts(x, w, t)
    assert rdw[-1].abs().max().item() < 1e-24  # they are that small
    assert worst(dw, rdw, sdw) <= 3.3e-5 and worst(dx, rdx, sdx) <= 3.3e-5


def test_columns_of_other_sizes_keep_fp32():
    """Columns of x and w from 1e-12 to 1e6 of the others: dx and dw keep fp32 in each
    (losses and probabilities as in test_loss_and_gradients: 1e-5)."""
    n, d, v = 150, 96, 400
    x, w, t = make(n, d, v, FP)
    size = torch.logspace(-12, 6, d, device="cuda")
    xs, ws = x * size, w / size.clamp(min=1)  # x . w is no larger than before
    loss, dx, dw = run(xs, ws, t)
    rl = plain(xs, ws, t)[0]
    rdx, rdw, sdx, sdw = parts(xs, ws, t)
    assert abs(loss.item() - rl.item()) <= 1e-5 * rl.item()
    assert worst(dw, rdw, sdw) <= 1e-5 and worst(dx, rdx, sdx) <= 1e-5


def test_rows_of_other_sizes_keep_fp32():
    """Rows of x and w of other magnitudes; the logits of each at most of usual size."""
    n, d, v = 150, 96, 400
    x, w, t = make(n, d, v, FP)
    xs = x * torch.logspace(-10, 0, n, device="cuda")[:, None]
    ws = w * torch.logspace(0, -10, v, device="cuda")[:, None]
    per = linear_cross_entropy(xs, ws, t, reduction="none").double()
    ref = plain(xs, ws, t, "none")[0]
    assert ((per - ref).abs() <= 1e-5 * ref).all()
    _, dx, dw = run(xs, ws, t)
    rdx, rdw, sdx, sdw = parts(xs, ws, t)
    assert worst(dw, rdw, sdw) <= 1e-5 and worst(dx, rdx, sdx) <= 1e-5


@pytest.mark.parametrize("dtype", [BF, FP])
def test_weighted_tokens_keep_their_own_precision(dtype):
    """reduction none: upstream gradients from 1e-12 to 1, each row of dx for itself
    (bf16: G rounded once, its row's sum once more: 2 x 2^-9 and a quarter on top)."""
    n, d, v = 130, 72, 500
    x, w, t = make(n, d, v, dtype)
    up = torch.logspace(-12, 0, n, device="cuda")
    xr, wr = x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(linear_cross_entropy(xr, wr, t, reduction="none"), (xr, wr), up)
    rdx, rdw, _, _ = parts(x, w, t, up)
    tol = 5e-3 if dtype == BF else 1e-5
    size = rdx
    if dtype == FP:  # p - 1 cancels where p is near 1: its error is one of p and 1
        p = torch.softmax(x.detach().double() @ w.detach().double().T, 1)
        p[torch.arange(n, device="cuda"), t] += 1
        size = up.double()[:, None] * p @ w.detach().double().abs()
    assert ((dx.double() - rdx).norm(dim=1) <= tol * size.norm(dim=1)).all()
    assert rel(dw, rdw) <= tol


@pytest.mark.parametrize("dtype", [BF, FP])
def test_one_bad_token_leaves_the_others_precise(dtype):
    """An infinite upstream gradient, or an infinite x, of one token: the other rows of dx are as good as ever."""
    n, d, v = 40, 72, 300
    x, w, t = make(n, d, v, dtype)
    x = (x.float() * 1e-3).to(dtype)  # (losses near log v)
    up = torch.full((n,), 1e-6, device="cuda")
    rdx = parts(x, w, t, up)[0]
    keep = torch.arange(n, device="cuda") != 7
    tol = 5e-3 if dtype == BF else 1e-5
    for what in ("upstream", "x"):
        xr, wr, g = x.detach().clone(), w.detach().clone().requires_grad_(True), up.clone()
        if what == "upstream":
            g[7] = math.inf
        else:
            xr[7, 3] = math.inf
        xr.requires_grad_(True)
        dx, _ = torch.autograd.grad(linear_cross_entropy(xr, wr, t, reduction="none"), (xr, wr), g)
        assert not torch.isfinite(dx[7]).all()
        assert ((dx.double() - rdx).norm(dim=1) <= tol * rdx.norm(dim=1))[keep].all(), what

@pytest.mark.parametrize("n", [17, 33, 64])
def test_few_tokens_round_once(n):
    """bf16, up to 64 tokens: a row of dx is off by its own rounding, 2^-9 of each
    entry, and what G's two planes leave (2^-17): no token's row by more."""
    x, w, t = make(n, 264, 2000, BF)
    _, dx, dw = run(x, w, t)
    _, rdx, rdw = plain(x, w, t)
    assert ((dx.double() - rdx).norm(dim=1) <= (2**-9 + 2**-15) * rdx.norm(dim=1)).all()
    assert rel(dw, rdw) <= 2**-9 + 2**-15
