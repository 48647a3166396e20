"""gated_mlp's sums of very many products of one sign, in bf16.

A tensor-core addition of 16 products drops what lies below the running sum's last bit (2^-24 to 2^-23 of it, 0.72 2^-23 on
average over its sizes). One sum of 2^19 and more random or equal products came out K 2^-27.3 short: 2.3 such bits an
addition, of a running sum that is half the last one on average. The bounds take 4. Sums of at most 2^16 products, added
up in fp32, then are 2^12 4 0.72 2^-23 / 2 = 7.0e-4 < 2^-10 short."""

import pytest
import torch

from llattn_b200 import gated_mlp

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
CHAIN = 2.0 ** -10


def silu(g):
    s = torch.sigmoid(g)
    return g * s, s * (1 + g * (1 - s))


@pytest.mark.parametrize("n", (40, 100))
@pytest.mark.parametrize("d", (1 << 18, 1 << 20))
def test_many_columns(n, d):
    """g, u (sums over d), dh (over d_out) and the results: constants, whose every addition drops the same."""
    ff = 16
    full = lambda *s, v: torch.full(s, v, device="cuda", dtype=BF)
    x, w = full(n, d, v=1.0), full(ff, d, v=0.713 / d)
    eye = torch.eye(ff, device="cuda", dtype=BF)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    y = gated_mlp(x, w, w, eye)
    s = w.detach()[0].double().sum()
    a, slope = silu(s)
    # g and u short, which act(g) u sees 1 + g act'(g) / act(g) < 2.3 times; h and y rounded (2^-8 each at most)
    want = a * s
    assert ((y.double() - want).abs() <= (2 * 2.0 ** -8 + 2.3 * CHAIN + 2.0 ** -16) * want).all()
    # dx = dy (a + s act'(s)) w + ..., rounded: dg, du and dx, on top of g's and u's
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    want = ff * (s * slope + a) * w.detach()[0, 0].double()
    assert ((dx.double() - want).abs() <= (2 * 2.0 ** -8 + 2.0 ** -11 + 3 * CHAIN) * want).all()
    del x, leaves, y, dx
    # dh over d_out: dx of a single large output
    x, wg = full(n, ff, v=1.0), full(ff, ff, v=0.0625)
    wd = full(d, ff, v=0.713 / d)
    x.requires_grad_(True)
    y = gated_mlp(x, wg, wg, wd)
    (dx,) = torch.autograd.grad(y, x, full(n, d, v=1.0))
    a, slope = silu(torch.tensor(1.0, dtype=torch.float64, device="cuda"))
    want = (a + slope) * wd[:, 0].double().sum()  # (ff / 16 = 1: the sums over ff and d of the rest)
    assert ((dx.double() - want).abs() <= (2 * 2.0 ** -8 + 2.0 ** -11 + CHAIN) * want).all()


def test_many_tokens():
    """dw_gate and dw_up over 2^19 tokens whose tiles fill the GPU, so that their sums are not split: positive random
    values, whose roundings average out over 1.2 M entries, and what the sums drop does not."""
    n, d, ff = 1 << 19, 148 * 128, 64
    gen = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.rand(*s, generator=gen, device="cuda") + 0.5
    x = torch.empty(n, d, dtype=BF, device="cuda")
    for i in range(0, n, 1 << 15):
        x[i:i + (1 << 15)] = r(1 << 15, d)
    ws = [(r(ff, d) / d).to(BF), (r(ff, d) / d).to(BF), (r(8, ff) / ff).to(BF)]
    dy = r(n, 8).to(BF)
    leaves = [w.requires_grad_(True) for w in ws]
    got = torch.autograd.grad(gated_mlp(x, *leaves), leaves, dy)
    wg, wu, wd = (w.detach().double() for w in ws)
    want = [torch.zeros_like(w) for w in (wg, wu, wd)]
    for i in range(0, n, 1 << 14):
        xs, ds = x[i:i + (1 << 14)].double(), dy[i:i + (1 << 14)].double()
        g, u, dh = xs @ wg.T, xs @ wu.T, ds @ wd
        a, slope = silu(g)
        for k, (p, q) in enumerate(((dh * u * slope, xs), (dh * a, xs), (ds, a * u))):
            want[k].addmm_(p.T, q)
    for v, w in zip(got[:2], want[:2]):
        # the sums over the tokens 7.0e-4, g's and u's over d 18944 / 16 4 0.72 2^-23 / 2 = 2.0e-4, seen up to 1.4 times
        mean = (v.double() / w - 1).mean().item()
        assert abs(mean) <= 9.9e-4, mean
    for v, w in zip(got, want):
        # every entry: operands and results rounded, what is dropped
        assert ((v.double() - w).abs() <= (2 * 2.0 ** -8 + 2.0 ** -10 + CHAIN) * w).all()
