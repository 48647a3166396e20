"""gated_mlp's gelu where it is close to 0, relative to its value: y = gelu(g) 1 1 for inputs that make the products exact.

Bounds, relative: bf16 rounds h (over 64 tokens, 2^-8; else 2^-16) and y (2^-8); phi is off by 2^-16 (ex2's
argument up to 2^7), up to 64 tokens by 2^-18. dx rounds dg and itself. fp32: erfc's 4 ulp of 2^-23, exp's and the
correction's two each, two products, and 24 bits of h, 2^-23, down to where its third plane is a bf16 number (1e-18)."""

import math

import pytest
import torch

from llattn_b200 import gated_mlp

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float32


def case(n, dt, low, high):
    g = torch.linspace(low, high, n, device="cuda").bfloat16().to(dt)
    x = torch.stack([g, torch.ones_like(g)], 1)
    one = lambda *v: torch.tensor([v], device="cuda", dtype=dt)
    return g.double(), x, (one(1.0, 0.0), one(0.0, 1.0), one(1.0))


def relative(got, want):
    return (got.double() / want - 1).abs().max().item()


@pytest.mark.parametrize("dt", (BF, FP), ids=("bf16", "f32"))
@pytest.mark.parametrize("n", (3, 16, 24, 33, 64, 65, 300, 3000))
@pytest.mark.parametrize("grad", (False, True))
def test_gelus_tail(n, dt, grad):
    g, x, ws = case(n, dt, -12.5 if dt == BF else -8.5, -1.5)
    x.requires_grad_(grad)
    y = gated_mlp(x, *ws, activation="gelu")
    phi = torch.special.erfc(-g / math.sqrt(2)) / 2
    few, exact = 2.0 ** -8 + 2.0 ** -16 + 2.0 ** -18, 8 * 2.0 ** -23 + 2 * 2.0 ** -24 + 2.0 ** -23
    assert relative(y[:, 0], g * phi) <= (exact if dt == FP else few if n <= 64 else 2 * 2.0 ** -8 + 2.0 ** -14)
    if grad:
        (dx,) = torch.autograd.grad(y.sum(), x)
        slope = phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        # (phi and g times the density: of different signs, the first at most 0.5 of the second from -1.5 on)
        assert relative(dx[:, 0], slope) <= (3 * exact if dt == FP else 2 * 2.0 ** -8 + 2.0 ** -14)


@pytest.mark.parametrize("dt", (BF, FP), ids=("bf16", "f32"))
@pytest.mark.parametrize("name", ("silu", "gelu"))
@pytest.mark.parametrize("n", (4, 40, 100))
def test_far_and_no_numbers(n, dt, name):
    """Both ends: 0 and g itself, infinities and NaN as torch's activations have them."""
    f = torch.nn.functional.silu if name == "silu" else torch.nn.functional.gelu
    values = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 30.0, 1e4, -1e4, 1e18, -1e18, 1e30, -1e30, float("inf"), float("nan")], device="cuda")
    for at in range(0, len(values), n):
        g = values[at:at + n]
        _, x, ws = case(n, dt, 0.0, 1.0)
        x[:len(g), 0] = g.to(dt)
        with torch.no_grad():
            y = gated_mlp(x, *ws, activation=name)
        want = f(x[:len(g), 0].double())
        ok = want.isfinite()
        assert torch.equal(y[:len(g), 0].isnan() | y[:len(g), 0].isinf(), ~ok)
        assert ((y[:len(g), 0].double() - want)[ok].abs() <= 2 * 2.0 ** -8 * want[ok].abs() + 1e-38).all()


@pytest.mark.parametrize("dt", (BF, FP), ids=("bf16", "f32"))
@pytest.mark.parametrize("name", ("silu", "gelu"))
@pytest.mark.parametrize("n", (5, 64, 90))
@pytest.mark.parametrize("which", (0, 1))
def test_an_overflowing_row_leaves_its_neighbours_gradients(n, name, dt, which):
    """Columns of g or u that are infinite are kept beside finite ones, whose weights' gradients are what they are without."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dt)
    x, ws, dy = r(n, 40) + 3, [r(48, 40) / 8, r(48, 40) / 8, r(24, 48)], r(n, 24)
    x.abs_()
    rows = [3, 16, 47]
    rest = torch.ones(48, dtype=torch.bool, device="cuda")
    rest[rows] = False

    def grads():
        leaves = [w.clone().requires_grad_(True) for w in ws]
        return torch.autograd.grad(gated_mlp(x, *leaves, activation=name), leaves[:2], dy)

    want = grads()
    ws[which][rows[0]] = float("inf")
    ws[which][rows[1]] = -float("inf")
    # above fp32's range with every token (x's rows are positive and sum to more than 2; one entry of 3e38 alone leaves tokens
    # with x[0] < 1.13 a finite 3e38, of which a block keeps 11 bits and its neighbours, 2^-28 of that and less, nothing)
    assert x.sum(1).min() > 2
    ws[which][rows[2]] = 3e38
    for got, w in zip(grads(), want):
        assert torch.equal(got[rest], w[rest])
        assert (w[rest] != 0).any(1).all()
