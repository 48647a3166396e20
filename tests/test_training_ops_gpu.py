"""linear_cross_entropy and newton_schulz on the GPU against plain
implementations in 64 bits.

Tolerances (2-norm of the difference over the 2-norm of the result), fixed
from the arithmetic:
  * bf16 gradients: G is rounded once to 8 bits (relative error at most 2^-9,
    independent per element) and the result once more: 2 * 2^-9, and a quarter
    on top for what an unlucky sum adds: 5e-3.
  * fp32 gradients: operands of at least 22 bits, sums of up to 1024 products on
    the tensor cores: 1e-5.
  * losses: fp32 sums of d products of magnitude |x||w|: 1e-5 of the losses'
    norm, plus 1e-5 absolute where they are near 0.
  * newton_schulz: one rounding to bf16 at the end (2^-9) and what the fp16
    products leave, up to 1.5e-3 on the spectra here: 4e-3.
"""

import math

import pytest
import torch
import torch.nn.functional as F

import llattn_b200
from llattn_b200 import linear_cross_entropy, newton_schulz

pytestmark = pytest.mark.gpu

GRAD_TOL = {torch.bfloat16: 5e-3, torch.float32: 1e-5}
BF, FP = torch.bfloat16, torch.float32


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    n = b.norm().item()
    return (a - b).norm().item() / n if n else a.norm().item()


def make(n, d, v, dtype, seed=0, ignored=0.0, lean=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(v, d, generator=gen, device="cuda") * (2 / math.sqrt(d))
    t = torch.randint(0, v, (n,), generator=gen, device="cuda")
    x = torch.randn(n, d, generator=gen, device="cuda") + lean * torch.rand(n, 1, generator=gen, device="cuda") * w[t]
    if ignored:
        t = torch.where(torch.rand(n, generator=gen, device="cuda") < ignored, -100, t)
    return x.to(dtype), w.to(dtype), t


def plain(x, w, t, reduction="mean", upstream=None, ignore_index=-100):
    """Loss, dx, dw in 64 bits, from the formulas; tokens that do not count left out."""
    xd, wd = x.detach().double(), w.detach().double()
    at = (t != ignore_index).nonzero()[:, 0]
    xs, ts = xd[at], t[at]
    z = xs @ wd.T
    lse = torch.logsumexp(z, 1)
    r = torch.arange(len(at), device=x.device)
    per = lse - z[r, ts]
    g = torch.exp(z - lse[:, None])
    g[r, ts] -= 1
    if reduction == "mean":
        scale = torch.full_like(per, 1 / max(1, len(at)))
        loss = (per * scale).sum()
    elif reduction == "sum":
        scale, loss = torch.ones_like(per), per.sum()
    else:
        scale = torch.ones_like(per)
        loss = torch.zeros(len(t), dtype=torch.float64, device=x.device)
        loss[at] = per
    if upstream is not None:
        scale = scale * (upstream.double()[at] if upstream.dim() else upstream.double())
    g = g * scale[:, None]
    dx = torch.zeros_like(xd)
    dx[at] = g @ wd
    return loss, dx, g.T @ xs


def check_loss(got, want):
    assert (got.double() - want).norm().item() <= 1e-5 * want.norm().item() + 1e-5 * math.sqrt(want.numel())


def run(x, w, t, **kw):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(x, w, t, **kw)
    return loss.detach(), *torch.autograd.grad(loss, (x, w))


SHAPES = [(1, 64, 97), (1, 8, 1), (2, 16, 2), (5, 96, 300), (64, 128, 128), (127, 72, 129), (129, 256, 1000),
          (300, 88, 513), (257, 264, 4097), (1000, 1536, 8000), (2049, 200, 12289)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n,d,v", SHAPES)
def test_loss_and_gradients(n, d, v, dtype):
    x, w, t = make(n, d, v, dtype)
    loss, dx, dw = run(x, w, t)
    rl, rdx, rdw = plain(x, w, t)
    assert loss.dtype == FP and loss.shape == () and dx.dtype == dtype and dw.dtype == dtype
    check_loss(loss, rl)
    if v == 1:  # the softmax of one class: no loss, no gradient
        assert loss.item() == 0 and not dx.any() and not dw.any()
        return
    assert rel(dx, rdx) <= GRAD_TOL[dtype]
    assert rel(dw, rdw) <= GRAD_TOL[dtype]
    per = linear_cross_entropy(x, w, t, reduction="none")
    check_loss(per, plain(x, w, t, "none")[0])


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n,d,v,ignored", [(200, 64, 301, 0.3), (1500, 136, 2000, 0.9), (65, 40, 50, 0.5), (9, 24, 33, 0.99)])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_ignored_tokens(n, d, v, ignored, reduction, dtype):
    x, w, t = make(n, d, v, dtype, ignored=ignored)
    t[n // 2] = 0  # one counts
    rl, rdx, rdw = plain(x, w, t, reduction)
    bad = x.clone()
    bad[t == -100] = float("nan")  # what an ignored token holds reaches nothing
    bad[(t == -100).nonzero()[:1, 0]] = float("inf")
    loss, dx, dw = run(bad, w, t, reduction=reduction)
    check_loss(loss, rl)
    assert rel(dx, rdx) <= GRAD_TOL[dtype] and rel(dw, rdw) <= GRAD_TOL[dtype]
    assert not dx[t == -100].any()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_nothing_counts(dtype):
    x, w, t = make(70, 64, 200, dtype)
    t[:] = 7
    loss, dx, dw = run(x, w, t, ignore_index=7)
    assert loss.item() == 0 and not dx.any() and not dw.any()
    assert linear_cross_entropy(x, w, t, ignore_index=7).item() == 0
    assert not linear_cross_entropy(x, w, t, ignore_index=7, reduction="none").any()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_no_tokens(dtype):
    x, w, t = make(1, 64, 200, dtype)
    loss, dx, dw = run(x[:0], w, t[:0])
    assert loss.item() == 0 and dx.shape == (0, 64) and not dw.any()
    assert linear_cross_entropy(x[:0], w, t[:0], reduction="none").shape == (0,)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_target_out_of_range_is_loud(dtype):
    x, w, t = make(40, 64, 200, dtype)
    t[3], t[5] = 200, -1
    loss, dx, dw = run(x, w, t)
    assert math.isnan(loss.item()) and dx[3].isnan().all() and dx[5].isnan().all() and dw.isnan().any()
    ok = torch.ones(40, dtype=torch.bool, device="cuda")
    ok[[3, 5]] = False
    assert torch.isfinite(dx[ok]).all()
    per = linear_cross_entropy(x, w, t, reduction="none")
    assert per[3].isnan() and per[5].isnan() and torch.isfinite(per[ok]).all()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_large_and_small_logits(dtype):
    """Logits of some +-1000 (softmax a single one, or far off the target) and near 0."""
    x, w, t = make(130, 128, 700, dtype, lean=0.0)
    scale = torch.logspace(-4, 2.5, 130, device="cuda")[:, None]
    x = (x.float() * scale).to(dtype)
    loss, dx, dw = run(x, w, t)
    rl, rdx, rdw = plain(x, w, t)
    check_loss(loss, rl)
    assert rel(dx, rdx) <= GRAD_TOL[dtype] and rel(dw, rdw) <= GRAD_TOL[dtype]
    per, want = linear_cross_entropy(x, w, t, reduction="none"), plain(x, w, t, "none")[0]
    assert ((per.double() - want).abs() <= 1e-5 * want.abs() + 2e-5 * scale[:, 0].clamp(min=1)).all()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_common_shift_far_from_zero(dtype):
    """All of a row's logits far below or above 0: only differences count."""
    n, d, v = 40, 64, 300
    x, w, t = make(n, d, v, dtype, lean=0.0)
    x[:, 0], w[:, 0] = torch.linspace(-120, 120, n, device="cuda").to(dtype), 4.0
    loss, dx, dw = run(x, w, t)
    rl, rdx, rdw = plain(x, w, t)
    # logits of up to 480 in fp32: 480 * 2^-23 = 6e-5 on each difference
    assert abs(loss.item() - rl.item()) <= 1e-3
    tol = max(GRAD_TOL[dtype], 1e-3)
    assert rel(dx[:, 1:], rdx[:, 1:]) <= tol and rel(dw, rdw) <= tol


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [64, 77])
def test_strides_and_alignment(d, dtype):
    n, v = 150, 333
    x, w, t = make(n, d, v, dtype)
    want = run(x, w, t)
    wide = torch.zeros(n, d + 13, dtype=dtype, device="cuda")
    wide[:, 5:5 + d] = x
    wt = w.t().contiguous().t()  # transposed storage
    flat = torch.zeros(v * d + 3, dtype=dtype, device="cuda")
    wo = flat[3:].view(v, d)
    wo.copy_(w)
    for xs, ws in ((wide[:, 5:5 + d], w), (x, wt), (x, wo), (wide[:, 5:5 + d], wo)):
        got = run(xs, ws, t)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    one = x[:1].expand(n, d)  # rows that share memory
    got, ref = run(one, w, t), plain(one, w, t)
    assert rel(got[1], ref[1]) <= GRAD_TOL[dtype] and rel(got[2], ref[2]) <= GRAD_TOL[dtype]
    t2 = torch.stack([t, t], 1)[:, 0]  # strided targets
    assert torch.equal(run(x, w, t2)[2], want[2])


@pytest.mark.parametrize("dtype", [BF, FP])
def test_leading_shape_upstream_and_partial_gradients(dtype):
    x, w, t = make(6 * 50, 96, 400, dtype, ignored=0.2)
    up = torch.tensor(0.37, device="cuda")
    rl, rdx, rdw = plain(x, w, t, "mean", up)
    x3 = x.view(6, 50, 96).requires_grad_(True)
    w1 = w.clone().requires_grad_(True)
    loss = linear_cross_entropy(x3, w1, t.view(6, 50))
    (loss * up).backward()
    assert rel(x3.grad.view(-1, 96), rdx) <= GRAD_TOL[dtype] and rel(w1.grad, rdw) <= GRAD_TOL[dtype]
    full = run(x, w, t)
    xo = x.detach().clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(xo, w, t), xo)[0], full[1])
    wo = w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x.detach(), wo, t), wo)[0], full[2])
    assert linear_cross_entropy(x.detach(), w, t).item() == pytest.approx(full[0].item(), rel=1e-5)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_per_token_upstream(dtype):
    x, w, t = make(210, 104, 500, dtype, ignored=0.1)
    up = torch.randn(210, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    _, rdx, rdw = plain(x, w, t, "none", up)
    xr, wr = x.requires_grad_(True), w.requires_grad_(True)
    losses = linear_cross_entropy(xr, wr, t, reduction="none")
    dx, dw = torch.autograd.grad(losses, (xr, wr), up)
    assert rel(dx, rdx) <= GRAD_TOL[dtype] and rel(dw, rdw) <= GRAD_TOL[dtype]


def test_retained_graph():
    x, w, t = make(100, 64, 300, BF)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    loss = linear_cross_entropy(x, w, t)
    a = torch.autograd.grad(loss * 3, (x, w), retain_graph=True)
    a = [v.clone() for v in a]
    b = torch.autograd.grad(loss * 3, (x, w))
    for u, v in zip(a, b):
        assert torch.equal(u, v)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("factor", [0.25, -1.7, 0.0])
def test_upstream_gradient(dtype, factor):
    """The upstream gradient scales the products before their only rounding;
    strided inputs; only one of the gradients wanted."""
    n, d, v = 130, 72, 301
    x, w, t = make(n, d, v, dtype, ignored=0.3)
    _, rdx, rdw = plain(x, w, t)
    xs = torch.empty(n, d + 9, device="cuda", dtype=dtype)[:, :d].copy_(x).requires_grad_(True)
    ws = torch.empty(v, d + 5, device="cuda", dtype=dtype)[:, :d].copy_(w).requires_grad_(True)
    dx, dw = torch.autograd.grad(linear_cross_entropy(xs, ws, t) * factor, (xs, ws))
    for got, want in ((dx, rdx), (dw, rdw)):
        if factor:
            assert rel(got, want * factor) <= GRAD_TOL[dtype]
        else:
            assert not got.any()
    assert not dx[t == -100].any()
    only_x, = torch.autograd.grad(linear_cross_entropy(xs, ws.detach(), t) * factor, (xs,))
    only_w, = torch.autograd.grad(linear_cross_entropy(xs.detach(), ws, t) * factor, (ws,))
    assert torch.equal(only_x, dx) and torch.equal(only_w, dw)


@pytest.mark.parametrize("n,v", [(9, 1_600_001), (20, 2_097_152)])
def test_largest_vocabularies(n, v):
    x, w, t = make(n, 16, v, BF)
    loss, dx, dw = run(x, w, t)
    rl, rdx, rdw = plain(x, w, t)
    assert abs(loss.item() - rl.item()) <= 1e-5 * rl.item()
    assert rel(dx, rdx) <= GRAD_TOL[BF] and rel(dw, rdw) <= GRAD_TOL[BF]


def test_changed_inputs_are_refused_in_the_backward():
    x, w, t = make(40, 64, 200, BF)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    loss = linear_cross_entropy(x, w, t)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("n,d,v,dtype", [(1, 2048, 4000, FP), (1, 2048, 4000, BF), (200, 2048, 3000, FP), (70, 1700, 900, BF)])
def test_long_products_keep_fp32(n, d, v, dtype):
    """Losses of long dot products: the tensor cores' truncating additions run in
    chains joined in fp32. A chain loses up to 2^-26 (bf16) or 2^-24 (fp32's
    planes) of itself per 16 products, so a logit of at most 14 is at most 14 x
    24 x 4 x 2^-26 / 2 = 1e-5 (bf16, 24 steps a chain) or 14 x 8 x 4 x 2^-24 / 2 =
    1.4e-5 (fp32, 8 steps) off, plus fp32's rounding of the loss itself."""
    x, w, t = make(n, d, v, dtype)
    ref = plain(x, w, t, "none")[0]
    got = linear_cross_entropy(x, w, t, reduction="none").double()
    assert (got - ref).abs().max().item() <= 2e-5


def test_gradient_against_differences():
    """fp32: the directional derivative of the loss by central differences in
    64 bits of the plain loss, at the same point."""
    x, w, t = make(60, 48, 150, FP, ignored=0.2)
    _, dx, dw = run(x, w, t)
    gen = torch.Generator(device="cuda").manual_seed(9)
    ux, uw = torch.randn(x.shape, generator=gen, device="cuda").double(), torch.randn(w.shape, generator=gen, device="cuda").double()
    h = 1e-5
    f = lambda s: plain(x.double() + s * h * ux, w.double() + s * h * uw, t)[0].item()
    num = (f(1) - f(-1)) / (2 * h)
    ana = ((dx.double() * ux).sum() + (dw.double() * uw).sum()).item()
    assert abs(num - ana) <= 1e-5 * (abs(num) + 1)


def test_several_pieces():
    """More rows than are held at a time: pieces joined in order, some of them
    with few or no counted tokens."""
    n, d, v = 8500, 64, 32768
    x, w, t = make(n, d, v, BF)
    t[200:] = torch.where(torch.rand(n - 200, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) < 0.02, t[200:], -100)
    for ts in (make(n, d, v, BF)[2], t):
        loss, dx, dw = run(x, w, ts)
        rl, rdx, rdw = plain(x, w, ts)
        check_loss(loss, rl)
        assert rel(dx, rdx) <= 5e-3 and rel(dw, rdw) <= 5e-3
    x, w, t = make(2500, 64, 3000, FP, ignored=0.1)
    loss, dx, dw = run(x, w, t)
    rl, rdx, rdw = plain(x, w, t)
    check_loss(loss, rl)
    assert rel(dx, rdx) <= 1e-5 and rel(dw, rdw) <= 1e-5


def test_same_bits_again_and_on_another_stream():
    x, w, t = make(700, 256, 5000, BF, ignored=0.1)
    want = run(x, w, t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(x, w, t)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_autocast_matches_the_cast_inputs():
    x, w, t = make(90, 64, 256, FP)
    want = run(x.to(BF), w.to(BF), t)
    xr, wr = x.requires_grad_(True), w.requires_grad_(True)
    with torch.autocast("cuda", dtype=BF):
        loss = linear_cross_entropy(xr, wr, t)
    loss.backward()
    assert torch.equal(loss, want[0]) and torch.equal(wr.grad, want[2].float()) and torch.equal(xr.grad, want[1].float())


def test_compiled_equals_eager():
    x, w, t = make(90, 64, 256, BF)

    def step(x, w):
        return linear_cross_entropy(x, w, t) * 2.0

    got = {}
    for name, f in (("eager", step), ("compiled", torch.compile(step, backend="aot_eager", fullgraph=True))):
        xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = f(xr, wr)
        loss.backward()
        got[name] = (loss.detach(), xr.grad, wr.grad)
    for a, b in zip(got["eager"], got["compiled"]):
        assert torch.equal(a, b)  # a factor of 2 rounds nowhere


def test_loss_refusals():
    x, w, t = make(10, 64, 100, BF)
    for bad, msg in (((x, w.float(), t), "dtype"), ((x.half(), w.half(), t), "dtype"), ((x, w[:, :32], t), "columns"),
                     ((x, w, t[:5]), "leading shape"), ((x, w, t.int()), "int64"), ((x, w.cpu(), t), "device"),
                     ((x, w[:0], t), "rows")):
        with pytest.raises(RuntimeError, match=msg):
            linear_cross_entropy(*bad)
    with pytest.raises(RuntimeError, match="reduction"):
        linear_cross_entropy(x, w, t, reduction="sums")


# ---------------------------------------------------------------------------

COEF = (3.4445, -4.7750, 2.0315)


def plain_ns(g, steps=5, coefficients=COEF, eps=1e-7):
    a, b, c = coefficients
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.mT if tall else x
    x = x / (x.norm() + eps)
    for _ in range(steps):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if tall else x


def spectrum(m, n, decay, dtype, seed=0, noise=0.3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k = min(m, n)
    low = torch.randn(m, k, generator=gen, device="cuda") * torch.arange(1, k + 1, device="cuda") ** -decay
    g = low @ torch.randn(k, n, generator=gen, device="cuda")
    g = g / g.square().mean().sqrt() + noise * torch.randn(m, n, generator=gen, device="cuda")
    return g.to(dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 40), (16, 16), (40, 7), (64, 1536), (1536, 64), (100, 77), (128, 384), (257, 255),
                                 (256, 256), (777, 1001), (1001, 776), (1536, 1536), (2100, 640)])
def test_newton_schulz(m, n, dtype):
    gs = [spectrum(m, n, d, dtype, i) * s for i, (d, s) in enumerate([(0.0, 1.0), (0.7, 1e-5), (1.0, 300.0)])]
    outs = newton_schulz(gs)
    for g, o in zip(gs, outs):
        assert o.dtype == BF and o.shape == g.shape
        assert rel(o, plain_ns(g)) <= 4e-3


def test_newton_schulz_batches_lists_and_layouts():
    gs = [spectrum(48, 80, 0.5, BF, i) for i in range(70)]  # more than one conversion launch
    outs = newton_schulz(gs)
    batch = newton_schulz(torch.stack(gs).view(7, 10, 48, 80))
    assert batch.shape == (7, 10, 48, 80)
    for i, (g, o) in enumerate(zip(gs, outs)):
        assert torch.equal(o, batch.view(70, 48, 80)[i])
        if i % 23 == 0:
            assert rel(o, plain_ns(g)) <= 4e-3
    mixed = [spectrum(48, 80, 0.5, FP, 1), gs[0], spectrum(30, 20, 0.5, BF, 2), gs[1]]
    for g, o in zip(mixed, newton_schulz(mixed)):
        assert o.shape == g.shape and rel(o, plain_ns(g)) <= 4e-3
    assert torch.equal(newton_schulz(gs[0].t().contiguous().t()), outs[0])  # transposed storage
    flat = torch.zeros(48 * 80 + 1, dtype=BF, device="cuda")
    flat[1:] = gs[0].reshape(-1)
    assert torch.equal(newton_schulz(flat[1:].view(48, 80)), outs[0])  # 2-byte alignment
    assert newton_schulz([]) == []
    assert newton_schulz(torch.zeros(0, 5, device="cuda")).shape == (0, 5)


def test_newton_schulz_zero_and_non_finite():
    z = newton_schulz(torch.zeros(64, 96, device="cuda", dtype=BF))
    assert not z.any()
    gs = [spectrum(64, 96, 0.5, FP, i) for i in range(3)]
    gs[1][3, 4] = float("nan")
    outs = newton_schulz(gs)
    assert outs[1].isnan().any()
    assert rel(outs[0], plain_ns(gs[0])) <= 4e-3 and rel(outs[2], plain_ns(gs[2])) <= 4e-3  # only its own matrix


@pytest.mark.parametrize("steps,coefficients", [(1, COEF), (2, COEF), (3, COEF), (8, COEF), (12, (1.5, -0.5, 0.0)),
                                                (6, (1.875, -1.25, 0.375))])
def test_newton_schulz_steps_and_coefficients(steps, coefficients):
    g = spectrum(200, 320, 0.3, BF)
    got = newton_schulz(g, steps=steps, coefficients=coefficients)
    assert rel(got, plain_ns(g, steps, coefficients)) <= 4e-3


def test_newton_schulz_refusals():
    g = torch.randn(8, 8, device="cuda")
    for bad, kw, msg in ((g[0], {}, "matrices"), (g.half(), {}, "dtype"), (g.cpu(), {}, "CUDA"), (g, {"steps": 0}, "steps"),
                         (g, {"coefficients": (99.0, 0.0, 0.0)}, "coefficients"), ([g, g[0]], {}, "matrices"),
                         (g, {"eps": -1.0}, "eps")):
        with pytest.raises(RuntimeError, match=msg):
            newton_schulz(bad, **kw)


def test_muon_step_follows_the_formula():
    gen = torch.Generator(device="cuda").manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(s, generator=gen, device="cuda") * 0.02) for s in ((96, 64), (64, 96), (96, 64))]
    ws = [p.detach().double().clone() for p in ps]
    bufs = [torch.zeros_like(w) for w in ws]
    opt = llattn_b200.Muon(ps, lr=1e-2, momentum=0.9, weight_decay=0.1)
    for _ in range(3):
        for p, w, b in zip(ps, ws, bufs):
            p.grad = torch.randn(p.shape, generator=gen, device="cuda")
            b.mul_(0.9).add_(p.grad.double())
            u = plain_ns(p.grad.double() + 0.9 * b)
            w.mul_(1 - 1e-2 * 0.1).sub_(1e-2 * 0.2 * math.sqrt(96) * u)
        opt.step()
        for p, w in zip(ps, ws):
            # the update is 0.02 of the weights' size at most here, itself 4e-3 off
            assert rel(p, w) <= 1e-3
