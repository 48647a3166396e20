"""gated_mlp on the GPU against the formulas in 64 bits, entry by entry.

Bounds (u = 2^-8 for bf16, the relative error of one rounding; all other factors in absolute values):
  fp32 sums of K products, per |a||b|: six products of three bf16 planes drop less than 2^-22; a tensor-core sum
    of 256 products is 16 additions that truncate, 2^-23 each; chains of 256 are added in fp32: s(K) = 2^-22 + 2^-19 +
    K 2^-32. bf16 products are exact, their sums truncate in one chain of K / 16 additions: s(K) = K 2^-27.
  h: one rounding (bf16), the activation's own error (2^-20 |a u|), and g's and u's sums.
  y: h's error through |Wd|, the sum's, one rounding.
  kept g, u (bf16): 2^-11 each, so that dg = dh u act'(g) is off by 2^-11 (|dg| + 1.1 |dh u|) (|g act''(g)| <= 1.1 for
    both activations) and du = dh act(g) by 2^-11 1.2 |dh g| (|act'| <= 1.2), and by one rounding.
"""

import itertools

import pytest
import torch

from llattn_b200 import gated_mlp, lm_ops, token_embedding

pytestmark = pytest.mark.gpu

DTYPES = (torch.bfloat16, torch.float32)


def unit(dt):
    return 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -24


def sums(K, dt):
    return 2.0 ** -22 + 2.0 ** -19 + K * 2.0 ** -32 if dt == torch.float32 else K * 2.0 ** -27


def tensors(n, d, ff, d_out, dt, seed=0, gain=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    return ((r(n, d) * gain).to(dt), (r(ff, d) * 1.5 / d ** 0.5).to(dt), (r(ff, d) / d ** 0.5).to(dt),
            (r(d_out, ff) / ff ** 0.5).to(dt), r(n, d_out).to(dt))


def act64(g, name):
    if name == "silu":
        s = torch.special.expit(g)
        return g * s, s * (1 + g * (1 - s))
    c = torch.special.ndtr(g)
    return g * c, c + g * torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5


def formula(x, wg, wu, wd, dy, name):
    """{output: (value, bound)} in 64 bits."""
    dt, u = x.dtype, unit(x.dtype)
    x, wg, wu, wd, dy = (t.detach().double() for t in (x, wg, wu, wd, dy))
    n, d, ff, d_out = x.shape[0], x.shape[1], wg.shape[0], wd.shape[0]
    rounds = 1.0  # (fp32 operands are whole)
    keep = 2.0 ** -11 if dt == torch.bfloat16 else 0.0
    g, up = x @ wg.T, x @ wu.T
    ag, au = x.abs() @ wg.T.abs(), x.abs() @ wu.T.abs()
    a, slope = act64(g, name)
    h = a * up
    eg, eu = sums(d, dt) * ag, sums(d, dt) * au
    eh = u * rounds * h.abs() + 2.0 ** -20 * h.abs() + 1.2 * eg * up.abs() + a.abs() * eu
    y = h @ wd.T
    ey = eh @ wd.T.abs() + sums(ff, dt) * (h.abs() @ wd.T.abs()) + u * y.abs()
    out = {"y": (y, ey)}
    dh = dy @ wd
    edh = sums(d_out, dt) * (dy.abs() @ wd.abs())
    dg, du = dh * up * slope, dh * a
    edg = (u + keep + 2.0 ** -20) * dg.abs() + 1.1 * (keep + 2.0 ** -20) * (dh * up).abs() + edh * (up * slope).abs()
    edg += dh.abs() * (eu * slope.abs() + 1.1 * eg * up.abs())
    edu = (u + 2.0 ** -20) * du.abs() + 1.2 * keep * (dh * g).abs() + edh * a.abs() + 1.2 * dh.abs() * eg
    ehk = eh + keep * (h.abs() + 1.2 * (g * up).abs())
    dx = dg @ wg + du @ wu
    out["dx"] = dx, (edg @ wg.abs() + edu @ wu.abs() + sums(2 * ff, dt) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
                     + u * dx.abs())
    for k, (v, e) in {"dw_gate": (dg, edg), "dw_up": (du, edu)}.items():
        w = v.T @ x
        out[k] = w, e.T @ x.abs() + sums(n, dt) * (v.T.abs() @ x.abs()) + u * w.abs()
    w = dy.T @ h
    out["dw_down"] = w, dy.T.abs() @ ehk + sums(n, dt) * (dy.T.abs() @ h.abs()) + u * w.abs()
    return out


def check(got, want, what):
    for k, v in got.items():
        value, bound = want[k]
        off = (v.double() - value).abs()
        worst = (off / bound.clamp(min=1e-300)).max().item() if off.numel() else 0.0
        assert v.shape == value.shape and worst <= 1.0, f"{what} {k}: {worst:.3g} of its bound"


def run(x, wg, wu, wd, dy, name):
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = gated_mlp(*leaves, activation=name)
    return dict(zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), (y.detach(), *torch.autograd.grad(y, leaves, dy))))


SIZES = [(1, 64, 64, 64), (1, 1, 1, 1), (2, 8, 40, 16), (3, 33, 7, 5), (16, 128, 96, 128), (17, 141, 377, 51), (32, 72, 31, 8),
         (33, 72, 33, 8), (64, 136, 65, 40), (65, 256, 129, 264), (127, 96, 512, 96), (129, 200, 1000, 72), (300, 512, 1365, 512),
         (1025, 320, 264, 320)]


@pytest.mark.parametrize("dt", DTYPES, ids=("bf16", "f32"))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(size, dt):
    for name in ("silu", "gelu"):
        ins = tensors(*size, dt, seed=sum(size))
        want = formula(*ins, name)
        check(run(*ins, name), want, name)
        with torch.no_grad():  # (another kernel for few tokens)
            check({"y": gated_mlp(*ins[:4], activation=name)}, want, name + " no grad")


@pytest.mark.parametrize("dt", DTYPES, ids=("bf16", "f32"))
def test_in_two_norm(dt):
    """Independent roundings: rms at most u / sqrt 3 each, two of them for bf16 (operand and result); fp32: what drops is
    far below its worst case, 1e-6 of it."""
    ins = tensors(700, 384, 1100, 384, dt, seed=5)
    want = formula(*ins, "silu")
    for k, v in run(*ins, "silu").items():
        off = ((v.double() - want[k][0]).norm() / want[k][0].norm()).item()
        assert off <= (2 / 3) ** 0.5 * 2.0 ** -8 if dt == torch.bfloat16 else off <= 1e-6, (k, off)


@pytest.mark.parametrize("dt", DTYPES, ids=("bf16", "f32"))
@pytest.mark.parametrize("n", (5, 100))
def test_strided_and_unaligned_rows(n, dt):
    d, ff, d_out = 72, 88, 56
    x, wg, wu, wd, dy = tensors(n, d, ff, d_out, dt)
    want = formula(x, wg, wu, wd, dy, "silu")

    def inside(t, pad, shift):
        wide = torch.full((t.shape[0] + 2, t.shape[1] + pad), float("nan"), dtype=t.dtype, device="cuda")
        view = wide[1:-1, shift:shift + t.shape[1]]
        view.copy_(t)
        return view

    for pads in ((8, 8, 8, 8, 8), (3, 5, 8, 1, 7), (0, 0, 0, 0, 0)):
        shifts = [p // 2 if p % 8 else 0 for p in pads]
        got = run(*(inside(t, p, s) for t, p, s in zip((x, wg, wu, wd, dy), pads, shifts)), "silu")
        check(got, want, f"pads {pads}")
        with torch.no_grad():
            ins = [inside(t, p, s) for t, p, s in zip((x, wg, wu, wd), pads, shifts)]
            check({"y": gated_mlp(*ins)}, want, f"pads {pads} no grad")
    # gate and up in one matrix, the rows of one off a 16-byte boundary by another shift than the other's
    for rows in (ff, ff - 1, 1):
        both = torch.cat([wg[:rows, :71], wu[:rows, :71]])
        ins = (x[:, :71], both[:rows], both[rows:], wd[:, :rows])
        with torch.no_grad():
            check({"y": gated_mlp(*ins)}, formula(*ins, dy, "silu"), f"{rows} rows of both in one")
    # columns that are not contiguous are copied; one weight in two places; broadcast upstream gradients
    got = run(x.t().contiguous().t(), wg.t().contiguous().t(), wu, wd, dy, "silu")
    check(got, want, "transposed")
    same = formula(x, wg, wg, wd, torch.ones_like(dy), "silu")
    leaf = wg.detach().requires_grad_(True)
    y = gated_mlp(x, leaf, leaf, wd)
    (dw,) = torch.autograd.grad(y.sum(), leaf)
    value = same["dw_gate"][0] + same["dw_up"][0]
    bound = same["dw_gate"][1] + same["dw_up"][1] + unit(dt) * value.abs()
    assert ((dw.double() - value).abs() <= bound).all()


@pytest.mark.parametrize("dt", DTYPES, ids=("bf16", "f32"))
def test_range_of_values(dt):
    """Columns of g and u from 1e-30 to 1e30 beside one another: what is kept holds 11 bits of each block's largest."""
    n, d, ff = 130, 64, 320
    x, wg, wu, wd, dy = tensors(n, d, ff, 64, dt, seed=3)
    scale = 10.0 ** torch.linspace(-12, 12, ff // 32, device="cuda").repeat_interleave(32)[:, None]
    wu, wd = (wu.float() * scale).to(dt), (wd.float() / scale.T).to(dt)
    want = formula(x, wg, wu, wd, dy, "gelu")
    check(run(x, wg, wu, wd, dy, "gelu"), want, "scaled")
    # far pre-activations: the gate is 0 or 1, nothing is NaN
    big = x * 300
    got = run(big, wg, wu, wd, dy, "silu")
    check(got, formula(big, wg, wu, wd, dy, "silu"), "far")
    assert all(torch.isfinite(v).all() for v in got.values())


@pytest.mark.parametrize("n", (3, 40, 200))
def test_nan_rows_stay_in_their_rows(n):
    x, wg, wu, wd, dy = tensors(n, 64, 96, 48, torch.bfloat16)
    clean = run(x, wg, wu, wd, dy, "silu")
    x[1] = float("nan")
    got = run(x, wg, wu, wd, dy, "silu")
    with torch.no_grad():
        y = gated_mlp(x, wg, wu, wd)
    rest = torch.arange(n, device="cuda") != 1
    assert got["y"][1].isnan().all() and y[1].isnan().all() and got["dx"][1].isnan().all()
    assert torch.equal(got["y"][rest], clean["y"][rest]) and torch.equal(got["dx"][rest], clean["dx"][rest])
    assert not y[rest].isnan().any() and got["dw_down"].isnan().any()


@pytest.mark.parametrize("n", (7, 90))
def test_some_gradients_only(n):
    ins = tensors(n, 96, 160, 64, torch.bfloat16, seed=8)
    full = run(*ins, "gelu")
    names = ("dx", "dw_gate", "dw_up", "dw_down")
    for need in itertools.product((False, True), repeat=4):
        if not any(need):
            continue
        leaves = [t.detach().requires_grad_(r) for t, r in zip(ins[:4], need)]
        y = gated_mlp(*leaves, activation="gelu")
        got = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], ins[4])
        for k, v in zip((k for k, r in zip(names, need) if r), got):
            assert torch.equal(v, full[k]), (need, k)


@pytest.mark.parametrize("dt", DTYPES, ids=("bf16", "f32"))
def test_same_bits_again_and_differences(dt):
    ins = tensors(257, 128, 333, 128, dt, seed=2)
    one, two = run(*ins, "silu"), run(*ins, "silu")
    assert all(torch.equal(one[k], two[k]) for k in one)
    if dt == torch.float32:  # a directional difference of the fp32 form: step 2^-10, the third derivative's 2^-20
        x, wg, wu, wd, dy = ins
        v = torch.randn(x.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
        step = 2.0 ** -10
        with torch.no_grad():
            up, down = (gated_mlp(x + s * v, wg, wu, wd).double() for s in (step, -step))
        slope = ((up - down) * dy.double()).sum() / (2 * step)
        value = (one["dx"].double() * v.double()).sum()
        # rounding of y: 1e-6 |y| over 2^-9, through the sum of |dy|
        noise = (1e-6 * one["y"].abs() * dy.abs()).double().norm() / step
        assert (slope - value).abs() <= 4 * noise + 2.0 ** -16 * value.abs().clamp(min=one["dx"].double().norm())


def test_shapes_autocast_and_empty():
    x, wg, wu, wd, dy = tensors(24, 64, 96, 40, torch.bfloat16)
    flat = gated_mlp(x, wg, wu, wd)
    assert torch.equal(gated_mlp(x.view(2, 3, 4, 64), wg, wu, wd).view(24, 40), flat)
    assert torch.equal(gated_mlp(x[0], wg, wu, wd)[None], gated_mlp(x[:1], wg, wu, wd))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = gated_mlp(x.float(), wg.float(), wu.float(), wd.float())
    assert y.dtype == torch.bfloat16 and torch.equal(y, flat)
    with torch.autocast("cuda", dtype=torch.float16):
        assert gated_mlp(x, wg, wu, wd).dtype == torch.float32
    leaves = [t.detach().requires_grad_(True) for t in (x[:0], wg, wu, wd)]
    y = gated_mlp(*leaves)
    assert y.shape == (0, 40)
    grads = torch.autograd.grad(y.sum(), leaves)
    assert grads[0].shape == (0, 64) and all((g == 0).all() for g in grads[1:])
    assert gated_mlp(x.view(24, 1, 64)[:, :0], wg, wu, wd).shape == (24, 0, 40)
    # fp32 leaves under autocast get fp32 gradients
    leaves = [t.float().requires_grad_(True) for t in (x, wg, wu, wd)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = gated_mlp(*leaves)
    y.backward(dy)
    assert all(t.grad.dtype == torch.float32 for t in leaves)


def test_graphs_streams_hooks_and_compile():
    x, wg, wu, wd, dy = tensors(80, 128, 160, 128, torch.bfloat16)
    want = run(x, wg, wu, wd, dy, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run(x, wg, wu, wd, dy, "silu")
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run(x, wg, wu, wd, dy, "silu")
            with torch.no_grad():
                few = gated_mlp(x[:4], wg, wu, wd)
        graphs.append((graph, got, few))
    small = gated_mlp(x[:4], wg, wu, wd)
    x.mul_(2)
    twice = run(x, wg, wu, wd, dy, "silu")
    small2 = gated_mlp(x[:4], wg, wu, wd)
    for graph, _, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, got, few in graphs:
        assert all(torch.equal(got[k], twice[k]) for k in got) and torch.equal(few, small2)
    x.div_(2)
    assert torch.equal(gated_mlp(x[:4], wg, wu, wd), small)
    # saved tensors may be moved
    with torch.autograd.graph.save_on_cpu():
        leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
        y = gated_mlp(*leaves)
    grads = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy)
    for k, a, b in zip(("dx", "dw_gate", "dw_up", "dw_down"), grads, again):
        assert torch.equal(a, want[k]) and torch.equal(b, want[k])
    f = torch.compile(lambda *t: gated_mlp(*t), backend="aot_eager", fullgraph=True)
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = f(*leaves)
    assert torch.equal(y, want["y"])
    for k, a in zip(("dx", "dw_gate", "dw_up", "dw_down"), torch.autograd.grad(y, leaves, dy)):
        assert torch.equal(a, want[k])
    y = gated_mlp(*leaves)
    (dx,) = torch.autograd.grad(y, leaves[0], dy.requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        dx.sum().backward()


@pytest.mark.parametrize("d", [256, 261])
@pytest.mark.parametrize("n", [1, 8, 30])
def test_behind_a_kernel_that_is_still_writing(n, d):
    """Each of the library's launches may start before the one that writes its input is done."""
    _, wg, wu, wd, _ = tensors(1, d, 640, d, torch.bfloat16)
    w = torch.randn(4096, d, device="cuda").bfloat16()
    ids = torch.randint(0, 4096, (64, n), device="cuda")
    with torch.no_grad():
        rows = [token_embedding(i, w) for i in ids]
        want = []
        for x in rows:
            torch.cuda.synchronize()
            want.append(gated_mlp(x, wg, wu, wd))
        torch.cuda.synchronize()
        # x's memory is the same in every step: what an SM has left of the step before is wrong
        got = [gated_mlp(token_embedding(i, w), wg, wu, wd) for i in ids]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            replayed = [gated_mlp(token_embedding(i, w), wg, wu, wd) for i in ids]
        for _ in range(3):
            graph.replay()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, replayed))


def test_refusals():
    x, wg, wu, wd, _ = tensors(4, 64, 96, 40, torch.bfloat16)
    for args, kw, msg in (((x, wg, wu, wd), dict(activation="relu"), "activation"), ((x[:, :32], wg, wu, wd), {}, "columns"),
                          ((x, wg, wu[:50], wd), {}, "w_up"), ((x, wg, wu, wd[:, :50]), {}, "w_down"),
                          ((x.float(), wg, wu, wd), {}, "one dtype"), ((x, wg, wu.float(), wd), {}, "one dtype"),
                          ((x.half(), wg.half(), wu.half(), wd.half()), {}, "dtype"),
                          ((x.cpu(), wg.cpu(), wu.cpu(), wd.cpu()), {}, "CUDA"), ((x, wg, wu, wd.cpu()), {}, "one device"),
                          ((x, wg[:0], wu[:0], wd[:, :0]), {}, "rows and columns"), ((x, wg, wu, wd[0]), {}, "w_down"),
                          # (sizes that 32 bits would take for small ones; the rows are one row)
                          ((x[:1].expand(2**32 + 4, 64), wg, wu, wd), {}, "too large"),
                          ((x, wg, wu, wd[:1].expand(2**32 + 4, 96)), {}, "too large")):
        with pytest.raises(RuntimeError, match=msg):
            gated_mlp(*args, **kw)
    with pytest.raises(RuntimeError, match=r"status 1\): gated: unknown activation 7"):
        lm_ops._native.gated(x, wg, wu, wd, 7)  # the library's own refusal, through the native path


@pytest.mark.parametrize("dt", DTYPES, ids=("bf16", "f32"))
@pytest.mark.parametrize("which", ["w_gate", "w_up", "w_down"])
@pytest.mark.parametrize("n", [1, 8, 16, 30])
def test_weights_behind_a_kernel_that_is_still_writing(n, which, dt):
    """A weight that the library's launch just ahead writes, to the same memory in every step."""
    d = ff = 520
    x, *weights, _ = tensors(n, d, ff, d, dt, seed=n)
    at = ("w_gate", "w_up", "w_down").index(which)
    table = (torch.randn(2048, d, device="cuda") / d ** 0.5).to(dt)
    ids = torch.randint(0, 2048, (40, ff), device="cuda")

    def step(i):
        own = list(weights)
        own[at] = token_embedding(i, table)
        return gated_mlp(x, *own)

    with torch.no_grad():
        want = []
        for i in ids:
            weights[at] = token_embedding(i, table)
            torch.cuda.synchronize()
            want.append(gated_mlp(x, *weights))
            torch.cuda.synchronize()
        got = [step(i) for i in ids]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            replayed = [step(i) for i in ids]
        for _ in range(3):
            graph.replay()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, replayed))
