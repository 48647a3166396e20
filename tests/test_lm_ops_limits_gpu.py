"""gated_mlp, token_embedding and the clipping at their far ends: offsets past 32
bits, several threads and streams at once, results and inputs changed in place."""

from __future__ import annotations

import threading

import pytest
import torch

from llattn_b200 import clip_grad_norm_, gated_mlp, token_embedding, total_norm

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float32


def randn(*shape, dtype=FP, scale=1.0):
    return (torch.randn(*shape, device="cuda") * scale).to(dtype)


def test_gated_mlp_past_32_bits():
    """h, and what is kept of g and u, have more than 2^31 elements: rows far apart against the same rows alone."""
    n, d, ff = 540_000, 24, 4000
    assert n * ff > 2**31
    x, dy = randn(n, d, dtype=BF), randn(n, d, dtype=BF)
    wg, wu = randn(ff, d, dtype=BF, scale=d**-0.5), randn(ff, d, dtype=BF, scale=d**-0.5)
    wd = randn(d, ff, dtype=BF, scale=ff**-0.5)
    leaf = x.clone().requires_grad_(True)
    weights = [w.clone().requires_grad_(True) for w in (wg, wu, wd)]
    y = gated_mlp(leaf, *weights)
    dx, *dws = torch.autograd.grad(y, (leaf, *weights), dy)
    # the rows of the same tiles, which start at multiples of 4096: same products, same bits
    for first in (0, 262_144, n // 4096 * 4096):
        part = x[first:first + 4096].clone().requires_grad_(True)
        yp = gated_mlp(part, *weights)
        (dxp,) = torch.autograd.grad(yp, part, dy[first:first + 4096])
        for got, want in ((y[first:first + 4096], yp), (dx[first:first + 4096], dxp)):
            # (the schedule of the sums over ff may differ with the number of tiles: half a step of bf16 each, and of
            # fp32 sums of 4000 products that agree to 2^-12 of the largest)
            bound = 2.0**-8 * (got.double().abs() + want.double().abs()) / 2 + 2.0**-12 * want.double().abs().max()
            assert ((got.double() - want.double()).abs() <= bound + 2.0**-8 * want.double().abs()).all()
    # gradients of the weights: sums over pieces of the tokens in 64 bits
    want = [torch.zeros_like(w, dtype=torch.float64) for w in weights]
    size = [torch.zeros_like(w, dtype=torch.float64) for w in weights]
    for first in range(0, n, 30_000):
        s = slice(first, first + 30_000)
        xs, ds = x[s].double(), dy[s].double()
        g, u = xs @ wg.double().T, xs @ wu.double().T
        sig = torch.sigmoid(g)
        h, dh = g * sig * u, ds @ wd.double()
        dg, du = dh * u * sig * (1 + g * (1 - sig)), dh * g * sig
        for k, (a, b) in enumerate(((dg, xs), (du, xs), (ds, h))):
            want[k] += a.T @ b
            size[k] += a.square().T @ b.square()
    for got, w, s in zip(dws, want, size):
        # n independent roundings of the operands (half a step at most each, kept values 2^-11) add up as their
        # squares do; eight deviations of it, and the result's own rounding
        bound = 2.0**-8 * w.abs() + 8 * 2.0**-7 * s.sqrt() + 2.0**-14 * w.abs().max()
        assert ((got.double() - w).abs() <= bound).all()


@pytest.mark.parametrize("dt", (BF, FP), ids=("bf16", "f32"))
def test_token_embedding_past_32_bits(dt):
    b, t, d, v = 11, 131_072, 1536, 500
    assert b * t * d > 2**31
    w, pos = randn(v, d, dtype=dt).requires_grad_(True), randn(t, d, dtype=dt).requires_grad_(True)
    ids = torch.randint(0, v, (b, t), device="cuda", dtype=torch.int32)
    out = token_embedding(ids, w, positions=pos)
    for i in (0, b // 2, b - 1):
        for at in (0, t - 2000):
            s = slice(at, at + 2000)
            want = (w.detach().float()[ids[i, s].long()] + pos.detach().float()[s]).to(dt)
            assert torch.equal(out[i, s].detach(), want)
    dout = torch.zeros_like(out)
    dout[-1] = 1.0
    dout[0, -3:] = 2.0
    dw, dp = torch.autograd.grad(out, (w, pos), dout)
    count = torch.bincount(ids[-1].long(), minlength=v) + 2 * torch.bincount(ids[0, -3:].long(), minlength=v)
    assert torch.equal(dw, count.to(dt)[:, None].expand(v, d))  # (integers below 2^24, rounded once)
    want = torch.ones(t, device="cuda")
    want[-3:] += 2.0
    assert torch.equal(dp, want.to(dt)[:, None].expand(t, d))


def test_clipping_past_32_bits():
    p = torch.nn.Parameter(torch.empty(2**31 + 77, device="cuda", dtype=BF))
    p.grad = torch.zeros_like(p)
    p.grad[-5:] = 3.0
    p.grad[2**31 - 2] = 4.0
    q = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    q.grad = torch.full_like(q, 1.0)
    norm = (5 * 9.0 + 16.0 + 3.0) ** 0.5
    assert abs(float(total_norm([p.grad, q.grad])) - norm) <= 2.0**-23 * norm
    clip_grad_norm_([p, q], 0.5 * norm)
    assert torch.equal(p.grad[-5:], torch.full((5,), 1.5, device="cuda", dtype=BF)) and float(p.grad[2**31 - 2]) == 2.0
    assert int((p.grad != 0).sum()) == 6


def test_threads_and_streams_at_once():
    n, d, ff, v = 130, 136, 264, 700
    jobs, want = [], []
    for k in range(4):
        torch.manual_seed(k)
        x, dy = randn(n, d, dtype=BF), randn(n, d, dtype=BF)
        ws = [randn(ff, d, dtype=BF, scale=0.1), randn(ff, d, dtype=BF, scale=0.1), randn(d, ff, dtype=BF, scale=0.1)]
        table, ids = randn(v, d, dtype=BF), torch.randint(0, v, (3, n // 3), device="cuda")
        jobs.append((x, dy, ws, table, ids))

    def work(job):
        x, dy, ws, table, ids = job
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, *ws, table)]
        e = token_embedding(ids, leaves[4])
        y = gated_mlp(leaves[0], *leaves[1:4])
        torch.autograd.backward((y, e), (dy, torch.ones_like(e)))
        norm = clip_grad_norm_(leaves, 1.0)
        with torch.no_grad():
            few = gated_mlp(x[:3], *ws)
        return [y.detach(), e.detach(), few, norm, *(t.grad for t in leaves)]

    want = [work(j) for j in jobs]
    torch.cuda.synchronize()
    got, errors = [None] * len(jobs), []

    def run(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[k] = work(jobs[k])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 (shown by the assertion below)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(k,)) for k in range(len(jobs))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_changes_in_place():
    ids, w = torch.randint(0, 50, (2, 7), device="cuda"), randn(50, 16).requires_grad_(True)
    out = token_embedding(ids, w)
    out += 1.0
    out.mul_(2.0)
    (dw,) = torch.autograd.grad(out.sum(), w)
    assert torch.equal(dw[:, 0], 2.0 * torch.bincount(ids.flatten(), minlength=50).float())
    ws = [randn(24, 16), randn(24, 16), randn(16, 24)]
    x = randn(3, 5, 16).requires_grad_(True)
    (want,) = torch.autograd.grad(gated_mlp(x, *ws).sum(), x)
    y = gated_mlp(x, *ws)
    y.add_(x).mul_(2.0)  # (a result of three dimensions is a view)
    (dx,) = torch.autograd.grad(y.sum(), x)
    # (the upstream gradients are powers of two: the same products, doubled)
    assert torch.allclose(dx, 2.0 * want + 2.0, rtol=2.0**-22, atol=2.0**-21)
    # a weight that changes between the two is refused, as by torch's own operators
    leaf = ws[0].clone().requires_grad_(True)
    y = gated_mlp(x, leaf, *ws[1:])
    with torch.no_grad():
        leaf.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gated_mlp_loses_no_row_past_32_bits():
    """Gradients of a few rows alone, around element 2^31 of h and in the last, partial step of the sums over the tokens: a
    row that is lost or read elsewhere shows, which sums over all of them would hide."""
    n, d, ff = 540_000, 24, 4000
    rows = torch.tensor([0, 63, 2**31 // ff - 1, 2**31 // ff, 2**31 // ff + 1, n - 65, n - 64, n - 32, n - 2, n - 1], device="cuda")
    assert n % 64 == 32
    x, dy = randn(n, d, dtype=BF), torch.zeros(n, d, device="cuda", dtype=BF)
    dy[rows] = randn(len(rows), d, dtype=BF)
    weights = [randn(ff, d, dtype=BF, scale=d**-0.5), randn(ff, d, dtype=BF, scale=d**-0.5), randn(d, ff, dtype=BF, scale=ff**-0.5)]
    leaves = [t.requires_grad_(True) for t in (x, *weights)]
    y = gated_mlp(*leaves)
    dx, *dws = torch.autograd.grad(y, leaves, dy)
    xs, ds, wg, wu, wd = (t.detach().double() for t in (x[rows], dy[rows], *weights))
    g, u = xs @ wg.T, xs @ wu.T
    sig = torch.sigmoid(g)
    a, slope, dh = g * sig, sig * (1 + g * (1 - sig)), ds @ wd
    # operands rounded (2^-8) and kept values (2^-11 of each, |slope| and |g act''| below 1.2), results rounded (2^-8), sums:
    # 2^-6 of the absolute terms
    assert ((y[rows].double() - (a * u) @ wd.T).abs() <= 2.0**-6 * ((a * u).abs() @ wd.T.abs())).all()
    dg, du = dh * u * slope, dh * a
    size = 1.2 * (dh * u).abs() @ wg.abs() + (1.2 * (dh * g).abs() + du.abs()) @ wu.abs()
    assert ((dx[rows].double() - dg @ wg - du @ wu).abs() <= 2.0**-6 * size).all()
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert (dx[rest] == 0).all()
    for got, left, big, right in zip(dws, (dg, du, ds), ((dh * u).abs(), (dh * g).abs(), ds.abs()), (xs, xs, a * u)):
        extra = 1.2 * (g * u).abs() if right is not xs else right.abs()
        bound = 2.0**-6 * (1.2 * big.T @ extra.abs() + left.abs().T @ right.abs())
        assert ((got.double() - left.T @ right).abs() <= bound).all()
        # what any one of the rows adds is beyond the bound somewhere
        assert all(((left[r, :, None] * right[r]).abs() > 2 * bound).any() for r in range(len(rows)))
