"""token_embedding on the GPU against its formulas in 64 bits, entry by entry.

Bounds (u: the output type's rounding, 2^-8 or 2^-24): out is one fp32 fused product-sum and one rounding,
(u + 2^-23) |out| + 2^-24 |scale w|. A word's gradient of c tokens is at most 64 fp32 additions of rows, then c / 64 of
sums: 2^-24 (66 + c / 64) of the absolute sum, one product by the scale, one rounding. A position's: at most
batch additions, 2^-24 (batch + 2), one rounding."""

import pytest
import torch
import torch.nn.functional as F

from llattn_b200 import token_embedding

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float32


def unit(dt):
    return 2.0 ** -8 if dt == BF else 2.0 ** -24


def make(b, t, d, v, dt, seed=0, positions=True, skew=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dt)
    if skew:
        ids = (v ** torch.rand(b, t, generator=gen, device="cuda") - 1).long().clamp_(0, v - 1)
    else:
        ids = torch.randint(0, v, (b, t), generator=gen, device="cuda")
    return ids, r(v, d), r(t, d) if positions else None, r(b, t, d)


def run(ids, w, pos, dout, **kw):
    w = w.detach().requires_grad_(True)
    leaves = [w] if pos is None else [w, pos.detach().requires_grad_(True)]
    out = token_embedding(ids, w, positions=None if pos is None else leaves[1], **kw)
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


def check(got, ids, w, pos, dout, scale=1.0, padding_idx=None):
    v, d = w.shape
    b, t = ids.shape
    u = unit(w.dtype)
    ids = ids.long()
    ok = (ids >= 0) & (ids < v)
    rows = scale * F.embedding(ids.clamp(0, v - 1), w.double())
    want = rows if pos is None else rows + pos.double()[:t]
    off = (got[0].double() - want).abs()
    assert (off <= (u + 2.0 ** -23) * want.abs() + 2.0 ** -24 * rows.abs())[ok].all()
    assert got[0][~ok].isnan().all()
    flat, g = ids.reshape(-1), dout.double().reshape(-1, d)
    keep = ok.reshape(-1)
    if padding_idx is not None:
        keep = keep & (flat != padding_idx % v)
    flat, g = flat[keep], g[keep]
    dw = scale * torch.zeros(v, d, dtype=torch.float64, device="cuda").index_add_(0, flat, g)
    size = abs(scale) * torch.zeros_like(dw).index_add_(0, flat, g.abs())
    count = torch.bincount(flat, minlength=v)[:, None].double()
    assert ((got[1].double() - dw).abs() <= u * dw.abs() + 2.0 ** -24 * (66 + count / 64) * size).all()
    assert (got[1][count[:, 0] == 0] == 0).all()
    if pos is not None:
        dp, size = dout.double().sum(0), dout.double().abs().sum(0)
        assert got[2].shape == pos.shape and (got[2][t:] == 0).all()
        assert ((got[2][:t].double() - dp).abs() <= u * dp.abs() + 2.0 ** -24 * (b + 2) * size).all()


@pytest.mark.parametrize("dt", (BF, FP), ids=("bf16", "f32"))
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (1, 1, 8, 3), (3, 5, 7, 11), (4, 128, 128, 128), (2, 33, 24, 5000), (16, 64, 130, 50),
                                  (1, 700, 65, 40), (70, 1, 256, 33), (300, 9, 40, 1), (5, 1000, 520, 1283), (37, 129, 1024, 3001),
                                  (2, 3, 2056, 40001)], ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(size, dt):
    for positions in (True, False):
        ins = make(*size, dt, seed=sum(size), positions=positions)
        check(run(*ins), *ins)
        check(run(*ins, scale=size[2] ** 0.5, padding_idx=-1), *ins, scale=size[2] ** 0.5, padding_idx=-1)


@pytest.mark.parametrize("dt", (BF, FP), ids=("bf16", "f32"))
@pytest.mark.parametrize("n", (64, 65, 128, 129, 1000, 4096))
def test_frequent_words(n, dt):
    """Words at, below and above what one warp sums, ending and starting anywhere in the pieces of the sorted order."""
    ids, w, _, dout = make(1, n, 136, 40, dt, seed=n, positions=False)
    for same in (lambda i: i * 0 + 7, lambda i: i % 2, lambda i: (i // 65), lambda i: (i % 3 == 0) * 5, lambda i: (i * i) // 997):
        ids = same(torch.arange(n, device="cuda"))[None].clamp(max=39)
        check(run(ids, w, None, dout), ids, w, None, dout)
    ids = make(1, n, 1, 40, dt, seed=n, skew=True)[0]
    check(run(ids, w, None, dout, padding_idx=0), ids, w, None, dout, padding_idx=0)


def test_large_vocabulary_and_zipf():
    # past one wave of word ranges, and past what a sorting CTA's counters hold
    ids, w, pos, dout = make(6, 777, 16, 300001, BF, skew=True)
    check(run(ids, w, pos, dout), ids, w, pos, dout)
    ids, w, pos, dout = make(16, 2048, 264, 32000, FP, skew=True)
    check(run(ids, w, pos, dout), ids, w, pos, dout)


def test_exact_in_fp32_without_scale():
    """One rounding of w + p: torch's own sum; rows of single tokens are copied."""
    ids, w, pos, dout = make(4, 100, 72, 5000, FP)
    assert torch.equal(token_embedding(ids, w, positions=pos), F.embedding(ids, w) + pos)
    assert torch.equal(token_embedding(ids, w), F.embedding(ids, w))


@pytest.mark.parametrize("dt", (BF, FP), ids=("bf16", "f32"))
def test_bad_ids(dt):
    ids, w, pos, dout = make(3, 50, 40, 100, dt)
    for k, bad in enumerate((-1, 100, -100, 2 ** 40, -(2 ** 62), 2 ** 31 + 5)):
        ids[k % 3, 7 * k] = bad
    check(run(ids, w, pos, dout), ids, w, pos, dout)
    ids[:] = -5
    check(run(ids, w, pos, dout, padding_idx=3), ids, w, pos, dout, padding_idx=3)


def test_strides_types_and_shapes():
    ids, w, pos, dout = make(6, 20, 40, 90, BF)
    want = run(ids, w, pos, dout)
    wide = torch.full((92, 51), float("nan"), dtype=BF, device="cuda")
    wide[1:91, 3:43] = w
    table = torch.full((31, 48), float("nan"), dtype=BF, device="cuda")
    table[5:25, 8:] = pos
    got = run(ids.int(), wide[1:91, 3:43], table[5:25, 8:], dout)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = run(ids.t().contiguous().t(), w, pos, dout.transpose(0, 1).contiguous().transpose(0, 1))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    shifted = torch.empty(dout.numel() + 1, dtype=BF, device="cuda")[1:].view(dout.shape)
    shifted.copy_(dout)
    got = run(ids, w, pos, shifted)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # more positions than the length; one id; other shapes; broadcast upstream gradients
    long = torch.cat([pos, pos])
    check(run(ids, w, long, dout), ids, w, long, dout)
    check(run(ids, w, pos, torch.ones((), dtype=BF, device="cuda").expand(dout.shape)), ids, w, pos, torch.ones_like(dout))
    assert torch.equal(token_embedding(ids.view(2, 3, 20), w, positions=pos).view(6, 20, 40), want[0])
    assert torch.equal(token_embedding(ids[0], w, positions=pos), want[0][0])
    assert torch.equal(token_embedding(ids[0, 3], w), w[ids[0, 3]])
    assert torch.equal(token_embedding(ids[:, 4:5], w, positions=pos[4:5]), want[0][:, 4:5])
    for empty in (ids[:0], ids[:, :0]):
        assert token_embedding(empty, w, positions=pos).shape == (*empty.shape, 40)
        leaf = w.detach().requires_grad_(True)
        (dw,) = torch.autograd.grad(token_embedding(empty, leaf).sum(), leaf)
        assert dw.shape == w.shape and (dw == 0).all()


def test_one_gradient_only_and_same_bits():
    ids, w, pos, dout = make(9, 300, 136, 700, BF, skew=True)
    full = run(ids, w, pos, dout)
    for _ in range(2):
        again = run(ids, w, pos, dout)
        assert all(torch.equal(a, b) for a, b in zip(full, again))
    leaf = w.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(token_embedding(ids, leaf, positions=pos), leaf, dout)[0], full[1])
    both = (leaf, pos.detach().requires_grad_(True))  # of two that have one, one at a time
    for k in range(2):
        assert torch.equal(torch.autograd.grad(token_embedding(ids, both[0], positions=both[1]), both[k], dout)[0], full[1 + k])
    leaf = pos.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(token_embedding(ids, w, positions=leaf), leaf, dout)[0], full[2])


def test_gradient_of_a_sum_by_differences():
    """The operator is linear: its gradient along a direction is the difference itself."""
    ids, w, pos, dout = make(5, 60, 48, 70, FP, skew=True)
    _, dw, dp = run(ids, w, pos, dout, scale=3.0)
    vw, vp = torch.randn_like(w), torch.randn_like(pos)
    diff = (token_embedding(ids, w + vw, positions=pos + vp, scale=3.0).double()
            - token_embedding(ids, w - vw, positions=pos - vp, scale=3.0).double()) / 2
    a, b = (diff * dout.double()).sum(), (dw.double() * vw.double()).sum() + (dp.double() * vp.double()).sum()
    # each of the 14400 outputs is off by some 2^-23 of values up to 20
    assert (a - b).abs() <= 2.0 ** -23 * 20 * (dout.double().abs().sum() + dw.abs().sum() + dp.abs().sum())


def test_graphs_streams_and_compile():
    ids, w, pos, dout = make(4, 500, 64, 300, FP, skew=True)
    want = run(ids, w, pos, dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(ids, w, pos, dout)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(ids, w, pos, dout)
    ids.copy_((ids * 7 + 1) % 300)
    want2 = run(ids, w, pos, dout)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want2))
    f = torch.compile(lambda i, a, b: token_embedding(i, a, positions=b, scale=2.0), backend="aot_eager", fullgraph=True)
    leaves = [w.detach().requires_grad_(True), pos.detach().requires_grad_(True)]
    out = f(ids, *leaves)
    eager = run(ids, w, pos, dout, scale=2.0)
    got = (out.detach(), *torch.autograd.grad(out, leaves, dout))
    assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_graph_kept_freed_and_hooked():
    ids, w, pos, dout = make(3, 40, 24, 30, FP)
    leaves = (w.requires_grad_(True), pos.requires_grad_(True))
    out = token_embedding(ids, leaves[0], positions=leaves[1])
    first = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    again = torch.autograd.grad(out, leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, leaves, dout)
    with torch.autograd.graph.save_on_cpu():
        out = token_embedding(ids, leaves[0], positions=leaves[1])
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(out, leaves, dout)))
    out = token_embedding(ids, leaves[0], positions=leaves[1])
    (dw,) = torch.autograd.grad(out, leaves[0], dout.requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        dw.sum().backward()
    out = token_embedding(ids, leaves[0])
    ids[0, 0] += 1  # (what the backward reads)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_refusals():
    ids, w, pos, _ = make(3, 8, 16, 20, BF)
    for args, kw, msg in (((ids.float(), w), {}, "int64"), ((ids.bool(), w), {}, "int64"), ((ids, w[0]), {}, "weight"),
                          ((ids, w.half()), {}, "dtype"), ((ids, w), dict(positions=pos[:7]), "positions"),
                          ((ids, w), dict(positions=pos[:, :8]), "positions"), ((ids, w), dict(positions=pos.float()), "one dtype"),
                          ((ids[0, 0], w), dict(positions=pos), "dimension"), ((ids, w), dict(padding_idx=20), "padding_idx"),
                          ((ids, w), dict(padding_idx=-21), "padding_idx"), ((ids.cpu(), w), {}, "one device"),
                          ((ids.cpu(), w.cpu()), {}, "CUDA"), ((ids, w), dict(positions=pos.cpu()), "one device"),
                          ((ids, w[:0]), {}, "rows and columns"), ((ids[:1].expand(2**32 + 1, 8), w), {}, "too large"),
                          ((ids, w[:1].expand(2**32 + 4, 16)), {}, "too large"),
                          ((ids, w), dict(positions=pos[:1].expand(2**32 + 8, 16)), "too many")):
        with pytest.raises(RuntimeError, match=msg):
            token_embedding(*args, **kw)


@pytest.mark.parametrize("n,v", [(256, 4), (2048, 4), (2048, 5000), (4096, 4), (65536, 5000), (1 << 20, 40)])
@pytest.mark.parametrize("large", ["first", "each 256th", "last"])
def test_a_words_sum_is_not_one_chain(n, v, large):
    """Rows that vanish one by one beside a large one, and not together: a sum of n additions in a row would be off by n
    half steps. Rows in pairs of pairs (8 and 2 additions for 32 of them), then such sums 32 at a time (31), then
    c / 1024; small calls n / 32, 2 and 8: within 66 + c / 64."""
    for small in (0.99 * 2.0 ** -24, 0.99 * 2.0 ** -29):  # of the large row: below its half step alone, or 32 of them
        dout = torch.full((1, n, 8), small, device="cuda")
        dout[0, {"first": slice(0, 1), "each 256th": slice(0, None, 256), "last": slice(-1, None)}[large]] = 1.0
        ids = torch.full((1, n), 1, device="cuda")
        w = torch.zeros(v, 8, device="cuda", requires_grad=True)
        (dw,) = torch.autograd.grad(token_embedding(ids, w), w, dout)
        want = dout.double().sum((0, 1))
        assert ((dw[1].double() - want).abs() <= 2.0 ** -24 * (67 + n / 64) * want).all()
        assert (dw[0] == 0).all() and (dw[2:] == 0).all()
