"""clip_grad_norm_ and total_norm on the GPU against 64 bits.

Bounds: a 16-byte vector's squares are summed by up to 8 fp32 operations, all else in fp64: the square of the norm is within
8 2^-24, the norm within 4 2^-24 and its own rounding, 5 2^-24. A scaled element: the factor (4 2^-24 and its rounding), the
product's rounding, and for bf16 the result's 2^-8: (7 2^-24 + u)."""

import pytest
import torch

from llattn_b200 import clip_grad_norm_, total_norm

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float32
NORM = 5 * 2.0 ** -24


def unit(dt):
    return 2.0 ** -8 if dt == BF else 0.0


def tiny(dt):
    """Below 2^-126 a result is rounded to a multiple of 2^-149 (fp32) or 2^-133 (bf16): half of that is its error."""
    return 2.0 ** -150 + (2.0 ** -134 if dt == BF else 0.0)


def params(shapes, dts, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i, s in enumerate(shapes):
        dt = dts[i % len(dts)]
        p = torch.nn.Parameter(torch.empty(s, dtype=dt, device="cuda"))
        p.grad = (torch.randn(s, generator=gen, device="cuda") * (scale * (1 + i % 5))).to(dt)
        out.append(p)
    return out


def norm64(grads, kind=2.0):
    flat = torch.cat([g.double().reshape(-1) for g in grads])
    return torch.linalg.vector_norm(flat, kind)


def check(ps, max_norm, kind=2.0):
    before = [p.grad.clone() for p in ps]
    want = norm64(before, kind)
    norm = clip_grad_norm_(ps, max_norm, kind)
    assert norm.dtype == FP and norm.shape == () and abs(norm.item() / want.item() - 1) <= NORM if want else norm.item() == 0
    f = min(1.0, max_norm / (want.item() + 1e-6))
    for p, g in zip(ps, before):
        off = (p.grad.double() - f * g.double()).abs()
        # (a bf16 result may round the other way where the factor's last bits decide: within its half step all the same)
        assert (off <= (unit(g.dtype) + 7 * 2.0 ** -24) * f * g.double().abs() + tiny(g.dtype)).all()
        if f == 1.0:
            assert torch.equal(p.grad, g)


SHAPES = [[(1,)], [(3,)], [(5, 7), (1,), (0,), (16,), (4096,), (4097,)], [(17, 33)] * 70, [(1024, 1025), (3, 1), (2, 4096)],
          [(n,) for n in range(1, 150)]]


@pytest.mark.parametrize("dts", ((FP,), (BF,), (BF, FP)), ids=("f32", "bf16", "mixed"))
@pytest.mark.parametrize("shapes", SHAPES, ids=range(len(SHAPES)))
def test_norm_and_clipping(shapes, dts):
    for kind in (2.0, float("inf")):
        for max_norm in (0.5, 1e9, 0.0):
            check(params(shapes, dts, seed=len(shapes)), max_norm, kind)


@pytest.mark.parametrize("count", (1299, 1300, 1301, 2601))
def test_more_tensors_than_a_launch_holds(count):
    ps = params([(1 + i % 37,) for i in range(count)], (FP, BF), seed=count)
    check(ps, 0.25)
    ps = params([(1 + i % 37,) for i in range(count)], (FP, BF), seed=count)
    want = norm64([p.grad for p in ps])
    assert abs(total_norm([p.grad for p in ps]).item() / want.item() - 1) <= NORM


@pytest.mark.parametrize("dt", (BF, FP), ids=("bf16", "f32"))
def test_views_of_a_bucket(dt):
    """Gradients one after the other in one buffer, starting and ending anywhere; what lies between them stays."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    sizes = [1, 2, 3, 5, 7, 8, 9, 31, 8191, 8192, 8193, 16385, 40000, 6, 1]
    for gap in (0, 1, 3):
        bucket = torch.randn(sum(sizes) + gap * len(sizes), generator=gen, device="cuda").to(dt)
        before, at, ps = bucket.clone(), 0, []
        outside = torch.ones_like(bucket, dtype=torch.bool)
        for n in sizes:
            p = torch.nn.Parameter(torch.empty(n, dtype=dt, device="cuda"))
            p.grad = bucket[at:at + n]
            outside[at:at + n] = False
            ps.append(p)
            at += n + gap
        check(ps, 1.5)
        assert torch.equal(bucket[outside], before[outside])


@pytest.mark.parametrize("dt", (BF, FP), ids=("bf16", "f32"))
@pytest.mark.parametrize("size", (1e-30, 1e-22, 1e-18, 1e18, 1e30))
def test_far_magnitudes(size, dt):
    """Squares outside fp32's range."""
    ps = params([(333, 77), (5,), (40,)], (dt,), scale=size)
    ps[2].grad.zero_()
    want = norm64([p.grad for p in ps])
    got = total_norm([p.grad for p in ps])
    assert abs(got.item() / want.item() - 1) <= NORM
    check(ps, size)


@pytest.mark.parametrize("dt", (BF, FP), ids=("bf16", "f32"))
def test_infinities_and_nan(dt):
    for bad, kind in ((float("nan"), 2.0), (float("nan"), float("inf")), (float("inf"), 2.0), (float("-inf"), float("inf"))):
        for at in (0, 4999):
            ps = params([(5000,), (7,)], (dt,))
            ps[0].grad[at] = bad
            before = [p.grad.clone() for p in ps]
            with pytest.raises(RuntimeError, match="not finite"):
                clip_grad_norm_(ps, 1.0, kind, error_if_nonfinite=True)
            assert torch.equal(ps[1].grad, before[1])
            ref = [torch.nn.Parameter(torch.empty_like(g)) for g in before]
            for r, g in zip(ref, before):
                r.grad = g.clone()
            want = torch.nn.utils.clip_grad_norm_(ref, 1.0, kind)
            norm = clip_grad_norm_(ps, 1.0, kind)
            assert norm.isnan().item() == want.isnan().item() and norm.isinf().item() == want.isinf().item()
            for p, r in zip(ps, ref):
                assert torch.equal(p.grad.isnan(), r.grad.isnan()) and torch.equal(p.grad.nan_to_num() == 0, r.grad.nan_to_num() == 0)


def test_against_torch():
    ps, ref = params([(300, 77), (64,), (1, 9)], (FP,), seed=9), params([(300, 77), (64,), (1, 9)], (FP,), seed=9)
    ref[1].grad, ps[1].grad = None, None
    a, b = clip_grad_norm_(iter(ps), 2.0), torch.nn.utils.clip_grad_norm_(ref, 2.0)
    assert abs(a.item() / b.item() - 1) < 1e-6
    for p, r in zip(ps, ref):
        assert p.grad is r.grad is None or torch.allclose(p.grad, r.grad, rtol=1e-6, atol=0)
    single = params([(50,)], (FP,))[0]
    assert abs(clip_grad_norm_(single, 0.1).item() / norm64([params([(50,)], (FP,))[0].grad]).item() - 1) <= NORM
    assert clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0) == 0 and total_norm([]) == 0
    p = torch.nn.Parameter(torch.zeros(0, device="cuda"))
    p.grad = torch.zeros(0, device="cuda")
    assert clip_grad_norm_([p], 1.0).item() == 0


def test_layouts():
    a, b, c = params([(40, 30), (4, 5, 6, 7), (64, 16)], (FP,))
    a.grad = torch.randn(30, 40, device="cuda").t()
    b.grad = torch.randn(4, 5, 6, 7, device="cuda").to(memory_format=torch.channels_last)
    wide = torch.randn(64, 48, device="cuda")
    keep = wide.clone()
    c.grad = wide[:, 8:24]
    check([a, b, c], 1.0)
    assert torch.equal(wide[:, :8], keep[:, :8]) and torch.equal(wide[:, 24:], keep[:, 24:])
    # a parameter given twice counts once
    (p,) = params([(100,)], (FP,))
    want = norm64([p.grad])
    assert abs(clip_grad_norm_([p, p], 1.0).item() / want.item() - 1) <= NORM
    assert abs(norm64([p.grad]).item() - 1) < 1e-5


def test_same_bits_graphs_streams_and_compile():
    shapes = [(700, 300), (11,), (5000,)]
    one, two = (clip_grad_norm_(ps, 1.0) for ps in (params(shapes, (FP, BF)), params(shapes, (FP, BF))))
    assert torch.equal(one, two)
    ps = params(shapes, (FP,))
    source = [p.grad.clone() for p in ps]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip_grad_norm_(ps, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(ps, 1.0)
    for k in (2.0, 5.0):
        for p, s in zip(ps, source):
            p.grad.copy_(s * k)
        graph.replay()
        assert abs(norm.item() / (k * norm64(source).item()) - 1) <= NORM + 2.0 ** -23
        assert abs(norm64([p.grad for p in ps]).item() - 1) < 1e-5
    f = torch.compile(lambda ts: total_norm(ts), backend="aot_eager", fullgraph=True)
    assert torch.equal(f(source), total_norm(source))


def test_autograd_sees_the_change():
    ps = params([(10,), (4, 6)], (FP,))
    ps[1].grad = torch.randn(6, 4, device="cuda").t()  # (dense)
    wide = params([(4, 4)], (FP,))[0]
    wide.grad = torch.randn(4, 9, device="cuda")[:, 2:6]  # (not dense: by way of a copy)
    w = torch.ones(10, device="cuda", requires_grad=True)
    y = (w * ps[0].grad).sum()  # saves the gradient
    before = [p.grad._version for p in (*ps, wide)]
    clip_grad_norm_([*ps, wide], 0.1)
    assert all(p.grad._version > v for p, v in zip((*ps, wide), before))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    version = ps[0].grad._version
    total_norm([p.grad for p in ps])
    assert ps[0].grad._version == version


def test_refusals():
    (p, q) = params([(10,), (10,)], (FP,))
    for kw, msg in ((dict(max_norm=-1.0), "max_norm"), (dict(max_norm=float("nan")), "max_norm"),
                    (dict(max_norm=1.0, norm_type=1), "norm_type"), (dict(max_norm=1.0, norm_type=3.0), "norm_type")):
        with pytest.raises(RuntimeError, match=msg):
            clip_grad_norm_([p], **kw)
    buf = torch.randn(15, device="cuda")
    p.grad, q.grad = buf[:10], buf[5:]
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_([p, q], 1.0)
    assert total_norm([buf[:10], buf[5:]]).item() > 0
    h = torch.nn.Parameter(torch.zeros(4, dtype=torch.half, device="cuda"))
    h.grad = torch.zeros_like(h)
    with pytest.raises(RuntimeError, match="dtype"):
        clip_grad_norm_([h], 1.0)
    c = torch.nn.Parameter(torch.zeros(4))
    c.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        clip_grad_norm_([c], 1.0)
    with pytest.raises(RuntimeError, match="one device"):
        clip_grad_norm_([q, c], 1.0)
    s = torch.nn.Parameter(torch.zeros(4, 4, device="cuda"))
    s.grad = torch.eye(4, device="cuda").to_sparse()
    with pytest.raises(RuntimeError, match="dense"):
        clip_grad_norm_([s], 1.0)


def through_c(tensors, norm_type=0, max_norm=1.0, scale=1):
    """llattn_clip with a workspace of exactly the size that it asks for, between guard bytes; returns the norm."""
    import ctypes

    from llattn_b200 import _lib

    n = len(tensors)
    args = _lib.ClipArgs(n, norm_type, scale, (ctypes.c_void_p * n)(*(t.data_ptr() for t in tensors)),
                         (ctypes.c_int64 * n)(*(t.numel() for t in tensors)),
                         (ctypes.c_int32 * n)(*(_lib.BF16 if t.dtype == BF else _lib.F32 for t in tensors)), max_norm)
    norm = torch.empty((), device="cuda")
    size = _lib.lib().llattn_clip_workspace_bytes(ctypes.byref(args))
    buf = torch.full((512 + size + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    args.norm, args.workspace, args.workspace_bytes = norm.data_ptr(), buf.data_ptr() + 512, size
    _lib.check(_lib.lib().llattn_clip(ctypes.byref(args), torch.cuda.current_stream().cuda_stream), "llattn_clip")
    assert (buf[:512] == 0xA5).all() and (buf[512 + size:] == 0xA5).all()
    return norm.item()


@pytest.mark.parametrize("before,after", ((0, 0), (0, 1), (3, 1500)))
@pytest.mark.parametrize("count", (0, 1, 96, 1299, 1300, 1301, 2600))
def test_empty_tensors_and_the_workspaces_size(count, before, after):
    """Empty tensors behind a full launch's make no further one: its sum would lie behind the workspace."""
    none = torch.empty(0, device="cuda")
    held = [p.grad for p in params([(1 + i % 37,) for i in range(count)], (FP, BF), seed=count)]
    want = norm64(held).item() if held else 0.0
    lists = [none] * before + held + [none] * after
    if lists:
        assert abs(through_c(lists, scale=0) - want) <= NORM * want
        assert abs(through_c(lists, max_norm=0.5) - want) <= NORM * want
    if held:  # clipped once (bf16: half a step an element)
        assert abs(norm64(held).item() / min(want, 0.5) - 1) <= 2.0 ** -8


@pytest.mark.parametrize("dt", (BF, FP), ids=("bf16", "f32"))
def test_a_norm_above_fp32s_range_is_infinite(dt):
    """Finite gradients whose norm no fp32 holds: infinity is returned and the gradients are 0, as torch's."""
    ps, ref = (params([(333, 77), (5,)], (dt,), seed=3) for _ in range(2))
    for p in (*ps, *ref):
        p.grad.fill_(3e38)
    for kind in (2.0, float("inf")):
        norm, want = clip_grad_norm_(ps, 1.0, kind), torch.nn.utils.clip_grad_norm_(ref, 1.0, kind)
        if kind == 2.0:
            assert norm.isinf() and want.isinf()
            assert all((p.grad == 0).all() for p in (*ps, *ref))
            with pytest.raises(RuntimeError, match="not finite"):
                ps[0].grad.fill_(3e38)
                clip_grad_norm_(ps, 1.0, kind, error_if_nonfinite=True)
            assert (ps[0].grad == torch.tensor(3e38, dtype=dt, device="cuda")).all()
        else:  # (the largest magnitude is finite)
            assert abs(norm.item() / 3e38 - 1) <= 2.0 ** -8
        for p in (*ps, *ref):
            p.grad.fill_(3e38)
    # just inside: as any other
    p = params([(4,)], (dt,))[0]
    p.grad.fill_(1e38)
    check([p], 3.0)


def test_given_twice_counts_once_in_the_check_too():
    p = torch.nn.Parameter(torch.zeros(1, device="cuda"))
    for kw in ({}, dict(error_if_nonfinite=True)):  # (twice it would be above fp32's range)
        p.grad = torch.full((1,), 3e38, device="cuda")
        norm = clip_grad_norm_([p, p], 1e38, **kw)
        assert abs(norm.item() / 3e38 - 1) <= NORM and abs(p.grad.item() / 1e38 - 1) <= 8 * 2.0 ** -24
