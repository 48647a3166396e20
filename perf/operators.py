"""What is measured of the training operators: the loss of the tied output head
(``linear_cross_entropy``: projection, softmax cross-entropy and their
gradients without the [tokens, vocabulary] logits) and the orthogonalised
update of the hidden matrices (``newton_schulz``).

``own`` false: plain torch operations in 32 bits, rounded once at the end.
``own`` true: the calls a user makes of this package.
"""

import math

import torch

own = False

IGNORE = -100
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _loss(name, tokens, d, vocab, dtype="bf16", train=True, ignored=0.0, accumulate=1):
    return {"name": name, "op": "loss", "tokens": tokens, "d": d, "vocab": vocab, "dtype": dtype, "train": train,
            "ignored": ignored, "accumulate": accumulate}


def _update(name, rows, cols, count, dtype="bf16"):
    return {"name": name, "op": "update", "rows": rows, "cols": cols, "count": count, "dtype": dtype}


def listed():
    return [
        # the next token's log-probability of one sequence: one row against the whole vocabulary, latency and W's bytes
        _loss("score_one_token", 1, 1536, 32000, train=False),
        # evaluation of one 2048-token sequence: per-token losses, no gradient
        _loss("score_sequence", 2048, 1536, 32000, train=False),
        # a toy LM step in fp32 (byte-sized vocabulary): launch-bound
        _loss("train_toy_f32", 512, 128, 128, dtype="f32"),
        # the fp32 step of a small model
        _loss("train_f32", 2048, 1024, 8192, dtype="f32"),
        # one short batch: few rows against a large vocabulary, both gradients
        _loss("train_few_tokens", 129, 1536, 32000),
        # a packed batch with padding, odd sizes, one of four accumulated micro-batches
        _loss("train_padded", 4095, 1408, 32003, ignored=0.2, accumulate=4),
        # the 24-layer LM's step: batch 16 x 2048 tokens, vocabulary 32000
        _loss("train_full", 32768, 1536, 32000),
        # the latent query projection of one layer: a flat matrix, latency
        _update("update_latent", 64, 1536, 1),
        # a small model's square projections
        _update("update_small", 256, 256, 4, dtype="f32"),
        # odd sizes, tall, gradients in fp32
        _update("update_odd", 1001, 777, 3, dtype="f32"),
        # the output projections of the 24-layer LM
        _update("update_square", 1536, 1536, 24),
        # the fused qkv projections of 12 layers (tall)
        _update("update_qkv", 4608, 1536, 12),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = "f32" if rng.random() < 0.3 else "bf16"
    if rng.random() < 0.55:
        tokens, d, vocab = _spread(rng, 1, 16384), _spread(rng, 64, 2048), _spread(rng, 97, 40000)
        if rng.random() < 0.7:
            d = max(64, d // 8 * 8)
        if dtype == "f32":
            tokens, vocab = max(1, tokens // 8), max(97, vocab // 4)
        return {"op": "loss", "tokens": tokens, "d": d, "vocab": vocab, "dtype": dtype, "train": rng.random() < 0.75,
                "ignored": rng.choice((0.0, 0.0, 0.1, 0.5)), "accumulate": rng.choice((1, 1, 2))}
    rows, cols = _spread(rng, 16, 4096), _spread(rng, 16, 4096)
    if rng.random() < 0.6:
        rows, cols = max(16, rows // 8 * 8), max(16, cols // 8 * 8)
    count = _spread(rng, 1, 24)
    while count > 1 and count * rows * cols > 12 * 4608 * 1536:
        count -= 1
    return {"op": "update", "rows": rows, "cols": cols, "count": count, "dtype": dtype}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if case["op"] == "loss":
        n, d, v = case["tokens"], case["d"], case["vocab"]
        # rows of the final norm (unit rms) that lean towards their target's
        # embedding, some much and some not at all: losses from near 0 to past log(vocab)
        w = randn(v, d) * (2.0 / math.sqrt(d))
        t = torch.randint(0, v, (n,), generator=gen, device="cuda")
        x = randn(n, d) + rand(n, 1) * 3.0 * w[t]
        x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-6)
        if case["ignored"]:
            t = torch.where(rand(n) < case["ignored"], torch.full_like(t, IGNORE), t)
        x, w = x.to(dt), w.to(dt)
        if case["train"]:
            x.requires_grad_(True)
            w.requires_grad_(True)
        return {"case": case, "x": x, "w": w, "targets": t}
    # momentum-like matrices: a decaying spectrum over a noise floor, each at its own scale
    m, n = case["rows"], case["cols"]
    k = min(m, n)
    decay = torch.arange(1, k + 1, device="cuda").float() ** -0.7
    gs = []
    for i in range(case["count"]):
        low = (randn(m, k) * decay) @ randn(k, n)
        g = low * (0.5 / low.square().mean().sqrt()) + 0.5 * randn(m, n)
        gs.append((g * 10.0 ** (-1 - i % 4)).to(dt))
    return {"case": case, "gs": gs}


def _plain_loss(x, w, targets, ignored, accumulate, train):
    """Loss (the mean over the tokens that count, or per token), and the
    gradients of loss / accumulate."""
    xf, wf = x.detach().float(), w.detach().float()
    keep = targets != IGNORE
    at = torch.where(keep, targets, torch.zeros_like(targets))
    logits = xf @ wf.t()
    top = logits.max(dim=1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(dim=1, keepdim=True)
    per = (top + torch.log(total) - logits.gather(1, at[:, None]))[:, 0]
    per = torch.where(keep, per, torch.zeros_like(per))
    if not train:
        return per
    count = keep.sum().clamp(min=1).float()
    scale = keep.float() / count / accumulate
    grad = e.mul_((scale / total[:, 0])[:, None])
    grad.scatter_add_(1, at[:, None], -scale[:, None])
    return per.sum() / count, (grad @ wf).to(x.dtype), (grad.t() @ xf).to(w.dtype)


def _plain_update(g):
    a, b, c = COEFFICIENTS
    x = g.float()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.square().sum().sqrt() + EPS)
    for _ in range(STEPS):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.t() if tall else x).to(torch.bfloat16)


def run(state):
    case = state["case"]
    if case["op"] == "loss":
        x, w, targets = state["x"], state["w"], state["targets"]
        if not own:
            got = _plain_loss(x, w, targets, case["ignored"], case["accumulate"], case["train"])
            return {"loss": got[0], "dx": got[1], "dw": got[2]} if case["train"] else {"losses": got}
        from llattn_b200 import linear_cross_entropy

        if not case["train"]:
            return {"losses": linear_cross_entropy(x, w, targets, ignore_index=IGNORE, reduction="none")}
        loss = linear_cross_entropy(x, w, targets, ignore_index=IGNORE)
        dx, dw = torch.autograd.grad(loss / case["accumulate"] if case["accumulate"] > 1 else loss, (x, w))
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    if not own:
        return [_plain_update(g) for g in state["gs"]]
    from llattn_b200 import newton_schulz

    return newton_schulz(state["gs"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)


def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "loss":
        n, d, v = case["tokens"], case["d"], case["vocab"]
        kept = n * (1.0 - case["ignored"])
        once = size * (n * d + v * d) + 8 * n
        if not case["train"]:
            return {"bytes": once + 4 * n, "flops": 2.0 * kept * v * d}
        return {"bytes": once + size * (n * d + v * d) + 4, "flops": 6.0 * kept * v * d}
    # the Gram matrix and its square are symmetric: half of their products are wanted
    m, n = sorted((case["rows"], case["cols"]))
    one = STEPS * (1.0 * m * m * n + 1.0 * m * m * m + 2.0 * m * m * n)
    return {"bytes": case["count"] * m * n * (size + 2), "flops": case["count"] * one}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "loss":
        x, w, targets = state["x"].detach().double(), state["w"].detach().double(), state["targets"]
        counted = torch.nonzero(targets != IGNORE)[:, 0]
        xs, ts = x[counted], targets[counted]
        rows = torch.arange(len(counted), device=x.device)
        z = torch.mm(xs, w.mT)
        lse = torch.logsumexp(z, dim=1)
        losses = lse - z[rows, ts]
        if not case["train"]:
            per = torch.zeros(len(targets), dtype=torch.float64, device=x.device)
            per[counted] = losses
            return {"losses": per}
        share = 1.0 / max(1, len(counted))
        p = torch.exp_(z.sub_(lse[:, None]))
        p[rows, ts] -= 1.0
        p *= share / case["accumulate"]
        dx = torch.zeros_like(x)
        dx[counted] = torch.mm(p, w)
        return {"loss": losses.sum() * share, "dx": dx, "dw": torch.mm(p.mT, xs)}
    a, b, c = COEFFICIENTS
    outs = []
    for g in state["gs"]:
        y = g.double()
        flip = y.shape[0] > y.shape[1]
        if flip:
            y = y.mT
        y = y / (torch.linalg.matrix_norm(y) + EPS)
        for _ in range(STEPS):
            gram = torch.mm(y, y.mT)
            poly = torch.mm(gram, gram).mul_(c).add_(gram, alpha=b)
            y = torch.addmm(y, poly, y, beta=a)
        outs.append(y.mT if flip else y)
    return outs
