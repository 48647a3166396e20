"""What is measured of the language model's operators around the attention
block: the gated feed-forward block (``gated_mlp``), the token embedding with
its positions and its gradients (``token_embedding``) and the clipping of the
gradients to a global norm (``clip_grad_norm_``).

``own`` false: plain torch operations in 32 bits, rounded once at the end.
``own`` true: the calls a user makes of this package.
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _mlp(name, tokens, d, ff, act="silu", dtype="bf16", train=True):
    return {"name": name, "op": "mlp", "tokens": tokens, "d": d, "ff": ff, "act": act, "dtype": dtype, "train": train}


def _embed(name, batch, length, d, vocab, dtype="f32", positions=True, padded=0.0, scale=1.0, train=True):
    return {"name": name, "op": "embed", "batch": batch, "length": length, "d": d, "vocab": vocab, "dtype": dtype,
            "positions": positions, "padded": padded, "scale": scale, "train": train}


def _clip(name, layers, d, ff, latent, vocab, dtype="f32", max_norm=1.0, spread=1.0):
    return {"name": name, "op": "clip", "layers": layers, "d": d, "ff": ff, "latent": latent, "vocab": vocab,
            "dtype": dtype, "max_norm": max_norm, "spread": spread}


def listed():
    return [
        # one layer's block for the next token of one sequence: the weights' bytes, latency
        _mlp("mlp_one_token", 1, 1536, 4096, train=False),
        # the next token of 24 sequences, sizes that no vector divides
        _mlp("mlp_few_tokens", 24, 1411, 3749, act="gelu", train=False),
        # a prompt of 2048 tokens
        _mlp("mlp_prompt", 2048, 1536, 4096, train=False),
        # the fp32 step of a small model, inner width 8/3 d
        _mlp("mlp_train_f32", 1000, 512, 1365, dtype="f32"),
        # a packed batch of odd sizes
        _mlp("mlp_train_odd", 4095, 1408, 3749, act="gelu"),
        # the 24-layer LM's step: batch 16 x 2048 tokens
        _mlp("mlp_train_full", 32768, 1536, 4096),
        # a toy LM with a byte-sized vocabulary: launches
        _embed("embed_toy", 4, 128, 128, 128),
        # bf16 weights, rows scaled by sqrt(d), no position table, a fifth of the batch padding
        _embed("embed_padded", 7, 1171, 1408, 32003, dtype="bf16", positions=False, padded=0.2, scale=1408.0 ** 0.5),
        # the 24-layer LM's embeddings: batch 16 x 2048 tokens, vocabulary 32000
        _embed("embed_full", 16, 2048, 1536, 32000),
        # the gradients of a toy LM of two layers
        _clip("clip_toy", 2, 128, 256, 64, 128),
        # bf16 gradients of odd sizes in one bucket: most tensors start off any vector's boundary
        _clip("clip_odd", 11, 515, 1371, 61, 5003, dtype="bf16", max_norm=0.5),
        # the gradients of the 24-layer LM (some 430 M fp32)
        _clip("clip_full", 24, 1536, 4096, 64, 32000),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = "f32" if rng.random() < 0.35 else "bf16"
    kind = rng.random()
    if kind < 0.5:
        tokens, d, ff = _spread(rng, 1, 16384), _spread(rng, 64, 2048), _spread(rng, 64, 6000)
        if rng.random() < 0.6:
            d, ff = max(64, d // 8 * 8), max(64, ff // 8 * 8)
        if dtype == "f32":
            tokens, ff = max(1, tokens // 8), max(64, ff // 2)
        return {"op": "mlp", "tokens": tokens, "d": d, "ff": ff, "act": rng.choice(("silu", "gelu")), "dtype": dtype,
                "train": rng.random() < 0.65}
    if kind < 0.75:
        length = _spread(rng, 1, 4096)
        batch = _spread(rng, 1, max(1, 32768 // length))
        d, vocab = _spread(rng, 24, 1536), _spread(rng, 97, 32000)
        if rng.random() < 0.6:
            d = max(24, d // 8 * 8)
        return {"op": "embed", "batch": batch, "length": length, "d": d, "vocab": vocab, "dtype": dtype,
                "positions": rng.random() < 0.6, "padded": rng.choice((0.0, 0.0, 0.1, 0.4)),
                "scale": rng.choice((1.0, d ** 0.5)), "train": rng.random() < 0.8}
    return {"op": "clip", "layers": _spread(rng, 1, 24), "d": _spread(rng, 48, 1400), "ff": _spread(rng, 64, 4000),
            "latent": _spread(rng, 8, 128), "vocab": _spread(rng, 97, 32000), "dtype": dtype,
            "max_norm": rng.choice((0.1, 1.0, 1.0, 1e9)), "spread": rng.uniform(0.0, 2.0)}


def _shapes(case):
    """The parameters' shapes of a LocalLatentLM."""
    d, ff, lat = case["d"], case["ff"], case["latent"]
    layer = [(d,), (3 * d, d), (3 * d,), (lat, d), (lat,), (2 * lat, d), (2 * lat,), (d, lat), (d,), (d, d), (d,),
             (1, d // 4), (1, d // 4), (d,), (ff, d), (ff,), (d, ff), (d,)]
    return [(case["vocab"], d), (case["d"], d)] + layer * case["layers"] + [(d,)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if case["op"] == "mlp":
        n, d, ff = case["tokens"], case["d"], case["ff"]
        # rows of a norm (unit rms) with a few large channels, projections that give pre-activations of rms 1 to 2
        x = randn(n, d) * (1.0 + 4.0 * (rand(d) < 0.01).float())
        x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-6)
        state = {"case": case, "x": x.to(dt), "w_gate": (randn(ff, d) * (1.5 / d ** 0.5)).to(dt),
                 "w_up": (randn(ff, d) * d ** -0.5).to(dt), "w_down": (randn(d, ff) * ff ** -0.5).to(dt)}
        if case["train"]:
            for k in ("x", "w_gate", "w_up", "w_down"):
                state[k].requires_grad_(True)
            # upstream gradients of a mean over the tokens
            state["dy"] = (randn(n, d) / n).to(dt)
        return state
    if case["op"] == "embed":
        b, t, d, v = case["batch"], case["length"], case["d"], case["vocab"]
        # Zipf-like words: word k about as often as 1 / (k + 1); sequences padded at their ends with the last word
        ids = (torch.exp(rand(b, t) * math.log(v)) - 1.0).long().clamp_(0, v - 2)
        if case["padded"]:
            keep = ((1.0 - 2.0 * case["padded"] * rand(b, 1)) * t).long().clamp_(min=1)
            ids = torch.where(torch.arange(t, device="cuda") < keep, ids, torch.full_like(ids, v - 1))
        state = {"case": case, "ids": ids, "weight": (randn(v, d) * 0.02).to(dt),
                 "positions": (randn(t, d) * 0.02).to(dt) if case["positions"] else None,
                 "padding": v - 1 if case["padded"] else None}
        if case["train"]:
            state["weight"].requires_grad_(True)
            if case["positions"]:
                state["positions"].requires_grad_(True)
            state["dout"] = (randn(b, t, d) / (b * t) ** 0.5).to(dt)
        return state
    # the gradients are views of one bucket, one after the other, as a data-parallel wrapper keeps them
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    bucket = torch.empty(sum(sizes), dtype=dt, device="cuda")
    params, at = [], 0
    for i, (s, n) in enumerate(zip(shapes, sizes)):
        g = bucket[at:at + n]
        g.normal_(generator=gen).mul_(10.0 ** (-3.0 + case["spread"] * math.sin(1.7 * i)))
        p = torch.nn.Parameter(torch.empty(s, dtype=dt, device="cuda"))
        p.grad = g.view(s)
        params.append(p)
        at += n
    return {"case": case, "params": params, "bucket": bucket}


def _activation(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1.0 + g * (1.0 - s))
    phi = 0.5 * (1.0 + torch.erf(g * 0.5 ** 0.5))
    return g * phi, phi + g * torch.exp(-0.5 * g * g) * (2.0 * math.pi) ** -0.5


def _plain_mlp(state, act, train):
    x, wg, wu, wd = (state[k].detach() for k in ("x", "w_gate", "w_up", "w_down"))
    dt = x.dtype
    xf, gf, uf, df = x.float(), wg.float(), wu.float(), wd.float()
    g, u = xf @ gf.t(), xf @ uf.t()
    a, slope = _activation(g, act)
    h = a * u
    y = (h @ df.t()).to(dt)
    if not train:
        return {"y": y}
    dyf = state["dy"].float()
    dh = dyf @ df
    dwd = (dyf.t() @ h).to(dt)
    dg, du = dh * u * slope, dh * a
    dx = (dg @ gf + du @ uf).to(dt)
    return {"y": y, "dx": dx, "dw_gate": (dg.t() @ xf).to(dt), "dw_up": (du.t() @ xf).to(dt), "dw_down": dwd}


def _plain_embed(state, case):
    ids, w, pos = state["ids"], state["weight"].detach(), state["positions"]
    dt = w.dtype
    out = w.float()[ids] * case["scale"]
    if pos is not None:
        out = out + pos.detach().float()
    got = {"out": out.to(dt)}
    if not case["train"]:
        return got
    d = state["dout"].float()
    rows, flat = d.reshape(-1, d.shape[-1]), ids.reshape(-1)
    if state["padding"] is not None:
        rows = rows * (flat != state["padding"])[:, None]
    # a word's rows in 64 bits: a frequent word has thousands of them
    dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device).index_add_(0, flat, rows.double())
    got["dweight"] = (dw * case["scale"]).to(dt)
    if pos is not None:
        got["dpositions"] = d.sum(0).to(dt)
    return got


def run(state):
    case = state["case"]
    if case["op"] == "mlp":
        if not own:
            return _plain_mlp(state, case["act"], case["train"])
        from llattn_b200 import gated_mlp

        ins = state["x"], state["w_gate"], state["w_up"], state["w_down"]
        y = gated_mlp(*ins, activation=case["act"])
        if not case["train"]:
            return {"y": y}
        dx, dg, du, dd = torch.autograd.grad(y, ins, state["dy"])
        return {"y": y.detach(), "dx": dx, "dw_gate": dg, "dw_up": du, "dw_down": dd}
    if case["op"] == "embed":
        if not own:
            return _plain_embed(state, case)
        from llattn_b200 import token_embedding

        out = token_embedding(state["ids"], state["weight"], positions=state["positions"], scale=case["scale"],
                              padding_idx=state["padding"])
        if not case["train"]:
            return {"out": out}
        leaves = (state["weight"],) if state["positions"] is None else (state["weight"], state["positions"])
        grads = torch.autograd.grad(out, leaves, state["dout"])
        return dict(zip(("out", "dweight", "dpositions"), (out.detach(), *grads)))
    # In place, as a training loop clips. Another pass on the same state finds a norm just above the limit less the
    # formula's 1e-6 and scales again, by almost 1: the same work.
    if own:
        from llattn_b200 import clip_grad_norm_

        return {"norm": clip_grad_norm_(state["params"], case["max_norm"]), "grads": state["bucket"]}
    bucket = state["bucket"]
    norm = bucket.float().square().sum(dtype=torch.float64).sqrt()
    factor = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    bucket.copy_(bucket.float() * factor)
    return {"norm": norm.float(), "grads": bucket}


def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "mlp":
        n, d, ff = case["tokens"], case["d"], case["ff"]
        rows, weights = size * n * d, size * d * ff
        if not case["train"]:
            return {"bytes": 2 * rows + 3 * weights, "flops": 6.0 * n * d * ff}
        return {"bytes": 4 * rows + 6 * weights, "flops": 18.0 * n * d * ff}
    if case["op"] == "embed":
        t, d, v = case["length"], case["d"], case["vocab"]
        n = case["batch"] * t
        table = size * t * d if case["positions"] else 0
        once = 8 * n + size * min(n, v) * d + table + size * n * d
        if not case["train"]:
            return {"bytes": once, "flops": 2.0 * n * d}
        return {"bytes": once + size * n * d + size * v * d + table, "flops": 4.0 * n * d}
    total = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": 2 * size * total + 4, "flops": 3.0 * total}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "mlp":
        x, wg, wu, wd = (state[k].detach().double() for k in ("x", "w_gate", "w_up", "w_down"))
        g, u = torch.mm(x, wg.mT), torch.mm(x, wu.mT)
        if case["act"] == "silu":
            gate = torch.special.expit(g)
            slope = gate + g * gate * torch.special.expit(-g)
        else:
            gate = torch.special.ndtr(g)
            slope = gate + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
        got = {"y": torch.mm(g * gate * u, wd.mT)}
        if not case["train"]:
            return got
        dy = state["dy"].double()
        got["dw_down"] = torch.mm(dy.mT, g * gate * u)
        dh = torch.mm(dy, wd)
        du = dh * g * gate
        dg = dh.mul_(u).mul_(slope)
        got["dx"] = torch.mm(dg, wg).addmm_(du, wu)
        got["dw_gate"], got["dw_up"] = torch.mm(dg.mT, x), torch.mm(du.mT, x)
        return got
    if case["op"] == "embed":
        ids, d = state["ids"], case["d"]
        out = torch.nn.functional.embedding(ids, state["weight"].detach().double()) * case["scale"]
        if state["positions"] is not None:
            out = out + state["positions"].detach().double()
        got = {"out": out}
        if not case["train"]:
            return got
        dout = state["dout"].double()
        if state["positions"] is not None:
            got["dpositions"] = torch.einsum("btd->td", dout)
        flat = ids.flatten()
        if state["padding"] is not None:
            at = torch.nonzero(flat != state["padding"])[:, 0]
        else:
            at = torch.arange(flat.numel(), device=ids.device)
        words, where = torch.unique(flat[at], return_inverse=True)
        sums = torch.zeros(words.numel(), d, dtype=torch.float64, device=ids.device)
        sums.index_put_((where,), dout.view(-1, d)[at], accumulate=True)
        dweight = torch.zeros(case["vocab"], d, dtype=torch.float64, device=ids.device)
        dweight[words] = sums * case["scale"]
        got["dweight"] = dweight
        return got
    bucket = state["bucket"].double()
    norm = torch.linalg.vector_norm(bucket)
    limit = float(case["max_norm"])
    return {"norm": norm, "grads": bucket * min(1.0, limit / (float(norm) + 1e-6))}
