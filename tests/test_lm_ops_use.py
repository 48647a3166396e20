"""The language model with its own operators (gated feed-forward blocks, token embedding, clipping) beside the loss and the
attention block: switches, agreement with torch's operators, generation, checkpoints, the example."""

import importlib.util
import os
from dataclasses import fields
from types import SimpleNamespace

import pytest
import torch
import torch.nn.functional as F

from llattn_b200 import clip_grad_norm_
from llattn_b200.lm import DecoderLayer, LocalLatentLM, ModelConfig, build_optimizer, train_step

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def small_cfg(**kw):
    base = dict(vocab_size=300, max_seq_len=160, d_model=128, n_heads=2, n_layers=2, d_ff=344, local_window=32,
                latent_tokens=8, latent_d_model=32, latent_heads=2)
    return ModelConfig(**{**base, **kw})


def torch_mlp(layer, h):
    act = F.silu if layer.gate == "silu" else F.gelu
    return layer.ff["w2"](act(layer.ff["w1"](h)) * layer.ff["w3"](h))


# --- host side ---------------------------------------------------------------------

def test_parameters_of_the_gated_block():
    plain, gated = LocalLatentLM(small_cfg()), LocalLatentLM(small_cfg(ff_gate="silu"))
    names = lambda m: [n for n, _ in m.named_parameters() if "blocks.0.ff" in n]
    assert names(plain) == [f"blocks.0.ff.{w}.{k}" for w in ("w1", "w2") for k in ("weight", "bias")]
    assert names(gated) == [f"blocks.0.ff.{w}.weight" for w in ("w1", "w3", "w2")]
    # w2 writes to the residual stream: its initial values are scaled down with the depth
    w1, w2 = (gated.blocks[1].ff[k].weight.std().item() for k in ("w1", "w2"))
    assert abs(w1 / 0.02 - 1) < 0.02 and abs(w2 / 0.01 - 1) < 0.02  # (128 x 344 values: within 0.5 % each)
    opt = build_optimizer(gated, hidden="muon")
    inside = {id(p) for g in opt.optimizers[0].param_groups for p in g["params"]}
    assert all(id(layer.ff[k].weight) in inside for layer in gated.blocks for k in ("w1", "w2", "w3"))


def test_the_reference_config_has_no_gate():
    """A config without the field (the reference's) builds the reference's MLP."""
    cfg = small_cfg()
    bare = SimpleNamespace(**{f.name: getattr(cfg, f.name) for f in fields(cfg) if f.name != "ff_gate"})
    torch.manual_seed(3)
    a = DecoderLayer(bare)
    torch.manual_seed(3)
    b = DecoderLayer(cfg)
    assert all(torch.equal(x, y) for x, y in zip(a.state_dict().values(), b.state_dict().values()))
    assert list(a.state_dict()) == list(b.state_dict())


def test_positions_past_the_table_are_refused():
    m, ids = LocalLatentLM(small_cfg()), torch.zeros(2, 3, dtype=torch.long)
    assert m._embed(ids, 157).shape == (2, 3, 128)
    for tok, first in ((ids[:, :1], 160), (ids, 158), (ids[:, :1], 1000)):
        with pytest.raises(IndexError):
            m._embed(tok, first)


# --- on the GPU ----------------------------------------------------------------------

def model(**kw):
    torch.manual_seed(0)
    return LocalLatentLM(small_cfg(**kw)).cuda()


def tokens(n=129, batch=3, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, 300, (batch, n), generator=gen).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["silu", "gelu"])
@pytest.mark.parametrize("autocast", [True, False])
def test_loss_and_gradients_match_torchs_operators(gate, autocast, monkeypatch):
    """The same model and tokens through this package's operators and through torch's. fp32: 1e-4 of every gradient's norm (the
    attention block's own tolerance); bf16 autocast: 2e-2, intermediates are rounded at different places."""
    m, ids = model(ff_gate=gate), tokens()
    got = {}
    for own in (True, False):
        m.fused_embedding = m.fused_loss = own
        if not own:
            monkeypatch.setattr(DecoderLayer, "mlp", torch_mlp)
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            loss = m(ids[:, :-1], ids[:, 1:])
        loss.backward()
        got[own] = loss.item(), {n: p.grad.clone() for n, p in m.named_parameters()}
    tol = 2e-2 if autocast else 1e-4
    assert abs(got[True][0] - got[False][0]) <= tol * got[False][0]
    for n, g in got[False][1].items():
        assert (got[True][1][n] - g).norm() <= tol * g.norm() + 1e-12, n


@pytest.mark.gpu
def test_embedding_is_torchs_in_fp32():
    m, ids = model(), tokens()
    want = m._embed(ids)
    m.fused_embedding = True
    assert torch.equal(m._embed(ids), want)
    assert torch.equal(m._embed(ids[:, 7:9], 7), want[:, 7:9])
    logits = m(ids)
    m.fused_embedding = False
    assert torch.equal(m(ids), logits)
    # the tied head's gradient and the embedding's meet in one tensor
    for own in (True, False):
        m.fused_embedding = own
        m.zero_grad(set_to_none=True)
        m(ids[:, :-1], ids[:, 1:]).backward()
        if own:
            first = m.embedding.weight.grad.clone(), m.position.weight.grad.clone()
    for a, b in zip(first, (m.embedding.weight.grad, m.position.weight.grad)):
        assert (a - b).norm() <= 1e-6 * b.norm() and torch.equal(a == 0, b == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("remat", [False, True])
def test_training_step(remat):
    """One step of everything together against torch's clipping: the same updated parameters to fp32's last bits (the norm
    differs by 1e-7, AdamW's first step is lr * sign(g) but for gradients near its eps of 1e-8)."""
    ids = tokens()
    got = []
    for fused in (True, False):
        m = model(ff_gate="silu", checkpoint_blocks=remat)
        m.train()
        m.fused_loss = m.fused_embedding = True
        opt = build_optimizer(m, lr=1e-3)
        loss = train_step(m, opt, ids[:, :-1], ids[:, 1:], grad_clip=0.05, fused_clip=fused)
        got.append((loss, [p.detach().clone() for p in m.parameters()]))
    assert torch.equal(got[0][0], got[1][0])
    for a, b in zip(got[0][1], got[1][1]):
        assert (a - b).abs().max() <= 1e-3 * 1e-4


@pytest.mark.gpu
def test_clipping_of_a_models_gradients():
    m, ids = model(ff_gate="gelu"), tokens()
    m(ids[:, :-1], ids[:, 1:]).backward()
    norm = torch.linalg.vector_norm(torch.cat([p.grad.double().reshape(-1) for p in m.parameters()]))
    got = clip_grad_norm_(m.parameters(), 0.5 * norm.item())
    assert abs(got.item() / norm.item() - 1) < 1e-6
    after = torch.linalg.vector_norm(torch.cat([p.grad.double().reshape(-1) for p in m.parameters()]))
    assert abs(after.item() / (0.5 * norm.item()) - 1) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_generation(dtype):
    """Greedy tokens through decode caches (single tokens: the few-token kernel) and by whole forwards."""
    m = model(ff_gate="silu").to(dtype).eval()
    m.fused_embedding = True
    ids = tokens(20, 2)
    a = m.generate(ids, 12, incremental=True)
    b = m.generate(ids, 12, incremental=False)
    assert a.shape == (2, 32)
    if dtype == torch.float32:
        assert torch.equal(a, b)
    m.fused_embedding = False
    assert torch.equal(m.generate(ids, 12, incremental=True), a)


@pytest.mark.gpu
def test_compiled_layer():
    """The gated block and the embedding inside compiled functions: the same bits."""
    m, ids = model(ff_gate="silu"), tokens()
    m.fused_embedding = True
    x = m._embed(ids).detach()
    f = torch.compile(m.blocks[0].mlp, backend="aot_eager", fullgraph=True)
    assert torch.equal(f(x), m.blocks[0].mlp(x))
    e = torch.compile(m._embed, backend="aot_eager", fullgraph=True)
    assert torch.equal(e(ids), m._embed(ids))


@pytest.mark.gpu
@pytest.mark.parametrize("flags", [["--ff-gate", "silu"], ["--embedding", "plain", "--clip", "plain", "--hidden", "adamw"]])
def test_example_runs(flags):
    spec = importlib.util.spec_from_file_location("train_lm_example", os.path.join(ROOT, "examples", "train_lm.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses = mod.main(["--steps", "3", "--layers", "1", *flags])
    assert len(losses) == 3 and all(v == v for v in losses)


@pytest.mark.gpu
def test_decoding_past_the_last_position_is_refused():
    m = model().eval()
    ids = tokens(159, 2)
    caches = [blk.attn.new_decode_cache(160) for blk in m.blocks]
    with torch.no_grad():
        m._prefill(ids, caches)
        m._decode_one(ids[:, :1], 159, caches)
        with pytest.raises(IndexError):
            m._decode_one(ids[:, :1], 160, caches)
        m.fused_embedding = True
        with pytest.raises(RuntimeError, match="positions"):
            m._decode_one(ids[:, :1], 160, caches)


@pytest.mark.gpu
def test_generation_calls_the_position_module():
    """A forward hook on model.position sees the prompt's rows, as it does in torch's own call."""
    m, seen = model().eval(), []
    m.position.register_forward_hook(lambda mod, args, out: seen.append(out.shape))
    m.generate(tokens(20, 2), 3)
    assert seen == [(20, 128)]
