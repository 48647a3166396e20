"""Trains a small LocalLatentLM on synthetic tokens with the training step's own
operators: the head's loss without logits (linear_cross_entropy) and
orthogonalised updates of the layers' matrices (newton_schulz, through Muon).

    python examples/train_lm.py                       # fused loss, Muon
    python examples/train_lm.py --loss plain --hidden adamw
"""

from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from llattn_b200.lm import LocalLatentLM, ModelConfig, build_optimizer, train_step


def run(args) -> list[float]:
    torch.manual_seed(0)
    cfg = ModelConfig(vocab_size=args.vocab, max_seq_len=args.seq_len, d_model=args.d_model, n_heads=args.d_model // 64,
                      n_layers=args.layers, d_ff=4 * args.d_model, local_window=64, latent_tokens=16, latent_d_model=64,
                      latent_heads=2)
    model = LocalLatentLM(cfg).cuda()
    model.fused_loss = args.loss == "fused"
    optimizer = build_optimizer(model, lr=args.lr, hidden=args.hidden)
    gen = torch.Generator().manual_seed(1)
    losses = []
    for step in range(args.steps):
        # token t + 1 follows token t, from a random start: learnable, and new every step
        start = torch.randint(0, cfg.vocab_size, (args.batch, 1), generator=gen)
        seq = ((start + torch.arange(args.seq_len + 1)) % cfg.vocab_size).cuda()
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        losses.append(train_step(model, optimizer, seq[:, :-1], seq[:, 1:]).item())
        print(f"step {step:3d}  loss {losses[-1]:.4f}  {1e3 * (time.perf_counter() - t0):.2f} ms", flush=True)
    return losses


def main(argv=None) -> list[float]:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--loss", choices=("fused", "plain"), default="fused")
    ap.add_argument("--hidden", choices=("muon", "adamw"), default="muon")
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--seq-len", type=int, default=128)
    ap.add_argument("--d-model", type=int, default=256)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--vocab", type=int, default=512)
    ap.add_argument("--lr", type=float, default=1e-3)
    return run(ap.parse_args(argv))


if __name__ == "__main__":
    main()
