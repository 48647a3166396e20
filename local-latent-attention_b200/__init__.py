"""llattn_b200 — B200 (sm_100a) kernels of the fused local + latent attention
block of Fenix46/local-latent-attention, behind the reference's module API.

    from llattn_b200 import LocalLatentAttentionB200, build_attention
    from llattn_b200.ops import llattn_attention, pool_chunks, pool_query_blocks
    from llattn_b200 import linear_cross_entropy, newton_schulz, Muon   # the training step's loss and update
    from llattn_b200 import gated_mlp, token_embedding, clip_grad_norm_   # the rest of a language model's step

The CUDA work happens in libllattn.so (C ABI: include/llattn.h), loaded on
first use; it is built by ``csrc/build.py``, and with it _torch_ops.so, the eager path
of the last three.
"""

from . import ops
from .lm_ops import clip_grad_norm_, gated_mlp, token_embedding, total_norm
from .module import DecodeCache, LocalLatentAttentionB200, build_attention
from .ops import LLAttnFunction, llattn_attention
from .optim import Muon
from .training_ops import linear_cross_entropy, newton_schulz

__all__ = ["LocalLatentAttentionB200", "DecodeCache", "build_attention", "llattn_attention", "LLAttnFunction", "ops",
           "linear_cross_entropy", "newton_schulz", "Muon", "gated_mlp", "token_embedding",
           "clip_grad_norm_", "total_norm"]
