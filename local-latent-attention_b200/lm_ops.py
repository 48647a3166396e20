"""Operators of the language model around the attention block, over
libllattn.so: the gated feed-forward block (``gated_mlp``), the token embedding
with its positions (``token_embedding``) and the clipping of gradients to a
global norm (``clip_grad_norm_``, ``total_norm``).

As in ``training_ops.py``: CUDA only, torch's current stream, torch-allocated
outputs and workspaces, ``RuntimeError`` on bad arguments, no CPU implementation;
custom ops with fake implementations for tracers, dispatch modes and tensor
subclasses, which plain eager calls leave out.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor

from . import _lib
from .ops import _dtype_code, _require
from .training_ops import _direct, _on, _rows, _stream

_PLAIN = torch.contiguous_format


def _common_dtype(*tensors: Tensor) -> list[Tensor]:
    """Under autocast all in its dtype, as a linear layer's inputs are (float32 where that is float16)."""
    if not torch.is_autocast_enabled("cuda"):
        return list(tensors)
    dt = torch.get_autocast_dtype("cuda")
    dt = torch.float32 if dt == torch.float16 else dt  # (no fp16 kernels)
    return [t.to(dt) if t.is_cuda else t for t in tensors]


# --------------------------------------------------------------------------
# gated feed-forward block

_ACTIVATIONS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}
_TYPES = (torch.bfloat16, torch.float32)


def _check_gated(x: Tensor, wg: Tensor, wu: Tensor, wd: Tensor) -> None:
    if (x.is_cuda and x.dim() == 2 and wg.dim() == 2 and wd.dim() == 2 and wg.shape == wu.shape
            and x.shape[1] == wg.shape[1] and wd.shape[1] == wg.shape[0] and x.dtype in _TYPES and x.dtype == wg.dtype
            and x.dtype == wu.dtype and x.dtype == wd.dtype and x.device == wg.device and x.device == wu.device
            and x.device == wd.device and wg.numel() and wd.numel()):
        return
    _require(x.is_cuda, "gated_mlp needs CUDA tensors")
    _require(x.dim() == 2 and wg.dim() == 2 and wg.shape == wu.shape and x.shape[1] == wg.shape[1],
             f"x {tuple(x.shape)}, w_gate {tuple(wg.shape)} and w_up {tuple(wu.shape)} must be [tokens, d], [ff, d] and [ff, d]")
    _require(wd.dim() == 2 and wd.shape[1] == wg.shape[0],
             f"w_down {tuple(wd.shape)} must be [d_out, ff] with w_gate's ff = {wg.shape[0]}")
    _require(x.dtype == wg.dtype == wu.dtype == wd.dtype,
             f"x is {x.dtype}, the weights {wg.dtype}, {wu.dtype} and {wd.dtype}: one dtype (or autocast) is needed")
    _require(x.device == wg.device == wu.device == wd.device, "x and the weights must be on one device")
    _dtype_code(x)
    _require(False, "the weights must have rows and columns")


def _gated_args(x: Tensor, wg: Tensor, wu: Tensor, wd: Tensor, act: int):
    """The library's arguments, and the tensors that they point to."""
    x, wg, wu, wd = _rows(x), _rows(wg), _rows(wu), _rows(wd)
    (n, d), (d_out, ff) = x.shape, wd.shape
    args = _lib.GatedArgs(n, d, ff, d_out, _dtype_code(x), act, x.data_ptr(), max(x.stride(0), d), wg.data_ptr(),
                          max(wg.stride(0), d), wu.data_ptr(), max(wu.stride(0), d), wd.data_ptr(), max(wd.stride(0), ff))
    return args, (x, wg, wu, wd)


def _gated_fwd(x: Tensor, wg: Tensor, wu: Tensor, wd: Tensor, act: int, keep: bool) -> tuple[Tensor, Tensor]:
    """y, and what the backward needs (empty without `keep`)."""
    _check_gated(x, wg, wu, wd)
    dev = x.device
    y = torch.empty(x.shape[0], wd.shape[0], dtype=x.dtype, device=dev)
    if not x.shape[0]:
        return y, torch.empty(0, dtype=torch.uint8, device=dev)
    args, held = _gated_args(x, wg, wu, wd, act)
    L, ref = _lib.lib(), ctypes.byref(args)
    with _on(dev):
        kept = torch.empty(L.llattn_gated_kept_bytes(ref) if keep else 0, dtype=torch.uint8, device=dev)
        args.y, args.kept = y.data_ptr(), kept.data_ptr() if keep else None
        size = L.llattn_gated_workspace_bytes(ref, 0)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        args.workspace, args.workspace_bytes = ws.data_ptr(), size
        _lib.check(L.llattn_gated_fwd(ref, _stream(x)), "llattn_gated_fwd")
    return y, kept


def _gated_bwd(x: Tensor, wg: Tensor, wu: Tensor, wd: Tensor, act: int, kept: Tensor, dy: Tensor, need_x: bool, need_g: bool,
               need_u: bool, need_d: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """The gradients that are needed (others empty)."""
    make = torch.empty if x.shape[0] else torch.zeros
    outs = [make(t.shape if need else (0,), dtype=x.dtype, device=x.device)
            for t, need in ((x, need_x), (wg, need_g), (wu, need_u), (wd, need_d))]
    if not x.shape[0]:
        return tuple(outs)
    args, held = _gated_args(x, wg, wu, wd, act)
    dy = _rows(dy)
    L, ref = _lib.lib(), ctypes.byref(args)
    with _on(x.device):
        args.kept, args.dy, args.lddy = kept.data_ptr(), dy.data_ptr(), max(dy.stride(0), dy.shape[1])
        args.dx, args.dw_gate, args.dw_up, args.dw_down = (o.data_ptr() if o.numel() else None for o in outs)
        size = L.llattn_gated_workspace_bytes(ref, 1)
        ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), size
        _lib.check(L.llattn_gated_bwd(ref, _stream(x)), "llattn_gated_bwd")
    return tuple(outs)


gated_mlp_op = torch.library.custom_op("llattn_b200::gated_mlp", _gated_fwd, mutates_args=(), device_types="cuda")
gated_mlp_grads_op = torch.library.custom_op("llattn_b200::gated_mlp_grads", _gated_bwd, mutates_args=(),
                                             device_types="cuda")


def _up256(v):
    return (v + 255) // 256 * 256


def _kept_bytes(n, ff, dtype):
    blocks = n * ((ff + 31) // 32)
    return _up256(blocks * 256) if dtype == torch.float32 else _up256(blocks * 128) + _up256(blocks * 2)


@gated_mlp_op.register_fake
def _gated_fake(x, wg, wu, wd, act, keep):
    return (x.new_empty(x.shape[0], wd.shape[0]),
            x.new_empty(_kept_bytes(x.shape[0], wg.shape[0], x.dtype) if keep else 0, dtype=torch.uint8))


@gated_mlp_grads_op.register_fake
def _gated_grads_fake(x, wg, wu, wd, act, kept, dy, need_x, need_g, need_u, need_d):
    return tuple(x.new_empty(t.shape if need else (0,))
                 for t, need in ((x, need_x), (wg, need_g), (wu, need_u), (wd, need_d)))


class _GatedMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, wd, act):
        f = _gated_fwd if _direct(x, wg, wu, wd) else gated_mlp_op
        y, kept = f(x, wg, wu, wd, act, True)
        ctx.save_for_backward(x, wg, wu, wd, kept)
        ctx.act = act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, wg, wu, wd, kept = ctx.saved_tensors
        need = ctx.needs_input_grad[:4]
        f = _gated_bwd if _direct(x, wg, wu, wd, dy) else gated_mlp_grads_op
        outs = f(x, wg, wu, wd, ctx.act, kept, dy, *need)
        return (*(o if n else None for o, n in zip(outs, need)), None)


def gated_mlp(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, *, activation: str = "silu") -> Tensor:
    """Gated feed-forward block: ``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T``,
    differentiable in all four (gradients of gradients are not supported).

    x [..., d], w_gate and w_up [ff, d], w_down [d_out, ff], all bfloat16 or all
    float32 (under autocast all are cast to its dtype, as a linear layer's inputs
    are, or to float32 where that is float16), with any row strides; sizes up to
    2^20, 2^26 tokens. activation: "silu", or "gelu" (by erf). Returns
    [..., d_out] in x's dtype.

    Neither x @ w_gate.T nor x @ w_up.T nor their gradients before the activation are
    returned to memory in full: with gradients the call keeps 4 bytes (bfloat16; 8
    for float32) a token and inner column for its backward.

    Precision: sums are fp32. float32 inputs keep 24 bits in every product.
    bfloat16: the products' operands act(g) u and its gradients are rounded to
    bfloat16 once (for up to 64 tokens to 16 bits, for up to 32 without gradients
    not below 16 bits), what is kept to 11 bits relative to the largest of 32 neighbours, and
    the results once."""
    act = _ACTIVATIONS.get(activation)
    if act is None:
        _require(False, f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 1 or w_gate.dim() != 2 or x.shape[-1] != w_gate.shape[1]:
        _require(False, f"x {tuple(x.shape)} must end in w_gate's columns {tuple(w_gate.shape)}")
    x, w_gate, w_up, w_down = _common_dtype(x, w_gate, w_up, w_down)
    flat = x.dim() == 2
    x2 = x if flat else x.reshape(-1, x.shape[-1])
    if torch.is_grad_enabled() and (x2.requires_grad or w_gate.requires_grad or w_up.requires_grad or w_down.requires_grad):
        y = _GatedMlp.apply(x2, w_gate, w_up, w_down, act)
    else:
        y = (_gated_fwd if _direct(x2, w_gate, w_up, w_down) else gated_mlp_op)(x2, w_gate, w_up, w_down, act, False)[0]
    return y if flat else y.view(*x.shape[:-1], w_down.shape[0])
