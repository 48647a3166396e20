"""Operators of the language model around the attention block, over
libllattn.so: the gated feed-forward block (``gated_mlp``), the token embedding
with its positions (``token_embedding``) and the clipping of gradients to a
global norm (``clip_grad_norm_``, ``total_norm``).

As in ``training_ops.py``: CUDA only, torch's current stream, torch-allocated
outputs and workspaces, ``RuntimeError`` on bad arguments, no CPU implementation;
custom ops with fake implementations for tracers, dispatch modes and tensor
subclasses. Plain eager calls leave them out: they go through ``_torch_ops.so``
(csrc/torch_ops.cpp, built with the library), whose autograd nodes are C++, and what that does
not handle (empty inputs, bad arguments) comes back to the functions here.
"""

from __future__ import annotations

import ctypes
from array import array
from typing import Iterable, Optional, Sequence, Union

import torch
from torch import Tensor

from . import _lib
from .ops import _DT, _dtype_code, _require
from .training_ops import _direct, _no_tangents, _on, _rows, _stream

try:
    from . import _torch_ops as _native
except ImportError as missing:  # calls say so: there is no other eager path to fall back to
    _native, _why = None, missing


def _eager():
    """The native calls, or None where somebody traces or intercepts."""
    if torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack():
        return None
    if _native is None:
        raise RuntimeError("llattn: _torch_ops.so is missing or does not load: build it with "
                           f"`python local-latent-attention_b200/csrc/build.py` ({_why})")
    return _native


def _common_dtype(*tensors: Tensor) -> list[Tensor]:
    """All in autocast's dtype, as a linear layer's inputs are (float32 where that is float16): float64 and
    integers are not, and are refused then."""
    dt = torch.get_autocast_dtype("cuda")
    dt = torch.float32 if dt == torch.float16 else dt  # (no fp16 kernels)
    return [t.to(dt) if t.is_cuda and t.is_floating_point() and t.dtype != torch.float64 else t for t in tensors]


# --------------------------------------------------------------------------
# gated feed-forward block

_ACTIVATIONS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}
_TYPES = (torch.bfloat16, torch.float32)


def _check_gated(x: Tensor, wg: Tensor, wu: Tensor, wd: Tensor) -> None:
    if (x.is_cuda and x.dim() == 2 and wg.dim() == 2 and wd.dim() == 2 and wg.shape == wu.shape
            and x.shape[1] == wg.shape[1] and wd.shape[1] == wg.shape[0] and x.dtype in _TYPES and x.dtype == wg.dtype
            and x.dtype == wu.dtype and x.dtype == wd.dtype and x.device == wg.device and x.device == wu.device
            and x.device == wd.device and wg.numel() and wd.numel() and x.shape[0] <= 1 << 26
            and max(*wg.shape, wd.shape[0]) <= 1 << 20):
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
    _require(wg.numel() > 0 and wd.numel() > 0, "the weights must have rows and columns")
    _require(False, f"{x.shape[0]} tokens or weights {tuple(wg.shape)} and {tuple(wd.shape)} too large (2^26 tokens, sizes of 2^20)")


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


def _kept_bytes(n, ff, dtype):
    return (n + 31) // 32 * ((ff + 15) // 16) * (4096 if dtype == torch.float32 else 2048 + 64)


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
        _no_tangents("gated_mlp's backward", dy)
        x, wg, wu, wd, kept = ctx.saved_tensors
        need = ctx.needs_input_grad[:4]
        f = _gated_bwd if _direct(x, wg, wu, wd, dy) else gated_mlp_grads_op
        outs = f(x, wg, wu, wd, ctx.act, kept, dy, *need)
        return (*(o if n else None for o, n in zip(outs, need)), None)


def gated_mlp(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, *, activation: str = "silu") -> Tensor:
    """Gated feed-forward block: ``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T``,
    differentiable in all four (gradients of gradients and forward-mode derivatives
    are not supported).

    x [..., d], w_gate and w_up [ff, d], w_down [d_out, ff], all bfloat16 or all
    float32 (under autocast all are cast to its dtype, as a linear layer's inputs
    are, or to float32 where that is float16), with any row strides; sizes up to
    2^20, 2^26 tokens. activation: "silu", or "gelu" (by erf). Returns
    [..., d_out] in x's dtype.

    Memory, bytes a token and inner column: with gradients the call keeps x @ w_gate.T and x @ w_up.T
    for its backward, 4 and 1 / 8 in bfloat16, 8 in float32; its workspace holds act(g) u, 2 in bfloat16 (4 up to
    64 tokens), 6 in float32; the backward's holds that again, where w_down's gradient is wanted, and both gradients
    before the activation, 4 (8; 12). Without gradients nothing but act(g) u is in memory; its gradient never is.
    Rows off a 16-byte boundary, and all float32 operands, are copied besides (2 and 6 bytes an element).

    Precision: sums are fp32, by the tensor cores, whose additions drop what lies below a sum's last
    bits: bfloat16 products of one sign come out up to 2^-27 each short, in sums of at most 2^17
    that are added up in fp32 (float32: of 256). float32 inputs keep 24 bits in every product, and the
    activation is to 2^-19 of its value.
    bfloat16: the products' operands act(g) u and its gradients are rounded to bfloat16 once (for up to 64 tokens to
    16 bits, of an activation to 2^-19 of its value), what is kept to 11 bits relative to the largest of 16 neighbours,
    and the results once. Infinities in a token's inputs make its results infinite or NaN."""
    act = _ACTIVATIONS.get(activation)
    if act is None:
        _require(False, f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if torch.is_autocast_enabled("cuda"):
        x, w_gate, w_up, w_down = _common_dtype(x, w_gate, w_up, w_down)
    native = _eager()
    y = native.gated(x, w_gate, w_up, w_down, act) if native else None
    if y is not None:
        return y
    _no_tangents("gated_mlp", x, w_gate, w_up, w_down)
    if x.dim() < 1 or w_gate.dim() != 2 or x.shape[-1] != w_gate.shape[1]:
        _require(False, f"x {tuple(x.shape)} must end in w_gate's columns {tuple(w_gate.shape)}")
    flat = x.dim() == 2
    x2 = x if flat else x.reshape(-1, x.shape[-1])
    if torch.is_grad_enabled() and (x2.requires_grad or w_gate.requires_grad or w_up.requires_grad or w_down.requires_grad):
        y = _GatedMlp.apply(x2, w_gate, w_up, w_down, act)
    else:
        y = (_gated_fwd if _direct(x2, w_gate, w_up, w_down) else gated_mlp_op)(x2, w_gate, w_up, w_down, act, False)[0]
    return y if flat else y.view(*x.shape[:-1], w_down.shape[0])


# --------------------------------------------------------------------------
# token embedding

_IDS = {torch.int64: 1, torch.int32: 0}


def _embed_args(ids: Tensor, w: Tensor, rows: int, scale: float, padding: int):
    length = ids.shape[1]
    return _lib.EmbedArgs(ids.shape[0], length, w.shape[1], _dtype_code(w), _IDS[ids.dtype], rows, w.shape[0], padding, scale,
                          ids.data_ptr())


def _check_embed(ids: Tensor, w: Tensor, pos: Optional[Tensor]) -> None:
    if (w.is_cuda and ids.dim() == 2 and w.dim() == 2 and ids.dtype in _IDS and w.dtype in _TYPES and ids.device == w.device
            and w.numel() and ids.numel() <= 1 << 30 and w.shape[0] <= 1 << 24 and w.shape[1] <= 1 << 20
            and (pos is None or (pos.dim() == 2 and ids.shape[1] <= pos.shape[0] < 1 << 31 and pos.shape[1] == w.shape[1]
                                 and pos.dtype == w.dtype and pos.device == w.device))):
        return
    _require(w.is_cuda, "token_embedding needs CUDA tensors")
    _require(ids.dtype in _IDS, f"ids must be int64 or int32, got {ids.dtype}")
    _require(w.dim() == 2, f"weight must be [vocab, d], got {tuple(w.shape)}")
    _dtype_code(w)
    _require(w.numel() > 0, "weight must have rows and columns")
    if pos is not None:
        _require(pos.dim() == 2 and pos.shape[0] >= ids.shape[1] and pos.shape[1] == w.shape[1],
                 f"positions {tuple(pos.shape)} must be [at least {ids.shape[1]}, {w.shape[1]}]")
        _require(pos.dtype == w.dtype, f"weight is {w.dtype} and positions {pos.dtype}: one dtype is needed")
        _require(pos.shape[0] < 1 << 31, f"{pos.shape[0]} positions: too many")
    _require(ids.numel() <= 1 << 30 and w.shape[0] <= 1 << 24 and w.shape[1] <= 1 << 20,
             f"{ids.numel()} ids or weight {tuple(w.shape)} too large (2^30 ids, 2^24 words of 2^20)")
    _require(False, "ids, weight and positions must be on one device")


def _embed_fwd(ids: Tensor, w: Tensor, pos: Optional[Tensor], scale: float) -> Tensor:
    """ids [batch, length] -> [batch, length, d]."""
    _check_embed(ids, w, pos)
    out = torch.empty(*ids.shape, w.shape[1], dtype=w.dtype, device=w.device)
    if out.numel():
        ids, w = ids.contiguous(), _rows(w)
        pos = None if pos is None else _rows(pos)
        args = _embed_args(ids, w, 0 if pos is None else pos.shape[0], scale, -1)
        args.w, args.ldw, args.out = w.data_ptr(), max(w.stride(0), w.shape[1]), out.data_ptr()
        if pos is not None:
            args.positions, args.ldp = pos.data_ptr(), max(pos.stride(0), pos.shape[1])
        with _on(w.device):
            _lib.check(_lib.lib().llattn_embed_fwd(ctypes.byref(args), _stream(w)), "llattn_embed_fwd")
    return out


def _embed_bwd(ids: Tensor, dout: Tensor, vocab: int, position_rows: int, scale: float, padding: int, need_w: bool,
               need_p: bool) -> tuple[Tensor, Tensor]:
    """dweight and dpositions where needed (else empty)."""
    d = dout.shape[2]
    make = torch.empty if dout.numel() else torch.zeros
    dw = make((vocab, d) if need_w else (0,), dtype=dout.dtype, device=dout.device)
    dp = make((position_rows, d) if need_p else (0,), dtype=dout.dtype, device=dout.device)
    if dout.numel() and (need_w or need_p):
        ids, dout = ids.contiguous(), dout.contiguous()
        args = _lib.EmbedArgs(*ids.shape, d, _dtype_code(dout), _IDS[ids.dtype], position_rows, vocab, padding, scale,
                              ids.data_ptr())
        args.dout, args.dw, args.dpositions = (dout.data_ptr(), dw.data_ptr() if need_w else None,
                                               dp.data_ptr() if need_p else None)
        L, ref = _lib.lib(), ctypes.byref(args)
        with _on(dout.device):
            size = L.llattn_embed_workspace_bytes(ref) or 256
            ws = torch.empty(size, dtype=torch.uint8, device=dout.device)
            args.workspace, args.workspace_bytes = ws.data_ptr(), size
            _lib.check(L.llattn_embed_bwd(ref, _stream(dout)), "llattn_embed_bwd")
    return dw, dp


token_embedding_op = torch.library.custom_op("llattn_b200::token_embedding", _embed_fwd, mutates_args=(), device_types="cuda")
token_embedding_grads_op = torch.library.custom_op("llattn_b200::token_embedding_grads", _embed_bwd, mutates_args=(),
                                                   device_types="cuda")


@token_embedding_op.register_fake
def _embed_fake(ids, w, pos, scale):
    return w.new_empty(*ids.shape, w.shape[1])


@token_embedding_grads_op.register_fake
def _embed_grads_fake(ids, dout, vocab, position_rows, scale, padding, need_w, need_p):
    d = dout.shape[2]
    return (dout.new_empty((vocab, d) if need_w else (0,)), dout.new_empty((position_rows, d) if need_p else (0,)))


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, w, pos, scale, padding):
        f = _embed_fwd if _direct(ids, w, *(() if pos is None else (pos,))) else token_embedding_op
        ctx.save_for_backward(ids)
        ctx.cfg = (w.shape[0], 0 if pos is None else pos.shape[0], scale, padding)
        return f(ids, w, pos, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        _no_tangents("token_embedding's backward", dout)
        (ids,) = ctx.saved_tensors
        _, need_w, need_p = ctx.needs_input_grad[:3]
        f = _embed_bwd if _direct(ids, dout) else token_embedding_grads_op
        dw, dp = f(ids, dout, *ctx.cfg, need_w, need_p)
        return None, dw if need_w else None, dp if need_p else None, None, None


def token_embedding(ids: Tensor, weight: Tensor, *, positions: Optional[Tensor] = None, scale: float = 1.0,
                    padding_idx: Optional[int] = None) -> Tensor:
    """Rows of an embedding: ``scale * weight[ids]``, plus ``positions[t]`` for the t-th
    id along ids' last dimension; differentiable in weight and positions
    (gradients of gradients and forward-mode derivatives are not supported).

    ids [...] int64 or int32, weight [vocab, d] bfloat16 or float32, positions
    [at least ids.shape[-1], d] in weight's dtype; any row strides. Returns [..., d]
    in weight's dtype (autocast does not change it, as it does not change
    torch's embedding). At most 2^30 ids, 2^24 words.

    weight's gradient sums the tokens of each word in fp32 in an order of their places: the same
    bits every run. Tokens of the word padding_idx (which may count from the end)
    do not take part in it. An id outside [0, vocab) makes its row NaN and has no
    gradient (it is an error that no launch can raise)."""
    padding = -1
    if padding_idx is not None:
        vocab = weight.shape[0] if weight.dim() else 0
        _require(-vocab <= padding_idx < vocab, f"padding_idx {padding_idx} outside the {vocab} words")
        padding = padding_idx % vocab
    scale = float(scale)
    native = _eager()
    out = native.embed(ids, weight, positions, scale, padding) if native else None
    if out is not None:
        return out
    _no_tangents("token_embedding", weight, positions)
    _require(ids.dim() >= 1 or positions is None, "positions need ids with a dimension")
    _require(weight.dim() == 2, f"weight must be [vocab, d], got {tuple(weight.shape)}")
    ids2 = ids if ids.dim() == 2 else ids.reshape(-1, ids.shape[-1] if ids.dim() and ids.shape[-1] else 1)
    if torch.is_grad_enabled() and (weight.requires_grad or (positions is not None and positions.requires_grad)):
        out = _Embed.apply(ids2, weight, positions, scale, padding)
    else:
        f = _embed_fwd if _direct(ids2, weight, *(() if positions is None else (positions,))) else token_embedding_op
        out = f(ids2, weight, positions, scale)
    return out if ids.dim() == 2 else out.view(*ids.shape, weight.shape[1])


# --------------------------------------------------------------------------
# norm over many tensors, clipping

_LISTS = (ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_int32))
_NORMS = {2.0: _lib.NORM_2, float("inf"): _lib.NORM_INF}


def _dense(t: Tensor) -> bool:
    """Whether t's elements are numel() consecutive ones, in whatever order."""
    if t.is_contiguous():
        return True
    run = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != run:
            return False
        run *= size
    return True


_KINDS = {Tensor, torch.nn.Parameter}


def _plain(tensors: Sequence[Tensor]) -> bool:
    return set(map(type, tensors)) <= _KINDS


def _dense_all(tensors: list[Tensor], what: str) -> list[Tensor]:
    """The tensors, copies in the place of those that are not dense, checked for `what`."""
    devices, dtypes, layouts = set(map(Tensor.get_device, tensors)), {t.dtype for t in tensors}, {t.layout for t in tensors}
    if len(devices) != 1 or -1 in devices or not tensors[0].is_cuda:
        _require(tensors[0].is_cuda, f"{what} needs CUDA tensors")
        _require(False, f"{what} needs tensors of one device")
    _require(layouts == {torch.strided}, f"{what} needs dense tensors, got {layouts}")
    for dt in dtypes:
        if dt not in _DT:
            _dtype_code(next(t for t in tensors if t.dtype == dt))
    if all(map(Tensor.is_contiguous, tensors)):
        return tensors
    return [t if _dense(t) else t.contiguous() for t in tensors]


def _clip(tensors: list[Tensor], norm_type: int, max_norm: float, scale: bool) -> Tensor:
    """tensors: dense, of one device and not empty as a list."""
    n, device = len(tensors), tensors[0].device
    norm = torch.empty((), dtype=torch.float32, device=device)
    pointers, sizes = array("Q", map(Tensor.data_ptr, tensors)), array("q", map(Tensor.numel, tensors))
    codes = array("i", [_DT[t.dtype] for t in tensors])
    args = _lib.ClipArgs(n, norm_type, scale, *(ctypes.cast(a.buffer_info()[0], kind) for a, kind in
                                                zip((pointers, sizes, codes), _LISTS)), max_norm, norm.data_ptr())
    L, ref = _lib.lib(), ctypes.byref(args)
    with _on(device):
        size = L.llattn_clip_workspace_bytes(ref)
        ws = torch.empty(size or 256, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), size or 256
        _lib.check(L.llattn_clip(ref, _stream(norm)), "llattn_clip")
    return norm


def _norm_of(tensors: list[Tensor], norm_type: int) -> Tensor:
    return _clip(_dense_all(tensors, "total_norm"), norm_type, 0.0, False)


def _clip_of(grads: list[Tensor], max_norm: float, norm_type: int) -> Tensor:
    dense = _dense_all(grads, "clip_grad_norm_")
    norm = _clip(dense, norm_type, max_norm, True)
    for g, c in zip(grads, dense):
        if c is not g:
            g.copy_(c)
        elif not g.is_inference():
            torch.autograd.graph.increment_version(g)  # autograd has to see that it changed
    return norm


total_norm_op = torch.library.custom_op("llattn_b200::total_norm", _norm_of, mutates_args=(), device_types="cuda",
                                        schema="(Tensor[] tensors, int norm_type) -> Tensor")
clip_grads_op = torch.library.custom_op("llattn_b200::clip_grads_", _clip_of, mutates_args=("grads",), device_types="cuda",
                                        schema="(Tensor(a!)[] grads, float max_norm, int norm_type) -> Tensor")


@total_norm_op.register_fake
def _norm_fake(tensors, norm_type):
    return tensors[0].new_empty((), dtype=torch.float32)


@clip_grads_op.register_fake
def _clip_fake(grads, max_norm, norm_type):
    return grads[0].new_empty((), dtype=torch.float32)


def _norm_code(norm_type) -> int:
    code = _NORMS.get(float(norm_type))
    _require(code is not None, f"norm_type must be 2 or inf, got {norm_type!r}")
    return code


def total_norm(tensors: Union[Tensor, Iterable[Tensor]], norm_type: float = 2.0) -> Tensor:
    """The norm of all tensors' elements together, as a float32 scalar on their
    device: the 2-norm (squares summed in fp32 within 16 bytes and in fp64 from there on, in a fixed
    order; finite for any finite float32 result) or, for norm_type=inf, the largest magnitude. NaN where one of them is. Not
    differentiable.
    Tensors are bfloat16 or float32, of any shapes and mix, on one CUDA device; 0
    on the CPU for an empty list."""
    code = _norm_code(norm_type)
    tensors = [tensors] if isinstance(tensors, Tensor) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    native = _eager()
    norm = native.clip(tensors, False, code, 0.0, False) if native else None
    if norm is not None:
        return norm
    with torch.no_grad():
        return (_norm_of if native and _plain(tensors) else total_norm_op)(tensors, code)


def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> Tensor:
    """torch.nn.utils.clip_grad_norm_ in two launches: the norm of all gradients
    together (``total_norm``), and every gradient times min(1, max_norm / (norm + 1e-6))
    in place, untouched where that is 1. Returns the norm, a float32 scalar on the
    gradients' device.

    Gradients are bfloat16 or float32, of any mix and layout, on one CUDA device; no two may
    share memory. Parameters without a gradient are skipped, one given twice counts
    once. norm_type: 2 or inf. A norm that is not finite makes the gradients NaN or 0, as
    torch's does; error_if_nonfinite raises instead, before they change (it waits for the
    device)."""
    code = _norm_code(norm_type)
    max_norm = float(max_norm)
    _require(max_norm >= 0, f"max_norm must be >= 0, got {max_norm}")
    parameters = [parameters] if isinstance(parameters, Tensor) else list(parameters)
    native = _eager()
    if error_if_nonfinite:
        norm = total_norm([g for p in {id(p): p for p in parameters}.values() if (g := p.grad) is not None], norm_type)
        if not torch.isfinite(norm):
            raise RuntimeError(f"llattn: the total norm of order {norm_type} of the gradients is not finite, so they cannot "
                               "be clipped; error_if_nonfinite=False scales them all the same")
    norm = native.clip(parameters, True, code, max_norm, True) if native else None
    if norm is not None:
        return norm
    grads = [g for p in {id(p): p for p in parameters}.values() if (g := p.grad) is not None]
    if not grads:
        return torch.tensor(0.0)
    _no_tangents("clip_grad_norm_", *grads)
    with torch.no_grad():
        return (_clip_of if native and _plain(grads) else clip_grads_op)(grads, max_norm, code)
