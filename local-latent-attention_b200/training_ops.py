"""Operators of the training step around the attention block, over
libllattn.so: the loss of the output head without its logits
(``linear_cross_entropy``) and the orthogonalised update of the hidden
matrices (``newton_schulz``).

As in ``ops.py``: custom ops ``llattn_b200::linear_xent / linear_xent_none /
linear_xent_none_grads / newton_schulz`` for CUDA only with fake
implementations, torch's current stream, torch-allocated outputs and
workspaces, ``RuntimeError`` on bad arguments, no CPU implementation. Plain
tensors outside ``torch.compile`` and dispatch modes go to the same functions
directly, without the dispatcher (16 us of host time a training call); fake
tensors, tracers, counters and tensor subclasses see the custom ops.
"""

from __future__ import annotations

import ctypes
from contextlib import nullcontext
from typing import Optional, Sequence

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from .ops import _dtype_code, _ptr, _require

_REDUCTIONS = {"none": _lib.XENT_NONE, "mean": _lib.XENT_MEAN, "sum": _lib.XENT_SUM}


def _stream(t: Tensor) -> int:
    """torch's current stream on t's device (without building a Stream object)."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


_HERE = nullcontext()


def _on(device: torch.device):
    """Makes `device` current where it is not."""
    return _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _no_tangents(what: str, *tensors: Optional[Tensor]) -> None:
    """Refuses forward-mode derivatives, which the kernels would drop (an autograd.Function refuses
    them itself, but calls without gradients do not go through one)."""
    if not torch.compiler.is_compiling() and forward_ad._current_level >= 0:
        for t in tensors:
            _require(t is None or forward_ad.unpack_dual(t).tangent is None,
                     f"{what} has no forward-mode derivatives (an input is a dual tensor)")


_TENSORS = (Tensor, torch.nn.Parameter)


def _direct(*tensors: Tensor) -> bool:
    """Whether a call may leave out the dispatcher: nobody traces or intercepts it."""
    return (not torch.compiler.is_compiling() and not torch._C._len_torch_dispatch_stack()
            and all(type(t) in _TENSORS for t in tensors))


# --------------------------------------------------------------------------
# softmax cross-entropy of the output projection

def _rows(t: Tensor) -> Tensor:
    """t [R, C] with contiguous columns and non-overlapping rows."""
    return t if t.stride(1) == 1 and (t.shape[0] == 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


_TYPES = (torch.bfloat16, torch.float32)
_PLAIN = torch.contiguous_format


def _check_xent(x: Tensor, w: Tensor, targets: Tensor) -> None:
    # one test on the way of every call; the messages are put together only when it fails
    if (x.is_cuda and x.dim() == 2 and w.dim() == 2 and x.shape[1] == w.shape[1] and x.dtype == w.dtype
            and x.dtype in _TYPES and targets.dtype == torch.int64 and targets.shape == x.shape[:1]
            and w.device == x.device and targets.device == x.device and w.shape[0] and w.shape[1]):
        return
    _require(x.is_cuda, "linear_cross_entropy needs CUDA tensors")
    _require(x.dim() == 2 and w.dim() == 2 and x.shape[1] == w.shape[1],
             f"x {tuple(x.shape)} and weight {tuple(w.shape)} must be [tokens, d] and [vocab, d]")
    _require(x.dtype == w.dtype, f"x is {x.dtype} and weight {w.dtype}: one dtype (or autocast) is needed")
    _require(targets.dtype == torch.int64 and targets.shape == x.shape[:1],
             f"targets must be int64 [tokens], got {targets.dtype} {tuple(targets.shape)}")
    _require(w.device == x.device and targets.device == x.device, "x, weight and targets must be on one device")
    _dtype_code(x)
    _require(False, "weight must have rows and columns")


def _xent_loss(x: Tensor, w: Tensor, targets: Tensor, ignore_index: int, reduction: int):
    """The loss, and for _xent_grads the arguments and the tensors that they
    point to (weight, targets, kept workspace); None where the tokens do not fit
    at once."""
    rows, weight, at = _rows(x), _rows(w), targets.contiguous()
    (n, d), v, dev = rows.shape, weight.shape[0], rows.device
    args = _lib.XentArgs(n, d, v, _dtype_code(rows), reduction, ignore_index, rows.data_ptr(), max(rows.stride(0), d),
                         weight.data_ptr(), max(weight.stride(0), d), at.data_ptr(), None, None, None, None, None, None, 0,
                         _lib.XENT_LOSS)
    L, ref = _lib.lib(), ctypes.byref(args)
    with _on(dev):
        size = L.llattn_xent_workspace_bytes(ref)
        if not size:
            return None
        loss = torch.empty((), dtype=torch.float32, device=dev)
        kept = torch.empty(size, dtype=torch.uint8, device=dev)
        args.loss, args.workspace, args.workspace_bytes = loss.data_ptr(), kept.data_ptr(), size
        _lib.check(L.llattn_xent(ref, _stream(x)), "llattn_xent")
    return loss, args, weight, at, kept


def _xent_grads(made, x: Tensor, w: Tensor, targets: Tensor, kept: Tensor, dx: Optional[Tensor], dw: Optional[Tensor],
                factor: Tensor) -> None:
    """dx and dw of *factor times the loss that _xent_loss made with the arguments
    `made`. Their addresses are those of then: x, w, targets and kept, the saved
    tensors, are where they are now, or copies (an offload's, a checkpoint's)."""
    L, dev = _lib.lib(), factor.device
    weight, at = _rows(w), targets.contiguous()
    args = _lib.XentArgs.from_buffer_copy(made)
    ref = ctypes.byref(args)
    args.x, args.w, args.ldw, args.targets = x.data_ptr(), weight.data_ptr(), max(weight.stride(0), args.d), at.data_ptr()
    with _on(dev):
        if L.llattn_xent_workspace_bytes(ref) != kept.numel():
            # weight's rows are aligned otherwise than kept was made for (with or without a packed copy of them)
            kept = _xent_loss(x, weight, at, args.ignore_index, args.reduction)[-1]
        args.kept, args.loss, args.stage = kept.data_ptr(), None, _lib.XENT_GRADS
        args.dx, args.dw = dx.data_ptr() if dx is not None else None, dw.data_ptr() if dw is not None else None
        size = L.llattn_xent_workspace_bytes(ref)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        args.factor, args.workspace, args.workspace_bytes = factor.data_ptr(), ws.data_ptr(), size
        _lib.check(L.llattn_xent(ref, _stream(factor)), "llattn_xent")


def _xent(x: Tensor, w: Tensor, targets: Tensor, ignore_index: int, reduction: int, *, grad_rows: Optional[Tensor] = None,
          losses: Optional[Tensor] = None, loss: Optional[Tensor] = None, dx: Optional[Tensor] = None,
          dw: Optional[Tensor] = None) -> None:
    x, w, targets = _rows(x), _rows(w), targets.contiguous()
    p = lambda t: t.data_ptr() if t is not None else None
    (n, d), v, dev = x.shape, w.shape[0], x.device
    args = _lib.XentArgs(n, d, v, _dtype_code(x), reduction, ignore_index, x.data_ptr(), max(x.stride(0), d), w.data_ptr(),
                         max(w.stride(0), d), targets.data_ptr(), p(grad_rows), p(losses), p(loss), p(dx), p(dw), None, 0)
    L, ref = _lib.lib(), ctypes.byref(args)
    with _on(dev):
        size = L.llattn_xent_workspace_bytes(ref) or 256
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        args.workspace, args.workspace_bytes = ws.data_ptr(), size
        _lib.check(L.llattn_xent(ref, _stream(x)), "llattn_xent")


def _linear_xent(x: Tensor, w: Tensor, targets: Tensor, ignore_index: int, reduction: int, need_dx: bool,
                 need_dw: bool) -> tuple[Tensor, Tensor, Tensor]:
    """Reductions mean and sum: the loss, and dx / dw of it where needed (else empty)."""
    _check_xent(x, w, targets)
    make = torch.empty if x.shape[0] else torch.zeros
    loss = make((), dtype=torch.float32, device=x.device)
    dx = make(x.shape if need_dx else (0,), dtype=x.dtype, device=x.device)
    dw = make(w.shape if need_dw else (0,), dtype=w.dtype, device=x.device)
    if x.shape[0]:
        _xent(x, w, targets, ignore_index, reduction, loss=loss, dx=dx if need_dx else None, dw=dw if need_dw else None)
    return loss, dx, dw


def _linear_xent_none(x: Tensor, w: Tensor, targets: Tensor, ignore_index: int) -> Tensor:
    """Reduction none: per-token losses."""
    _check_xent(x, w, targets)
    losses = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    if x.shape[0]:
        _xent(x, w, targets, ignore_index, _lib.XENT_NONE, losses=losses)
    return losses


def _linear_xent_none_grads(x: Tensor, w: Tensor, targets: Tensor, ignore_index: int, grad_rows: Tensor, need_dx: bool,
                            need_dw: bool) -> tuple[Tensor, Tensor]:
    """dx / dw of sum_n grad_rows[n] loss[n] (the logits recomputed)."""
    _check_xent(x, w, targets)
    make = torch.empty if x.shape[0] else torch.zeros
    dx = make(x.shape if need_dx else (0,), dtype=x.dtype, device=x.device)
    dw = make(w.shape if need_dw else (0,), dtype=w.dtype, device=x.device)
    if x.shape[0] and (need_dx or need_dw):
        _xent(x, w, targets, ignore_index, _lib.XENT_NONE, grad_rows=grad_rows.float().contiguous(),
              dx=dx if need_dx else None, dw=dw if need_dw else None)
    return dx, dw


linear_xent_op = torch.library.custom_op("llattn_b200::linear_xent", _linear_xent, mutates_args=(), device_types="cuda")
linear_xent_none_op = torch.library.custom_op("llattn_b200::linear_xent_none", _linear_xent_none, mutates_args=(),
                                              device_types="cuda")
linear_xent_none_grads_op = torch.library.custom_op("llattn_b200::linear_xent_none_grads", _linear_xent_none_grads,
                                                    mutates_args=(), device_types="cuda")


@linear_xent_op.register_fake
def _linear_xent_fake(x, w, targets, ignore_index, reduction, need_dx, need_dw):
    return (x.new_empty((), dtype=torch.float32), x.new_empty(x.shape if need_dx else (0,)),
            w.new_empty(w.shape if need_dw else (0,)))


@linear_xent_none_op.register_fake
def _linear_xent_none_fake(x, w, targets, ignore_index):
    return x.new_empty(x.shape[0], dtype=torch.float32)


@linear_xent_none_grads_op.register_fake
def _linear_xent_none_grads_fake(x, w, targets, ignore_index, grad_rows, need_dx, need_dw):
    return x.new_empty(x.shape if need_dx else (0,)), w.new_empty(w.shape if need_dw else (0,))


def _scale_(a: Tensor, b: Tensor, factor: Tensor) -> None:
    """a *= factor, b *= factor (device scalar), in one launch that leaves them alone for a factor of 1."""
    if a.numel() + b.numel():
        with _on(a.device):
            _lib.check(_lib.lib().llattn_scale(_ptr(a), a.numel(), _ptr(b), b.numel(), _dtype_code(a), _ptr(factor),
                                               _stream(a)), "llattn_scale")


class _XentReduced(torch.autograd.Function):
    """mean / sum. Where all tokens' exponentials fit in the workspace it is kept
    until the backward, whose products apply the upstream gradient; otherwise the
    gradients for an upstream gradient of 1 are computed with the loss, piece by
    piece, and scaled in the backward (27 us more for 32003 x 1408 of them)."""

    @staticmethod
    def forward(ctx, x, w, targets, ignore_index, reduction):
        need = ctx.needs_input_grad
        direct = ctx.direct = _direct(x, w, targets)
        ctx.args = None
        if direct:
            _check_xent(x, w, targets)
            got = _xent_loss(x, w, targets, ignore_index, reduction) if x.shape[0] else None
            if got is not None:
                loss, ctx.args, *saved = got
                ctx.save_for_backward(x, *saved)
                return loss
        f = _linear_xent if direct else linear_xent_op
        loss, dx, dw = f(x, w, targets, ignore_index, reduction, need[0], need[1])
        ctx.save_for_backward(x, w, targets, dx, dw)
        ctx.cfg = (ignore_index, reduction)
        ctx.spent = False
        return loss

    @staticmethod
    def backward(ctx, grad):
        # under create_graph the wrapper refuses to be differentiated; otherwise it only costs time
        return _reduced_backward_once(ctx, grad) if torch.is_grad_enabled() else _reduced_backward(ctx, grad)


def _reduced_backward(ctx, grad):
    _no_tangents("linear_cross_entropy's backward", grad)
    need = ctx.needs_input_grad
    if ctx.args is not None:
        x, w, targets, kept = ctx.saved_tensors
        dx = torch.empty_like(x, memory_format=_PLAIN) if need[0] else None
        dw = torch.empty_like(w, memory_format=_PLAIN) if need[1] else None
        _xent_grads(ctx.args, x, w, targets, kept, dx, dw, grad)
        return dx, dw, None, None, None
    x, w, targets, dx, dw = ctx.saved_tensors
    if not ctx.direct:
        return ((dx * grad).to(x.dtype) if need[0] else None, (dw * grad).to(w.dtype) if need[1] else None, None, None,
                None)
    if ctx.spent:  # a retained graph's next backward: the first one scaled the stored gradients in place
        _, dx, dw = _linear_xent(x, w, targets, *ctx.cfg, need[0], need[1])
    ctx.spent = True
    _scale_(dx, dw, grad)
    return dx if need[0] else None, dw if need[1] else None, None, None, None


_reduced_backward_once = torch.autograd.function.once_differentiable(_reduced_backward)


class _XentNone(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, targets, ignore_index):
        f = _linear_xent_none if _direct(x, w, targets) else linear_xent_none_op
        ctx.save_for_backward(x, w, targets)
        ctx.ignore_index = ignore_index
        return f(x, w, targets, ignore_index)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _no_tangents("linear_cross_entropy's backward", grad)
        x, w, targets = ctx.saved_tensors
        need = ctx.needs_input_grad
        f = _linear_xent_none_grads if _direct(x, w, targets, grad) else linear_xent_none_grads_op
        dx, dw = f(x, w, targets, ctx.ignore_index, grad, need[0], need[1])
        return dx if need[0] else None, dw if need[1] else None, None, None


def linear_cross_entropy(x: Tensor, weight: Tensor, targets: Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> Tensor:
    """Softmax cross-entropy of the logits x @ weight.T against targets, without
    the logits: what ``F.cross_entropy(F.linear(x, weight).float(), targets)``
    returns, differentiable in x and weight.

    x [..., d] and weight [vocab, d], both bfloat16 or both float32 (under
    autocast both are cast to its dtype, as a linear layer's are, or to float32
    where that is float16); targets
    [...] int64 (vocab at most 2^21, d at most 2^20). The gradients come back in
    the inputs' dtype. reduction: "mean" over the tokens whose target is not
    ignore_index (0 when there is none), "sum", or "none" (losses [...] fp32,
    0 for ignored tokens). Ignored tokens get zero gradients and their rows of x
    are not read for weight's. A target outside [0, vocab) makes the loss NaN.

    "mean" and "sum" keep the exponentials until the backward where they take at
    most half a GiB; for more tokens, and under torch.compile and dispatch modes,
    they compute the gradients together with the loss, half a GiB of exponentials
    at a time, and keep those. "none" recomputes in the backward. Gradients of
    gradients and forward-mode derivatives are not supported.

    Precision: sums are fp32. fp32 inputs keep 24 bits and their range in every
    product. bfloat16: the exponentials are held in fp16 relative to the largest
    of 128 neighbouring words (a probability under 2^-40 of it counts as 0 in the
    gradients), softmax - onehot is rounded to bfloat16 for more than 64 tokens,
    and the gradients once more; those that were computed with the loss are
    rounded again by an upstream gradient that is no power of two."""
    code = _REDUCTIONS.get(reduction)
    if code is None:
        _require(False, f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        _require(False, f"x {tuple(x.shape)} must end in weight's columns {tuple(weight.shape)}")
    if targets.shape != x.shape[:-1]:
        _require(False, f"targets {tuple(targets.shape)} must have x's leading shape {tuple(x.shape[:-1])}")
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        dt = torch.float32 if dt == torch.float16 else dt  # (no fp16 kernels)
        x, weight = x.to(dt), weight.to(dt)
    _no_tangents("linear_cross_entropy", x, weight)
    flat = x.dim() == 2
    x2, t = (x, targets) if flat else (x.reshape(-1, x.shape[-1]), targets.reshape(-1))
    grads = torch.is_grad_enabled() and (x2.requires_grad or weight.requires_grad)
    if reduction == "none":
        if grads:
            out = _XentNone.apply(x2, weight, t, ignore_index)
        else:
            out = (_linear_xent_none if _direct(x2, weight, t) else linear_xent_none_op)(x2, weight, t, ignore_index)
        return out if flat else out.view(targets.shape)
    if grads:
        return _XentReduced.apply(x2, weight, t, ignore_index, code)
    f = _linear_xent if _direct(x2, weight, t) else linear_xent_op
    return f(x2, weight, t, ignore_index, code, False, False)[0]


# --------------------------------------------------------------------------
# orthogonalised updates

DEFAULT_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _orth(gs: Sequence[Tensor], steps: int, a: float, b: float, c: float, eps: float) -> Tensor:
    """gs: matrices of one shape, dtype and device -> [len(gs), m, n] bf16."""
    g0 = gs[0]
    m, n = g0.shape
    out = torch.empty(len(gs), m, n, dtype=torch.bfloat16, device=g0.device)
    if m == 0 or n == 0:
        return out
    gs = [g.contiguous() for g in gs]
    ptrs = (ctypes.c_void_p * len(gs))(*[g.data_ptr() for g in gs])
    args = _lib.OrthArgs(m, n, len(gs), steps, _dtype_code(g0), a, b, c, eps, ptrs, _ptr(out), None, 0)
    L = _lib.lib()
    with _on(g0.device):
        ws = torch.empty(L.llattn_orth_workspace_bytes(ctypes.byref(args)) or 256, dtype=torch.uint8, device=g0.device)
        args.workspace, args.workspace_bytes = _ptr(ws), ws.numel()
        _lib.check(L.llattn_orth(ctypes.byref(args), _stream(g0)), "llattn_orth")
    return out


def _newton_schulz(g: Tensor, steps: int, a: float, b: float, c: float, eps: float) -> Tensor:
    return _orth(g.unbind(0), steps, a, b, c, eps)


newton_schulz_op = torch.library.custom_op("llattn_b200::newton_schulz", _newton_schulz, mutates_args=(),
                                           device_types="cuda")


@newton_schulz_op.register_fake
def _newton_schulz_fake(g, steps, a, b, c, eps):
    return g.new_empty(g.shape, dtype=torch.bfloat16)


@torch.no_grad()
def newton_schulz(g, *, steps: int = 5, coefficients: tuple[float, float, float] = DEFAULT_COEFFICIENTS,
                  eps: float = 1e-7):
    """Orthogonalises matrices by Newton-Schulz products, as the Muon optimiser
    does with its momentum: X = g / (|g|_F + eps), then `steps` times
    X <- a X + (b S + c S^2) X with S = X X^T, on the shorter side, so that every
    singular value of X approaches 1.

    g: a matrix [m, n], a batch [..., m, n], or a list of matrices (of any mix
    of shapes; equal shapes run as one batch), bfloat16 or float32 on CUDA.
    Returns the same structure in bfloat16 (products of 16-bit operands summed
    in fp32, also for float32: 1.7 to 2.8e-3 off, 1.7e-3 of it the result's own
    rounding; not differentiable). An all-zero matrix stays zero.

    Refused: steps outside 1 to 64, coefficients outside [-16, 16] (the fp16
    operands' range rests on them), eps below 0, sides above 2^20, more than
    65536 matrices of a shape."""
    a, b, c = (float(v) for v in coefficients)
    steps, eps = int(steps), float(eps)
    if isinstance(g, Tensor):
        _require(g.dim() >= 2, f"newton_schulz expects matrices [..., m, n], got {tuple(g.shape)}")
        _require(g.is_cuda, "newton_schulz needs CUDA tensors")
        _dtype_code(g)
        if g.numel() == 0:
            return torch.empty(g.shape, dtype=torch.bfloat16, device=g.device)
        f = _newton_schulz if _direct(g) else newton_schulz_op
        return f(g.reshape(-1, *g.shape[-2:]), steps, a, b, c, eps).view(g.shape)
    gs = list(g)
    groups: dict = {}
    for i, t in enumerate(gs):
        _require(isinstance(t, Tensor) and t.dim() == 2, "newton_schulz expects a list of matrices")
        _require(t.is_cuda, "newton_schulz needs CUDA tensors")
        _dtype_code(t)
        groups.setdefault((t.shape, t.dtype, t.device), []).append(i)
    outs: list = [None] * len(gs)
    for members in groups.values():
        batch = [gs[i] for i in members]
        out = _orth(batch, steps, a, b, c, eps) if _direct(*batch) else newton_schulz_op(torch.stack(batch), steps, a, b, c, eps)
        for i, o in zip(members, out.unbind(0)):
            outs[i] = o
    return outs
