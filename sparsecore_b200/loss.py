"""The language-model head's loss: softmax cross entropy of ``x @ weight.T``
over a vocabulary, in pieces of it, without keeping the logits, with the
gradients of ``x`` and ``weight`` (``sl_xent_forward`` / ``sl_xent_backward``).

``F.cross_entropy(head(x), targets)`` holds logits of [tokens, vocab] and
their gradient in 32 bits; here a bounded piece of the gradient exists at a
time.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _native as N

__all__ = ["linear_cross_entropy"]

_REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}


def _args(x, weight, targets, loss, rows, prep, scratch, grad, dx, dw, ignore_index, reduction, train):
    """The bytes of sl_xent_args; pointers as numbers, 0 where there is none."""
    return N.XENT_ARGS.pack(x.data_ptr(), weight.data_ptr(), targets.data_ptr(), loss, rows, prep, scratch, grad, dx, dw,
                            x.shape[0], x.shape[1], weight.shape[0], ignore_index, N.DTYPES[x.dtype], reduction, train)


@functools.lru_cache(maxsize=256)
def _sizes_of(tokens, dim, vocab, dtype, reduction, train, x_off, w_off):
    out = (ctypes.c_int64 * 3)()
    at = ctypes.addressof(out)
    a = N.XENT_ARGS.pack(x_off, w_off, 0, 0, 0, 0, 0, 0, 0, 0, tokens, dim, vocab, 0, dtype, reduction, train)
    N.call("sl_xent_sizes", a, at, at + 8, at + 16)
    return tuple(out)


def _sizes(x, weight, reduction, train):
    """Bytes of the kept buffer, the forward and the backward call's scratch: they depend on the sizes, the
    type and on where the operands start within 16 bytes."""
    return _sizes_of(x.shape[0], x.shape[1], weight.shape[0], N.DTYPES[x.dtype], reduction, train, x.data_ptr() & 15,
                     weight.data_ptr() & 15)


def _laid_like(weight, off):
    """The weight at an address that is on 16 bytes, or is not, as it was in the forward call: that call's kept buffer is laid
    out by it.  (Hooks on saved tensors may bring it back elsewhere.)"""
    if (weight.data_ptr() & 15 != 0) == off:
        return weight
    n = weight.numel()
    return torch.empty(n + off, dtype=weight.dtype, device=weight.device)[int(off):].view(weight.shape).copy_(weight)


def _buffer(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device)


def _forward(x, weight, targets, ignore_index, reduction, train):
    dim, dev = weight.shape[1], x.device
    x, weight, targets = x.reshape(-1, dim).contiguous(), weight.contiguous(), targets.reshape(-1).contiguous()
    T = x.shape[0]
    if reduction == 2:
        loss = torch.empty(T, dtype=torch.float32, device=dev)
    elif T:
        loss = torch.empty((), dtype=torch.float32, device=dev)
    else:  # no tokens at all: the mean of nothing is NaN, their sum zero
        loss = torch.full((), 0.0 if reduction else float("nan"), device=dev)
    prep = None
    if T:
        kept, scratch, _ = _sizes(x, weight, reduction, train)
        if scratch <= 1 << 20:  # one buffer for both, where keeping the scratch too costs little
            prep = _buffer(kept + scratch, dev)
            at = prep.data_ptr() + kept
        else:
            prep, buf = _buffer(kept, dev), _buffer(scratch, dev)
            at = buf.data_ptr()
        to = loss.data_ptr()
        N.call_on(dev, "sl_xent_forward", _args(x, weight, targets, 0 if reduction == 2 else to, to if reduction == 2 else 0,
                                                prep.data_ptr(), at, 0, 0, 0, ignore_index, reduction, train))
    return loss, (x, weight, targets, prep)


def _backward(ctx, grad):
    x, weight, targets, prep = ctx.saved_tensors
    ignore_index, reduction, shape, off = ctx.opts
    weight = _laid_like(weight, off)
    need = ctx.needs_input_grad
    dev = x.device
    dx = torch.empty(shape, dtype=x.dtype, device=dev) if need[0] else None
    dw = torch.empty_like(weight) if need[1] else None
    if prep is None:
        return dx, None if dw is None else dw.zero_(), None, None, None
    grad = grad.contiguous()
    scratch = _buffer(_sizes(x, weight, reduction, 1)[2], dev)
    N.call_on(dev, "sl_xent_backward", _args(x, weight, targets, 0, 0, prep.data_ptr(), scratch.data_ptr(), grad.data_ptr(),
                                             0 if dx is None else dx.data_ptr(), 0 if dw is None else dw.data_ptr(),
                                             ignore_index, reduction, 1))
    return dx, dw, None, None, None


_backward_once = once_differentiable(_backward)


class _LinearCrossEntropyFunction(torch.autograd.Function):
    """Inputs ``(x, weight, targets, ignore_index, reduction)``; returns the loss.
    The operands' 16-bit planes, each row's maximum and its sum are kept for the
    backward pass; the logits are made again there (of a vocabulary of one
    tile their gradient is kept)."""

    @staticmethod
    def forward(ctx, x, weight, targets, ignore_index, reduction):
        loss, saved = _forward(x, weight, targets, ignore_index, reduction, 1)
        ctx.save_for_backward(*saved)
        ctx.opts = (ignore_index, reduction, x.shape, saved[1].data_ptr() & 15 != 0)
        return loss

    @staticmethod
    def backward(ctx, grad):
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, grad)


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """``F.cross_entropy(x @ weight.T, targets)`` in 32 bits, differentiable in
    ``x`` and ``weight``.

    ``x``: [..., dim], ``weight``: [vocab, dim], of one type (float32, bfloat16
    or float16); ``targets``: int64 of x's leading shape.  Tokens whose target is
    ``ignore_index`` count for nothing, whatever their row of x holds.  A target
    outside [0, vocab) gives that token (and so the sum and the mean) a NaN loss
    and NaN gradients.  ``reduction``: "mean" over the tokens that count (NaN
    where none does, with gradients of zero), "sum", or "none" (a loss for each
    token, 0 for ignored ones).  The loss is float32.

    Digits: a float32 operand is held as two fp16 planes under one power of two,
    22 bits of each element above 2^-17 of the operand's largest, smaller ones to
    within 2^-39 of the largest; softmax - onehot has 22 bits above 2^-17, and is
    held to within 2^-40 below.  For 16-bit operands it is rounded to their type
    before it is multiplied.  Sums are float32.

    Raises TypeError (not tensors), RuntimeError (not on one CUDA device,
    forward-mode derivatives) and ValueError (shapes, types, reduction).
    """
    for t, name in ((x, "x"), (weight, "weight"), (targets, "targets")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"linear_cross_entropy: {name} must be a torch.Tensor, got {type(t).__name__}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    if not x.is_cuda:
        raise RuntimeError(f"linear_cross_entropy: x must be on a CUDA device (got device={x.device}). "
                           f"sparsecore_b200 has no CPU path.")
    for t, name in ((weight, "weight"), (targets, "targets")):
        if t.get_device() != x.get_device():
            raise RuntimeError(f"linear_cross_entropy: {name} is on {t.device} but x is on {x.device}")
    if x.dtype not in N.DTYPES:
        raise ValueError(f"linear_cross_entropy: x must be float32, bfloat16 or float16, got {x.dtype}")
    if weight.dtype != x.dtype:
        raise ValueError(f"linear_cross_entropy: weight must be {x.dtype} like x, got {weight.dtype}")
    if targets.dtype != torch.int64:
        raise ValueError(f"linear_cross_entropy: targets must be torch.int64, got {targets.dtype}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_cross_entropy: x must be [..., dim] and weight [vocab, dim], got {tuple(x.shape)} "
                         f"and {tuple(weight.shape)}")
    if targets.shape != x.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: targets must have shape {tuple(x.shape[:-1])}, got {tuple(targets.shape)}")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"linear_cross_entropy: weight must not be empty, got {tuple(weight.shape)}")
    N.refuse_tangents("linear_cross_entropy", x, weight)
    code = _REDUCTIONS[reduction]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        loss = _LinearCrossEntropyFunction.apply(x, weight, targets, int(ignore_index), code)
    else:
        loss, _ = _forward(x, weight, targets, int(ignore_index), code, 0)
    return loss.view(targets.shape) if code == 2 and targets.dim() != 1 else loss
