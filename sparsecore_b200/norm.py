"""The norms around a transformer block, its gate and residual scale, and the
residual add, as one operator with its gradients (``sl_norm_forward`` /
``sl_norm_backward``).

    u   = N(y; post_weight, post_bias)   the norm after the block (optional)
    out = residual + scale * gate * u    the residual stream
    h   = N(out; weight, bias)           the norm before the next block

A pre-norm block ``x = x + block(norm(x))`` becomes ``x, h = residual_norm(
block(h), x, norm.weight, norm.bias)`` with the norm of the block that
follows, so the stream is read and written once between two blocks.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _native as N

__all__ = ["residual_norm"]

_KINDS = {"layer": 0, "rms": 1}
MAX_COLS = 16384


def _vector(t, name, D, y):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"residual_norm: {name} must be a torch.Tensor, got {type(t).__name__}")
    if t.get_device() != y.get_device():
        raise RuntimeError(f"residual_norm: {name} is on {t.device} but y is on {y.device}")
    if t.shape != (D,):
        raise ValueError(f"residual_norm: {name} must have shape ({D},), got {tuple(t.shape)}")
    if t.dtype not in (y.dtype, torch.float32):
        raise ValueError(f"residual_norm: {name} must be {y.dtype} or torch.float32, got {t.dtype}")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _solid(t):
    return t if t.is_contiguous() else t.contiguous()


@functools.lru_cache(maxsize=256)
def _workspace_bytes(device, T, D, groups):
    """A function of the sizes and of the device's SM count."""
    return int(N.lib_on(device).sl_norm_workspace_bytes(T, D, groups))


def _sizes(dtype, rdtype, weight, gate, T, D, opts):
    """The plain numbers of sl_norm_args."""
    kind, eps, post_eps, scale = opts
    kinds = N.DTYPES
    dt = kinds[dtype]
    return (T, D, 1 if gate is None else gate.numel() // D, scale, eps, post_eps, kind, dt, kinds[rdtype],
            kinds[weight.dtype], dt if gate is None else kinds[gate.dtype])


def _forward(y, residual, weight, bias, gate, scale_t, pw, pb, opts, keep_stats):
    D = weight.shape[0]
    T = y.numel() // D
    y, residual, weight = _solid(y), _solid(residual), _solid(weight)
    bias, gate, pw, pb = (t if t is None else _solid(t) for t in (bias, gate, pw, pb))
    out, h = torch.empty_like(residual), torch.empty_like(y)
    stats = torch.empty(4 * T, dtype=torch.float32, device=y.device) if keep_stats else None
    a = N.NORM_ARGS.pack(y.data_ptr(), residual.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(gate), _ptr(pw), _ptr(pb),
                         out.data_ptr(), h.data_ptr(), _ptr(stats), _ptr(scale_t), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0,
                         *_sizes(y.dtype, residual.dtype, weight, gate, T, D, opts))
    N.call_on(y.device, "sl_norm_forward", a)
    return out, h, (y, weight, bias, gate, pw, pb, stats)


def _backward(ctx, dout, dh):
    dtype, opts, (has_bias, has_pb) = ctx.opts
    if ctx.after:
        y, out, weight, gate, scale_t, pw, pb, stats = ctx.saved_tensors
    else:
        out, weight, stats = ctx.saved_tensors
        y = gate = scale_t = pw = pb = None
    need = ctx.needs_input_grad
    D, dev = weight.shape[0], out.device
    T = out.numel() // D
    dout = torch.zeros_like(out) if dout is None else _solid(dout)  # an output that nothing used
    dh = torch.zeros(out.shape, dtype=dtype, device=dev) if dh is None else _solid(dh)
    dr = torch.empty_like(out)
    # Without a norm, a gate or a scale after the block both gradients are the same numbers.
    same = not ctx.after and opts[3] == 1.0 and dtype == out.dtype
    dy = torch.empty(out.shape, dtype=dtype, device=dev) if need[0] and not same else None
    dw = torch.empty_like(weight) if need[2] else None
    db = torch.empty_like(weight) if has_bias and need[3] else None
    dgate = ds = dpw = dpb = None
    if ctx.after:
        dgate = torch.empty_like(gate) if gate is not None and need[4] else None
        ds = torch.empty_like(scale_t) if scale_t is not None and need[5] else None
        dpw = torch.empty_like(pw) if pw is not None and need[6] else None
        dpb = torch.empty_like(pb) if has_pb and need[7] else None
    if T:
        sizes = _sizes(dtype, out.dtype, weight, gate, T, D, opts)
        ws = torch.empty(_workspace_bytes(dev, T, D, sizes[2]), dtype=torch.uint8, device=dev)
        w = weight.data_ptr()
        # of the bias its presence is all that is asked for
        a = N.NORM_ARGS.pack((out if y is None else y).data_ptr(), 0, w, w if has_bias else 0, _ptr(gate), _ptr(pw),
                             _ptr(pb), out.data_ptr(), 0, stats.data_ptr(), _ptr(scale_t), dout.data_ptr(),
                             dh.data_ptr(), dr.data_ptr(), _ptr(dy), _ptr(dgate), _ptr(dw), _ptr(db), _ptr(dpw),
                             _ptr(dpb), _ptr(ds), ws.data_ptr(), *sizes)
        N.call_on(dev, "sl_norm_backward", a)
    else:
        for t in (dw, db, dpw, dpb, dgate, ds):
            if t is not None:
                t.zero_()
    if same and need[0]:
        dy = dr
    return dy, dr if need[1] else None, dw, db, dgate, ds, dpw, dpb, None


_backward_once = once_differentiable(_backward)


class _ResidualNormFunction(torch.autograd.Function):
    """Inputs ``(y, residual, weight, bias, gate, scale_t, post_weight,
    post_bias, (kind, eps, post_eps, scale))``, the vectors of one type.
    Returns ``(out, h)``."""

    @staticmethod
    def forward(ctx, y, residual, weight, bias, gate, scale_t, pw, pb, opts):
        dtype = y.dtype
        out, h, (y, weight, _, gate, pw, pb, stats) = _forward(y, residual, weight, bias, gate, scale_t, pw, pb, opts, True)
        ctx.after = pw is not None or gate is not None or scale_t is not None  # something after the block
        if ctx.after:
            ctx.save_for_backward(y, out, weight, gate, scale_t, pw, pb, stats)
        else:
            ctx.save_for_backward(out, weight, stats)
        ctx.opts = (dtype, opts, (bias is not None, pb is not None))
        ctx.set_materialize_grads(False)
        return out, h

    @staticmethod
    def backward(ctx, dout, dh):
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, dout, dh)


def residual_norm(y: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                  kind: str = "layer", eps: float = 1e-5, gate: torch.Tensor | None = None, scale=1.0,
                  post_weight: torch.Tensor | None = None, post_bias: torch.Tensor | None = None,
                  post_eps: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(out, h)`` with ``out = residual + scale * gate * u``, ``u`` the block
    output ``y`` (normed by ``post_weight`` / ``post_bias`` where given), and
    ``h`` the norm of ``out``; differentiable in every tensor.

    ``y`` and ``residual``: [..., D] of one shape, D up to 16384; ``y`` float32,
    bfloat16 or float16, ``residual`` of y's type or float32 (``out`` is held in
    residual's type, ``h`` in y's; sums and statistics in 32 bits).
    ``kind``: "layer" (LayerNorm) or "rms" (RMSNorm), of both norms.
    ``weight``, ``bias``, ``post_weight``, ``post_bias``: [D], all of y's type or
    all float32.  ``gate``: [D], y's shape, or [y.shape[0], 1, ..., 1, D] (a gate
    per sequence).  ``scale``: a number, or a float32 CUDA tensor of one element
    (a learned scale).

    Raises TypeError (not tensors), RuntimeError (not on one CUDA device,
    forward-mode derivatives) and ValueError (shapes, types, kind).
    """
    for t, name in ((y, "y"), (residual, "residual"), (weight, "weight")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"residual_norm: {name} must be a torch.Tensor, got {type(t).__name__}")
    if kind not in _KINDS:
        raise ValueError(f"residual_norm: kind must be 'layer' or 'rms', got {kind!r}")
    if not y.is_cuda:
        raise RuntimeError(f"residual_norm: y must be on a CUDA device (got device={y.device}). "
                           f"sparsecore_b200 has no CPU path.")
    if residual.get_device() != y.get_device():
        raise RuntimeError(f"residual_norm: residual is on {residual.device} but y is on {y.device}")
    dtype = y.dtype
    if dtype not in N.DTYPES:
        raise ValueError(f"residual_norm: y must be float32, bfloat16 or float16, got {dtype}")
    if residual.dtype not in (dtype, torch.float32):
        raise ValueError(f"residual_norm: residual must be {dtype} or torch.float32, got {residual.dtype}")
    shape = y.shape
    if not shape or shape != residual.shape:
        raise ValueError(f"residual_norm: y and residual must have one shape [..., D], got {tuple(shape)} "
                         f"and {tuple(residual.shape)}")
    D = shape[-1]
    if not 1 <= D <= MAX_COLS:
        raise ValueError(f"residual_norm: the last dimension must be 1 to {MAX_COLS}, got {D}")
    _vector(weight, "weight", D, y)
    for t, name in ((bias, "bias"), (post_weight, "post_weight"), (post_bias, "post_bias")):
        if t is not None:
            _vector(t, name, D, y)
            if t.dtype != weight.dtype:
                raise ValueError("residual_norm: weight, bias, post_weight and post_bias must have one type")
    if post_bias is not None and post_weight is None:
        raise ValueError("residual_norm: post_bias needs post_weight")
    eps, post_eps = float(eps), float(eps if post_eps is None else post_eps)
    if not eps >= 0.0 or not post_eps >= 0.0:
        raise ValueError(f"residual_norm: eps must not be negative, got {eps}, {post_eps}")
    if gate is not None:
        if not isinstance(gate, torch.Tensor):
            raise TypeError(f"residual_norm: gate must be a torch.Tensor, got {type(gate).__name__}")
        if gate.device != y.device:
            raise RuntimeError(f"residual_norm: gate is on {gate.device} but y is on {y.device}")
        if gate.dtype not in (y.dtype, torch.float32):
            raise ValueError(f"residual_norm: gate must be {y.dtype} or torch.float32, got {gate.dtype}")
        if gate.dim() < 1 or gate.shape[-1] != D:
            raise ValueError(f"residual_norm: gate's last dimension must be {D}, got shape {tuple(gate.shape)}")
        groups = gate.numel() // D
        got = tuple(gate.shape)
        whole = got == tuple(shape)
        runs = len(got) == len(shape) and got[0] == shape[0] and all(n == 1 for n in got[1:-1])
        if not (groups == 1 or whole or runs):
            raise ValueError(f"residual_norm: gate of shape {got} is not [D], y's shape {tuple(shape)}, or "
                             f"[y.shape[0], 1, ..., D]")
    scale_t = None
    if isinstance(scale, torch.Tensor):
        if scale.device != y.device:
            raise RuntimeError(f"residual_norm: scale is on {scale.device} but y is on {y.device}")
        if scale.numel() != 1 or scale.dtype != torch.float32:
            raise ValueError("residual_norm: a tensor scale must be one float32 element")
        scale, scale_t = 1.0, scale
    N.refuse_tangents("residual_norm", y, residual, weight, bias, gate, scale_t, post_weight, post_bias)
    opts = (_KINDS[kind], eps, post_eps, float(scale))
    if torch.is_grad_enabled() and (
            y.requires_grad or residual.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
            or (gate is not None and gate.requires_grad) or (scale_t is not None and scale_t.requires_grad)
            or (post_weight is not None and post_weight.requires_grad)
            or (post_bias is not None and post_bias.requires_grad)):
        return _ResidualNormFunction.apply(y, residual, weight, bias, gate, scale_t, post_weight, post_bias, opts)
    return _forward(y, residual, weight, bias, gate, scale_t, post_weight, post_bias, opts, False)[:2]
