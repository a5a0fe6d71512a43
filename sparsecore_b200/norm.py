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

import torch

from . import _native as N

__all__ = ["residual_norm"]

_KINDS = {"layer": 0, "rms": 1}
MAX_COLS = 16384


def _vector(t, name, D, y):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"residual_norm: {name} must be a torch.Tensor, got {type(t).__name__}")
    if t.device != y.device:
        raise RuntimeError(f"residual_norm: {name} is on {t.device} but y is on {y.device}")
    if t.shape != (D,):
        raise ValueError(f"residual_norm: {name} must have shape ({D},), got {tuple(t.shape)}")
    if t.dtype not in (y.dtype, torch.float32):
        raise ValueError(f"residual_norm: {name} must be {y.dtype} or torch.float32, got {t.dtype}")
    return t


def _forward(y, residual, weight, bias, gate, scale_t, pw, pb, kind, eps, post_eps, scale, keep_stats):
    T, D = y.shape
    y, residual = y.contiguous(), residual.contiguous()
    weight, bias, gate, pw, pb = (t if t is None else t.contiguous() for t in (weight, bias, gate, pw, pb))
    out, h = torch.empty_like(residual), torch.empty_like(y)
    stats = torch.empty(4, T, dtype=torch.float32, device=y.device) if keep_stats else None
    a = _args(y.dtype, residual.dtype, weight, gate, T, D, kind, eps, post_eps, scale, scale_t)
    a.y, a.residual, a.weight, a.bias = N.ptr(y), N.ptr(residual), N.ptr(weight), N.ptr(bias)
    a.gate, a.post_weight, a.post_bias = N.ptr(gate), N.ptr(pw), N.ptr(pb)
    a.out, a.h, a.stats = N.ptr(out), N.ptr(h), N.ptr(stats)
    N.call_on(y.device, "sl_norm_forward", N.byref(a))
    return out, h, (y, weight, bias, gate, pw, pb, stats)


class _ResidualNormFunction(torch.autograd.Function):
    """Inputs ``(y, residual, weight, bias, gate, scale_t, post_weight,
    post_bias, kind, eps, post_eps, scale)``; y and residual [rows, D], gate
    [groups, D], the vectors of one type.  Returns ``(out, h)``."""

    @staticmethod
    def forward(ctx, y, residual, weight, bias, gate, scale_t, pw, pb, kind, eps, post_eps, scale):
        out, h, (y, weight, bias, gate, pw, pb, stats) = _forward(y, residual, weight, bias, gate, scale_t, pw, pb, kind,
                                                                  eps, post_eps, scale, True)
        need = ctx.needs_input_grad
        keep_y = pw is not None or need[4] or need[5]
        ctx.save_for_backward(y if keep_y else None, out, weight, bias, gate, scale_t, pw, pb, stats)
        ctx.opts = (y.dtype, kind, eps, post_eps, scale)
        ctx.set_materialize_grads(False)
        return out, h

    @staticmethod
    def backward(ctx, dout, dh):
        y, out, weight, bias, gate, scale_t, pw, pb, stats = ctx.saved_tensors
        dtype, kind, eps, post_eps, scale = ctx.opts
        need = ctx.needs_input_grad
        T, D = out.shape
        dev = out.device
        dout, dh = (None if t is None else t.contiguous() for t in (dout, dh))
        dr = torch.empty_like(out)
        # Without a norm, a gate or a scale after the block both gradients are the same numbers.
        same = pw is None and gate is None and scale_t is None and scale == 1.0 and dtype == out.dtype
        like = lambda t, i: torch.empty_like(t) if t is not None and need[i] else None  # noqa: E731
        dy = torch.empty(T, D, dtype=dtype, device=dev) if need[0] and not same else None
        dw, db, dpw, dpb, dgate = like(weight, 2), like(bias, 3), like(pw, 6), like(pb, 7), like(gate, 4)
        ds = like(scale_t, 5)
        if T:
            a = _args(dtype, out.dtype, weight, gate, T, D, kind, eps, post_eps, scale, scale_t)
            groups = gate.shape[0] if gate is not None else 1
            ws = torch.empty(int(N.lib_on(dev).sl_norm_workspace_bytes(T, D, groups)), dtype=torch.uint8, device=dev)
            a.y, a.out, a.weight, a.bias = N.ptr(y), N.ptr(out), N.ptr(weight), N.ptr(bias)
            a.gate, a.post_weight, a.post_bias, a.stats = N.ptr(gate), N.ptr(pw), N.ptr(pb), N.ptr(stats)
            a.dout, a.dh, a.dresidual, a.dy = N.ptr(dout), N.ptr(dh), N.ptr(dr), N.ptr(dy)
            a.dgate, a.dweight, a.dbias = N.ptr(dgate), N.ptr(dw), N.ptr(db)
            a.dpost_weight, a.dpost_bias, a.dscale, a.workspace = N.ptr(dpw), N.ptr(dpb), N.ptr(ds), N.ptr(ws)
            N.call_on(dev, "sl_norm_backward", N.byref(a))
        else:
            for t in (dw, db, dpw, dpb, dgate, ds):
                if t is not None:
                    t.zero_()
        if same and need[0]:
            dy = dr
        return dy, dr if need[1] else None, dw, db, dgate, ds, dpw, dpb, None, None, None, None


def _args(dtype, rdtype, weight, gate, T, D, kind, eps, post_eps, scale, scale_t):
    a = N.SlNormArgs()
    a.rows, a.cols, a.gate_groups = T, D, gate.shape[0] if gate is not None else 1
    a.scale, a.eps, a.post_eps, a.kind = scale, eps, post_eps, kind
    a.dtype, a.residual_dtype, a.weight_dtype = N.DTYPES[dtype], N.DTYPES[rdtype], N.DTYPES[weight.dtype]
    a.gate_dtype = N.DTYPES[gate.dtype] if gate is not None else a.dtype
    a.scale_dev = N.ptr(scale_t)
    return a


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

    Raises TypeError (not tensors), RuntimeError (not on one CUDA device) and
    ValueError (shapes, types, kind).
    """
    for t, name in ((y, "y"), (residual, "residual"), (weight, "weight")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"residual_norm: {name} must be a torch.Tensor, got {type(t).__name__}")
    if kind not in _KINDS:
        raise ValueError(f"residual_norm: kind must be 'layer' or 'rms', got {kind!r}")
    if y.device.type != "cuda":
        raise RuntimeError(f"residual_norm: y must be on a CUDA device (got device={y.device}). "
                           f"sparsecore_b200 has no CPU path.")
    if residual.device != y.device:
        raise RuntimeError(f"residual_norm: residual is on {residual.device} but y is on {y.device}")
    if y.dtype not in N.DTYPES:
        raise ValueError(f"residual_norm: y must be float32, bfloat16 or float16, got {y.dtype}")
    if residual.dtype not in (y.dtype, torch.float32):
        raise ValueError(f"residual_norm: residual must be {y.dtype} or torch.float32, got {residual.dtype}")
    if y.dim() < 1 or y.shape != residual.shape:
        raise ValueError(f"residual_norm: y and residual must have one shape [..., D], got {tuple(y.shape)} "
                         f"and {tuple(residual.shape)}")
    D = y.shape[-1]
    if not 1 <= D <= MAX_COLS:
        raise ValueError(f"residual_norm: the last dimension must be 1 to {MAX_COLS}, got {D}")
    vectors = {"weight": weight, "bias": bias, "post_weight": post_weight, "post_bias": post_bias}
    for name, t in vectors.items():
        _vector(t, name, D, y)
    if len({t.dtype for t in vectors.values() if t is not None}) > 1:
        raise ValueError("residual_norm: weight, bias, post_weight and post_bias must have one type")
    if post_bias is not None and post_weight is None:
        raise ValueError("residual_norm: post_bias needs post_weight")
    eps, post_eps = float(eps), float(eps if post_eps is None else post_eps)
    if not eps >= 0.0 or not post_eps >= 0.0:
        raise ValueError(f"residual_norm: eps must not be negative, got {eps}, {post_eps}")
    rows = y.numel() // D
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
        shape = tuple(gate.shape)
        whole = shape == tuple(y.shape)
        runs = gate.dim() == y.dim() and shape[0] == y.shape[0] and all(n == 1 for n in shape[1:-1])
        if not (groups == 1 or whole or runs):
            raise ValueError(f"residual_norm: gate of shape {shape} is not [D], y's shape {tuple(y.shape)}, or "
                             f"[y.shape[0], 1, ..., D]")
        gate = gate.reshape(groups, D)
    scale_t = None
    if isinstance(scale, torch.Tensor):
        if scale.device != y.device:
            raise RuntimeError(f"residual_norm: scale is on {scale.device} but y is on {y.device}")
        if scale.numel() != 1 or scale.dtype != torch.float32:
            raise ValueError("residual_norm: a tensor scale must be one float32 element")
        scale, scale_t = 1.0, scale
    args = (y.reshape(rows, D), residual.reshape(rows, D), weight, bias, gate, scale_t, post_weight, post_bias,
            _KINDS[kind], eps, post_eps, float(scale))
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in args):
        out, h = _ResidualNormFunction.apply(*args)
    else:
        out, h, _ = _forward(*args, False)
    return out.reshape(y.shape), h.reshape(y.shape)
