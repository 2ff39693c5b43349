"""Root-mean-square norm over the last axis, with the residual's addition in front of it and an
8-bit output with scales behind it.

    rms_norm(x, weight=None, eps=1e-6, residual=None) -> y, or (y, h) with a residual
    rms_norm_quant(x, weight=None, eps=1e-6, residual=None, dtype=torch.float8_e4m3fn,
                   group_size=None) -> (q, scales), or (q, scales, h)

h = x + residual, rounded to x's dtype: the residual stream as the next layers read it, and what
is normalised.  y = h / sqrt(mean(h^2) + eps) * weight.  q * scales stands for y: fp8 e4m3 or
int8, a scale for each row (its last axis 1) or for each run of `group_size` columns, NaN where y has
one there.  GPU tensors
of any row width up to 65536 (float32: 32768) and any row alignment.  `rms_norm` is differentiable;
`rms_norm_quant` is for inference and records no gradient.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from . import autograd_state


def rms_norm_ref(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 residual: Optional[torch.Tensor] = None):
    """rms_norm in torch operations (fp32 or wider, rounded once), differentiable any number of times."""
    acc = torch.promote_types(x.dtype, torch.float32)
    h = x if residual is None else (x.to(acc) + residual.to(acc)).to(x.dtype)
    f = h.to(acc)
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.to(acc)
    y = y.to(x.dtype)
    return y if residual is None else (y, h)


class RmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        y, h, rstd, _ = _native.rms_norm(x, weight, eps, residual, want_rstd=True)
        ctx.eps, ctx.has_residual = eps, residual is not None
        ctx.set_materialize_grads(False)
        # the norm is of h alone; x and the residual come back only where the gradient is to be
        # differentiated again
        ctx.save_for_backward(x if residual is None else h, weight, rstd)
        return y if residual is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        if dy is None:
            return dh, None, None, (dh if ctx.has_residual else None)
        if autograd_state.graph_wanted(dy, h, weight, dh):
            dx, dw = _backward_ops(h, weight, dy, dh, ctx.eps)
        else:
            dx, dw = _native.rms_norm_backward(h, dy, dh, weight, rstd, want_dw=ctx.needs_input_grad[1])
        return dx, dw, None, (dx if ctx.has_residual else None)


def _backward_ops(h, weight, dy, dh, eps):
    """The gradients in differentiable torch operations."""
    acc = torch.promote_types(h.dtype, torch.float32)
    f, g = h.to(acc), dy.to(acc)
    rstd = torch.rsqrt(f.square().mean(-1, keepdim=True) + eps)
    wg = g if weight is None else g * weight.to(acc)
    dx = rstd * (wg - f * rstd.square() * (wg * f).mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.to(acc)
    dw = None if weight is None else (g * f * rstd).flatten(0, -2).sum(0).to(weight.dtype)
    return dx.to(h.dtype), dw


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
             residual: Optional[torch.Tensor] = None):
    """x (..., N), weight (N,) of x's dtype or float32, residual like x; returns y, or (y, h) with a
    residual, h = x + residual."""
    if autograd_state.recorded(x, weight, residual):
        return rms_norm_ref(x, weight, eps, residual)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return RmsNormFn.apply(x, weight, eps, residual)
    y, h, _, _ = _native.rms_norm(x, weight, eps, residual)
    return y if residual is None else (y, h)


_TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def rms_norm_quant_ref(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                       residual: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float8_e4m3fn,
                       group_size: Optional[int] = None):
    """rms_norm_quant in torch operations."""
    acc = torch.promote_types(x.dtype, torch.float32)
    h = x if residual is None else (x.to(acc) + residual.to(acc)).to(x.dtype)
    y = rms_norm_ref(h.to(acc), weight, eps)
    n, top = x.shape[-1], _TOP[dtype]
    width = group_size or max(n, 1)
    y = torch.nn.functional.pad(y, (0, -n % width)).unflatten(-1, (-1, width)) if n else y[..., None, :]
    amax = y.abs().amax(-1, keepdim=True) if n else y.new_zeros(y.shape[:-1] + (1,))
    scales = (amax / top).clamp_min(2.0 ** -126)
    q = (y * (1 / scales)).clamp(-top, top).flatten(-2)[..., :n]
    if dtype == torch.int8:
        q = torch.where(q.isnan(), -top, q.round())  # (what the kernel stores; the scale is NaN)
    q, scales = q.to(dtype), scales.squeeze(-1)
    return (q, scales) if residual is None else (q, scales, h)


def rms_norm_quant(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   residual: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float8_e4m3fn,
                   group_size: Optional[int] = None):
    """The norm in 8 bits: (q, scales), or (q, scales, h) with a residual.  q like x in `dtype`
    (torch.float8_e4m3fn or torch.int8), scales float32 (..., 1), or (..., ceil(N / group_size)) with a
    group_size (a power of two from 16 to 256)."""
    if dtype is None:
        raise RuntimeError("rms_norm: 8-bit outputs are torch.float8_e4m3fn and torch.int8")
    if torch._C._is_tracing():
        return rms_norm_quant_ref(x, weight, eps, residual, dtype, group_size)
    y, h, _, scales = _native.rms_norm(x, weight, eps, residual, quant=dtype, group=group_size or 0)
    return (y, scales) if residual is None else (y, scales, h)
