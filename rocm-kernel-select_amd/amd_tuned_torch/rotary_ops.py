"""Rotary positions: pairs of columns of each query and key, turned by an angle of their token's position.

    rotary_embedding(q, k, inv_freq, positions=0, interleaved=False, scale=1.0) -> (q, k), or q without a k
    rotary_frequencies(dim, base=10000.0, scaling=None, factor=1.0, original_length=4096)
                       -> (inv_freq float64 (dim / 2,), scale)

With angle = position * inv_freq[i], pair i's (a, b) become scale * (a cos - b sin, a sin + b cos).  Pair i
is columns i and i + rot / 2, or 2 i and 2 i + 1 with `interleaved`, rot = 2 * len(inv_freq); columns from
rot on are copied.  Angles are products in 64 bits with what their rounding leaves, so far positions lose nothing:
any in 62 bits.  `rotary_embedding` is
differentiable in q and k any number of times: the way back is the same by the opposite angle.
"""
from __future__ import annotations

import math
from typing import Optional, Union

import torch

from . import _native
from . import autograd_state


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: int = 4096, fast_turns: float = 32.0, slow_turns: float = 1.0, device=None):
    """(inv_freq, scale) for `rotary_embedding` of `dim` columns: base ** (-2 i / dim), in float64.

    For contexts `factor` times the `original_length` of training, `scaling` is
    "linear": positions interpolated, every frequency divided by factor;
    "base":   the base raised to base * factor ** (dim / (dim - 2)), which leaves the fastest pair as it was and
              divides the slowest by factor;
    "parts":  frequencies of at least `fast_turns` turns within the original length as they were, those of at most
              `slow_turns` divided by factor, a linear mixture between; and a scale of 1 + 0.1 ln(factor)."""
    if dim <= 0 or dim % 2:
        raise ValueError("rotary_frequencies: dim must be even and positive")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError("rotary_frequencies: scaling must be None, 'linear', 'base' or 'parts'")
    if base <= 0 or factor <= 0 or original_length <= 0 or fast_turns <= slow_turns:
        raise ValueError("rotary_frequencies: base, factor and original_length must be positive, fast_turns above slow_turns")
    scale = 1.0
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    inv_freq = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling == "linear":
        inv_freq = inv_freq / factor
    elif scaling == "parts":
        turns = original_length * inv_freq / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        inv_freq = inv_freq * (keep + (1 - keep) / factor)
        scale = 1.0 + 0.1 * math.log(factor) if factor > 1 else 1.0
    return inv_freq.to(device), scale


def _product(a, b):
    """(a * b in float64, what its rounding left), both exact: by halves of 26 bits."""
    halves = []
    for x in (a, b):
        high = 134217729.0 * x
        high = high - (high - x)
        halves += [high, x - high]
    p = a * b
    ah, al, bh, bl = halves
    return p, ((ah * bh - p) + ah * bl + al * bh) + al * bl


def _part_of_turn(positions, inv_freq):
    """positions * inv_freq in turns, without whole ones, in float64: as the kernel takes it."""
    low = positions & 2047
    p, rest = _product((positions - low).double(), inv_freq)
    turns, left = _product(p, torch.full((), 0.15915494309189535, dtype=torch.float64, device=p.device))   # 1 / (2 pi)
    left = left + (p * -9.839338337591243e-18 + (rest + low.double() * inv_freq) * 0.15915494309189535)    # and its next 53 bits
    part = (turns - turns.round()) + left
    return part - part.round()


def rotary_embedding_ref(q, k, inv_freq, positions=0, interleaved=False, scale=1.0, inverse=False):
    """rotary_embedding in torch operations (parts of a turn in float64, the rest in float32 or wider, rounded once)."""
    acc = torch.promote_types(q.dtype, torch.float32)
    if not isinstance(positions, torch.Tensor):
        positions = positions + torch.arange(q.shape[-3], device=q.device)
    angle = 2 * math.pi * _part_of_turn(positions.expand(q.shape[:-2])[..., None, None].long(), inv_freq.double())
    cos, sin = (scale * torch.cos(angle)).to(acc), (scale * torch.sin(angle)).to(acc)
    sin = -sin if inverse else sin
    rot = 2 * inv_freq.shape[0]

    def turned(x):
        f = x.to(acc)
        head, rest = f[..., :rot], f[..., rot:]
        a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :rot // 2], head[..., rot // 2:])
        both = a * cos - b * sin, a * sin + b * cos
        head = torch.stack(both, -1).reshape(head.shape) if interleaved else torch.cat(both, -1)
        return torch.cat((head, rest), -1).to(x.dtype)

    return turned(q) if k is None else (turned(q), turned(k))


class RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, inv_freq, positions, interleaved, scale, inverse):
        tensor = isinstance(positions, torch.Tensor)
        ctx.how = None if tensor else positions, interleaved, scale, inverse
        ctx.save_for_backward(inv_freq, positions if tensor else None)
        ctx.set_materialize_grads(False)
        oq, ok = _native.rotary(q, k, inv_freq, positions, interleaved, scale, inverse)
        return oq if k is None else (oq, ok)

    @staticmethod
    def backward(ctx, dq, dk=None):
        inv_freq, positions = ctx.saved_tensors
        offset, interleaved, scale, inverse = ctx.how
        positions = offset if positions is None else positions
        given = [d for d in (dq, dk) if d is not None]
        if not given:
            return (None,) * 7
        first, second = given[0], given[1] if len(given) > 1 else None
        if autograd_state.graph_wanted(first, second):
            # batched gradients and tangents too; the way back is linear, so any number of times
            got = rotary_embedding_ref(first, second, inv_freq, positions, interleaved, scale, not inverse)
        else:
            got = _native.rotary(first, second, inv_freq, positions, interleaved, scale, not inverse)
            got = got if second is not None else got[0]
        got = list(got) if second is not None else [got]
        return (*[got.pop(0) if d is not None else None for d in (dq, dk)], None, None, None, None, None)


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], inv_freq: torch.Tensor,
                     positions: Union[int, torch.Tensor] = 0, interleaved: bool = False, scale: float = 1.0):
    """q (batch, seqlen, heads, dim) and k, alike but for its heads (or None), of float32, float16 or bfloat16, with
    any strides (a copy is made where the last axis has one); or (tokens, heads, dim) each, for packed rows and
    decoding.  inv_freq float32 or float64 (rot / 2,), rot up to dim, on the same device.  positions: that of the first
    token, or an int32 or int64 tensor with one for each token, (batch, seqlen) or what broadcasts to it.  Results are
    dense.  Only q and k have gradients."""
    interleaved, scale = bool(interleaved), float(scale)
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("rotary_embedding: inv_freq has no gradient")
    if autograd_state.recorded(q, k, inv_freq, positions):
        return rotary_embedding_ref(q, k, inv_freq, positions, interleaved, scale)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return RotaryFn.apply(q, k, inv_freq, positions, interleaved, scale, False)
    oq, ok = _native.rotary(q, k, inv_freq, positions, interleaved, scale)
    return oq if k is None else (oq, ok)
