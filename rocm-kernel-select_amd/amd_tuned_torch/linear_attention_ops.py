"""Linear attention with a decay for each head: a mixer of linear-attention blocks, beside the gated delta rule.

For each sequence and value head h, with key head h // (heads_v // heads_k) and a state S of
(dim_k, dim_v) in float32:

    S_t = exp(g_t) S_{t-1} + k_t v_t^T;  out_t = scale S_t^T q_t

g is the logarithm of the decay: one for each token and value head, or one for each value head (0 is linear
attention without a decay, -inf forgets everything).

`linear_attention(q, k, v, g, scale=None, initial_state=None, return_final_state=False, cu_seqlens=None)`
runs whole sequences, of equal lengths in a batch or of any lengths packed into one row, from given states or
from nothing, and is differentiable.  The decode step `linear_attention_update(q, k, v, g, state, scale=None,
state_indices=None)` takes one token of each sequence and updates a cache of states in place.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from . import autograd_state


def linear_attention_ref(q, k, v, g, scale=None, initial_state=None, return_final_state=False, cu_seqlens=None):
    """linear_attention in torch operations, one token at a time (float32 or wider, rounded once), differentiable
    any number of times."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    acc = torch.promote_types(v.dtype, torch.float32)
    rep = v.shape[2] // q.shape[2]
    qf, kf = (t.to(acc).repeat_interleave(rep, dim=2) for t in (q, k))
    vf, gf = v.to(acc), g.to(acc).expand(v.shape[:3])
    if cu_seqlens is None:
        parts = [(slice(None), 0, v.shape[1])]
    else:
        ends = cu_seqlens.clamp(0, v.shape[1]).tolist()
        parts = [(slice(0, 1), a, max(a, b)) for a, b in zip(ends, ends[1:])]
    outs, states = [], []
    for i, (row, a, b) in enumerate(parts):
        if initial_state is None:
            S = vf.new_zeros(vf[row].shape[0], v.shape[2], q.shape[3], v.shape[3])
        else:
            S = initial_state.to(acc) if cu_seqlens is None else initial_state[i:i + 1].to(acc)
        out = []
        for t in range(a, b):
            S = S * gf[row, t].exp()[..., None, None] + kf[row, t][..., None] * vf[row, t][..., None, :]
            out.append(scale * (S * qf[row, t][..., None]).sum(-2))
        outs.append(torch.stack(out, 1) if out else vf[row, a:b])
        states.append(S)
    out = torch.cat(outs, 1) if outs else torch.zeros_like(vf)
    if cu_seqlens is not None and outs:
        out = torch.nn.functional.pad(out, (0, 0, 0, 0, ends[0], v.shape[1] - ends[-1]))
    out = out.to(v.dtype)
    if not return_final_state:
        return out
    return out, (torch.cat(states) if states else vf.new_zeros(0, v.shape[2], q.shape[3], v.shape[3]))


class LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, scale, initial_state, return_final_state, cu_seqlens):
        out, state = _native.linear_attn(q, k, v, g, scale, initial_state, cu_seqlens, return_final_state)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, g, initial_state, cu_seqlens)
        return (out, state) if return_final_state else out

    @staticmethod
    def backward(ctx, dout, dstate=None):
        q, k, v, g, initial_state, cu_seqlens = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dout is None and dstate is None:
            return (None,) * 8
        given = dout if dout is not None else dstate
        if autograd_state.graph_wanted(given, q, k, v, g, initial_state, dout, dstate):
            inputs = (q, k, v, g, initial_state)
            grads = _backward_ops(inputs, ctx.scale, cu_seqlens, dout, dstate, [need[i] for i in (0, 1, 2, 3, 5)])
        else:
            if dout is None:
                dout = torch.zeros_like(v, memory_format=torch.contiguous_format)
            grads = _native.linear_attn_backward(q, k, v, g, ctx.scale, initial_state, cu_seqlens, dout, dstate,
                                                 initial_state is not None and need[5], need[3])
        grads = [x if wanted else None for x, wanted in zip(grads, (*need[:4], need[5]))]
        return (*grads[:4], None, grads[4], None, None)


def _backward_ops(inputs, scale, cu_seqlens, dout, dstate, need):
    """The gradients from torch operations, for those that are to be differentiated again or that come
    batched (the kernels record nothing).  They are taken at views made here: an input may be computed
    from another, or be the same tensor, and the way between them is the outer backward's."""
    with torch.enable_grad():
        inputs = [None if x is None else x.view_as(x) for x in inputs]
        out, state = linear_attention_ref(*inputs[:4], scale, inputs[4], True, cu_seqlens)
        # (the final state does not depend on q, so without other gradients it has none)
        ends = [(y, dy) for y, dy in ((out, dout), (state, dstate)) if dy is not None and y.requires_grad]
        if not ends:
            return [None] * len(inputs)
        wanted = [x for x, wants in zip(inputs, need) if wants]
        grads = iter(torch.autograd.grad([y for y, _ in ends], wanted, [dy for _, dy in ends], create_graph=True,
                                         allow_unused=True))
    return [next(grads) if wants else None for wants in need]


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, scale: Optional[float] = None,
                     initial_state: Optional[torch.Tensor] = None, return_final_state: bool = False,
                     cu_seqlens: Optional[torch.Tensor] = None):
    """q, k (batch, seqlen, heads_k, dim_k), v (batch, seqlen, heads_v, dim_v), g (batch, seqlen, heads_v) or
    (heads_v,) -> out like v, or (out, final_state) with return_final_state.

    q, k and v share float32, float16 or bfloat16, with any strides (a copy is made where the last axis has one);
    g has that type or float32.  States are float32 (sequences, heads_v, dim_k, dim_v), dim_k up to 256.
    cu_seqlens int32 (sequences + 1,), on the device, packs sequences into a batch of one: sequence n has tokens
    cu_seqlens[n] to cu_seqlens[n + 1] (not decreasing); tokens of no sequence get an output, and a gradient, of
    zero.  scale: dim_k ** -0.5 by default.  A value that is not finite spoils no token before its own; gradients it
    may spoil throughout its sequence."""
    scale = float(max(q.shape[-1], 1)) ** -0.5 if scale is None else float(scale)  # (a trace has sizes as tensors)
    if autograd_state.transformed(q, k, v, g, initial_state):
        return linear_attention_ref(q, k, v, g, scale, initial_state, return_final_state, cu_seqlens)
    # (a trace records the function, to be called with whatever lengths come; the kernels' own work it cannot)
    if torch._C._is_tracing() or torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (q, k, v, g, initial_state)):
        return LinearAttentionFn.apply(q, k, v, g, scale, initial_state, return_final_state, cu_seqlens)
    out, state = _native.linear_attn(q, k, v, g, scale, initial_state, cu_seqlens, return_final_state)
    return (out, state) if return_final_state else out


class LinearAttentionUpdateFn(torch.autograd.Function):
    """The decode step where autograd is watching: the states it overwrites are gone, so it has no gradient
    and says so when asked for one."""

    @staticmethod
    def forward(ctx, q, k, v, g, state, scale, state_indices):
        return _native.linear_attn_update(q, k, v, g, state, scale, state_indices)

    @staticmethod
    def backward(ctx, dout):
        raise RuntimeError("linear_attention_update overwrites its states and has no gradient; linear_attention has one")


def linear_attention_update(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, state: torch.Tensor,
                            scale: Optional[float] = None, state_indices: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One decode step: q, k (batch, heads_k, dim_k), v (batch, heads_v, dim_v), g (batch, heads_v) or (heads_v,),
    state float32 (slots, heads_v, dim_k, dim_v) updated in place -> out (batch, heads_v, dim_v).  state_indices
    int32 (batch,): the slot of each sequence, all different; one outside [0, slots) marks a row of padding, whose
    output is zero.  Without it the state has one slot a sequence.  scale: dim_k ** -0.5 by default.  For decoding: it
    has no gradient, and a backward that comes to it, or a tangent, is an error."""
    scale = float(max(q.shape[-1], 1)) ** -0.5 if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad
                                    or state.requires_grad) or autograd_state.recorded(q, k, v, g, state):
        return LinearAttentionUpdateFn.apply(q, k, v, g, state, scale, state_indices)
    return _native.linear_attn_update(q, k, v, g, state, scale, state_indices)


def linear_attention_update_ref(q, k, v, g, state, scale=None, state_indices=None):
    """linear_attention_update in torch operations (float32; `state` is updated in place)."""
    rep = v.shape[1] // q.shape[1]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    slots = torch.arange(v.shape[0], device=v.device) if state_indices is None else state_indices.long()
    live = (slots >= 0) & (slots < state.shape[0])
    qf, kf = (t.float().repeat_interleave(rep, dim=1) for t in (q, k))
    decay = g.float().expand(v.shape[:2]).exp()[..., None, None]
    S = state[slots.clamp(0, state.shape[0] - 1)] * decay + kf[..., None] * v.float()[..., None, :]
    out = torch.where(live[:, None, None], scale * (S * qf[..., None]).sum(-2), 0.0)
    state[slots[live]] = S[live]
    return out.to(v.dtype)
