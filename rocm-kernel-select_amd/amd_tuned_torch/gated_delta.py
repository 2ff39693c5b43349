"""The gated delta rule: the mixer of linear-attention blocks, after their causal conv1d.

For each sequence and value head h, with key head h // (heads_v // heads_k) and a state S of
(dim_k, dim_v) in float32:

    S~ = exp(g_t) S_{t-1};  u_t = beta_t (v_t - S~^T k_t);  S_t = S~ + k_t u_t^T
    out_t = scale S_t^T q_t

g is the logarithm of the decay (-inf forgets everything), beta the strength with which the value
stored under k_t is replaced.

`gated_delta_rule(q, k, v, g, beta, scale=None, initial_state=None, return_final_state=False,
cu_seqlens=None)` runs whole sequences, of equal lengths in a batch or of any lengths packed into one
row, from given states or from nothing, and is differentiable.  The decode step
`gated_delta_rule_update(q, k, v, g, beta, state, scale=None, state_indices=None)` takes one token
of each sequence and updates a cache of states in place.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from . import autograd_state


def gated_delta_rule_ref(q, k, v, g, beta, scale=None, initial_state=None, return_final_state=False,
                         cu_seqlens=None):
    """gated_delta_rule in torch operations, one token at a time (float32 or wider, rounded once),
    differentiable any number of times."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    acc = torch.promote_types(v.dtype, torch.float32)
    rep = v.shape[2] // q.shape[2]
    qf, kf = (t.to(acc).repeat_interleave(rep, dim=2) for t in (q, k))
    vf, gf, bf = v.to(acc), g.to(acc), beta.to(acc)
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
            S = S * gf[row, t].exp()[..., None, None]
            u = bf[row, t][..., None] * (vf[row, t] - (S * kf[row, t][..., None]).sum(-2))
            S = S + kf[row, t][..., None] * u[..., None, :]
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


class GatedDeltaFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, scale, initial_state, return_final_state, cu_seqlens):
        out, state = _native.gated_delta(q, k, v, g, beta, scale, initial_state, cu_seqlens, return_final_state)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, g, beta, initial_state, cu_seqlens)
        return (out, state) if return_final_state else out

    @staticmethod
    def backward(ctx, dout, dstate=None):
        q, k, v, g, beta, initial_state, cu_seqlens = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dout is None and dstate is None:
            return (None,) * 9
        given = dout if dout is not None else dstate
        if autograd_state.graph_wanted(given, q, k, v, g, beta, initial_state, dout, dstate):
            inputs = (q, k, v, g, beta, initial_state)
            grads = _backward_ops(inputs, ctx.scale, cu_seqlens, dout, dstate, [need[i] for i in (0, 1, 2, 3, 4, 6)])
        else:
            if dout is None:
                dout = torch.zeros_like(v, memory_format=torch.contiguous_format)
            grads = _native.gated_delta_backward(q, k, v, g, beta, ctx.scale, initial_state, cu_seqlens, dout, dstate,
                                                 initial_state is not None and need[6])
        grads = [x if wanted else None for x, wanted in zip(grads, (*need[:5], need[6]))]
        return (*grads[:5], None, grads[5], None, None)


def _backward_ops(inputs, scale, cu_seqlens, dout, dstate, need):
    """The gradients from torch operations, for those that are to be differentiated again or that come
    batched (the kernels record nothing).  They are taken at views made here: an input may be computed
    from another, or be the same tensor, and the way between them is the outer backward's."""
    with torch.enable_grad():
        inputs = [None if x is None else x.view_as(x) for x in inputs]
        out, state = gated_delta_rule_ref(*inputs[:5], scale, inputs[5], True, cu_seqlens)
        # (the final state does not depend on q, so without other gradients it has none)
        ends = [(y, dy) for y, dy in ((out, dout), (state, dstate)) if dy is not None and y.requires_grad]
        if not ends:
            return [None] * len(inputs)
        wanted = [x for x, wants in zip(inputs, need) if wants]
        grads = iter(torch.autograd.grad([y for y, _ in ends], wanted, [dy for _, dy in ends], create_graph=True,
                                         allow_unused=True))
    return [next(grads) if wants else None for wants in need]


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                     return_final_state: bool = False, cu_seqlens: Optional[torch.Tensor] = None):
    """q, k (batch, seqlen, heads_k, dim_k), v (batch, seqlen, heads_v, dim_v), g and beta
    (batch, seqlen, heads_v) -> out like v, or (out, final_state) with return_final_state.

    q, k and v share float32, float16 or bfloat16, with any strides (a copy is made where the last
    axis has one); g and beta have that type or float32.  States are float32
    (sequences, heads_v, dim_k, dim_v), dim_k up to 256.  cu_seqlens int32 (sequences + 1,), on the
    device, packs sequences into a batch of one: sequence n has tokens cu_seqlens[n] to
    cu_seqlens[n + 1] (not decreasing); tokens of no sequence get an output, and a gradient, of zero.
    scale: dim_k ** -0.5 by default.  Keys are used as they come: with unit length and beta in [0, 1]
    the state cannot grow.  A value that is not finite spoils no token before its own; gradients it may
    spoil throughout its 64 tokens, counted from the sequence's start."""
    scale = float(max(q.shape[-1], 1)) ** -0.5 if scale is None else float(scale)  # (a trace has sizes as tensors)
    if autograd_state.transformed(q, k, v, g, beta, initial_state):
        return gated_delta_rule_ref(q, k, v, g, beta, scale, initial_state, return_final_state, cu_seqlens)
    # (a trace records the function, to be called with whatever lengths come; the kernels' own work it cannot)
    if torch._C._is_tracing() or torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_state)):
        return GatedDeltaFn.apply(q, k, v, g, beta, scale, initial_state, return_final_state, cu_seqlens)
    out, state = _native.gated_delta(q, k, v, g, beta, scale, initial_state, cu_seqlens, return_final_state)
    return (out, state) if return_final_state else out


class GatedDeltaUpdateFn(torch.autograd.Function):
    """The decode step where autograd is watching: the states it overwrites are gone, so it has no gradient
    and says so when asked for one."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, scale, state_indices):
        return _native.gated_delta_update(q, k, v, g, beta, state, scale, state_indices)

    @staticmethod
    def backward(ctx, dout):
        raise RuntimeError("gated_delta_rule_update overwrites its states and has no gradient; gated_delta_rule has one")


def gated_delta_rule_update(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                            state: torch.Tensor, scale: Optional[float] = None,
                            state_indices: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One decode step: q, k (batch, heads_k, dim_k), v (batch, heads_v, dim_v), g and beta
    (batch, heads_v), state float32 (slots, heads_v, dim_k, dim_v) updated in place ->
    out (batch, heads_v, dim_v).  state_indices int32 (batch,): the slot of each sequence, all
    different; one outside [0, slots) marks a row of padding, whose output is zero.  Without it the
    state has one slot a sequence.  scale: dim_k ** -0.5 by default.  For decoding: it has no gradient,
    and a backward that comes to it, or a tangent, is an error."""
    scale = float(max(q.shape[-1], 1)) ** -0.5 if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad
                                    or beta.requires_grad or state.requires_grad) \
            or autograd_state.recorded(q, k, v, g, beta, state):
        return GatedDeltaUpdateFn.apply(q, k, v, g, beta, state, scale, state_indices)
    return _native.gated_delta_update(q, k, v, g, beta, state, scale, state_indices)


def gated_delta_rule_update_ref(q, k, v, g, beta, state, scale=None, state_indices=None):
    """gated_delta_rule_update in torch operations (float32; `state` is updated in place)."""
    rep = v.shape[1] // q.shape[1]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    slots = torch.arange(v.shape[0], device=v.device) if state_indices is None else state_indices.long()
    live = (slots >= 0) & (slots < state.shape[0])
    qf, kf = (t.float().repeat_interleave(rep, dim=1) for t in (q, k))
    S = state[slots.clamp(0, state.shape[0] - 1)] * g.float().exp()[..., None, None]
    u = beta.float()[..., None] * (v.float() - (S * kf[..., None]).sum(-2))
    S = S + kf[..., None] * u[..., None, :]
    out = torch.where(live[:, None, None], scale * (S * qf[..., None]).sum(-2), 0.0)
    state[slots[live]] = S[live]
    return out.to(v.dtype)
