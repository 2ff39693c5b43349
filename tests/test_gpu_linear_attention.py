"""Linear attention with a decay for each head against its recurrence in 64 bits, one token at a time.

Tolerances, element by element, from the same recurrence of the inputs' magnitudes, which bounds the sum of the
magnitudes of everything that is added into a result (`size`).  A result is rounded once to its type.  Factors in
fp32 (decays, sums) have relative errors of a few 2^-24 each; at most T / 4 + dim_k + dim_v + 100 roundings follow
each other on the way to a result of a sequence of T tokens (T / 64 chunks with a decay and 6 partial products for
each 32 tokens, then as many for each 32 columns), each of 2^-24 of the partial sums, which `size` bounds.  Where a
result is in 16 bits, two factors that are fp32 meet in two bf16 parts each: 2^-16 of each term, so 2^-15."""
from __future__ import annotations

import pytest
import torch

ULP = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.bfloat16, torch.float16, torch.float32]
gpu = pytest.mark.gpu


def close(got, want, size, steps, what="", tiny=0.0):
    assert got.shape == want.shape, what
    if not want.numel():
        return
    cut = 2.0 ** -15 if ULP[got.dtype] else 0.0
    floor = 2.0 ** -24 if got.dtype == torch.float16 else 1e-30        # half of the least step of fp16
    off = (got.double() - want).abs() - ULP[got.dtype] * want.abs() - (cut + steps * 2.0 ** -24) * size - floor - tiny
    assert off.max().item() <= 0, (what, off.max().item(), want.abs().max().item())


def spans(cu, t, n):
    if cu is None:
        return [(slice(i, i + 1), 0, t) for i in range(n)]
    ends = [min(max(int(e), 0), t) for e in cu]
    return [(slice(0, 1), a, max(a, b)) for a, b in zip(ends, ends[1:])]


def forward64(q, k, v, g, scale, state, cu):
    """(out, final states, states before every token of every sequence) in 64 bits."""
    rep = v.shape[2] // q.shape[2]
    q, k = (x.double().repeat_interleave(rep, dim=2) for x in (q, k))
    v, g = v.double(), g.double().expand(v.shape[:3])
    out, finals, kept = torch.zeros_like(v), [], []
    for i, (row, a, b) in enumerate(spans(cu, v.shape[1], v.shape[0])):
        S = v.new_zeros(1, v.shape[2], q.shape[3], v.shape[3]) if state is None else state[i:i + 1].double()
        seen = [S]
        for t in range(a, b):
            S = S * g[row, t].exp()[..., None, None] + k[row, t][..., None] * v[row, t][..., None, :]
            out[row, t] = scale * (S * q[row, t][..., None]).sum(-2)
            seen.append(S)
        finals.append(S)
        kept.append(seen)
    return out, torch.cat(finals) if finals else v.new_zeros(0, v.shape[2], q.shape[3], v.shape[3]), kept


def backward64(q, k, v, g, scale, state, cu, dout, dstate, size=False):
    """The formulas' gradients (dq, dk, dv, dg, dinitial); with `size` sums of magnitudes, of what dg is summed
    from too: q . dq, k . dk from a token on and the state's inner product at the end."""
    _, _, kept = forward64(q, k, v, g, scale, state, cu)
    hk, rep = q.shape[2], v.shape[2] // q.shape[2]
    q, k = (x.double().repeat_interleave(rep, dim=2) for x in (q, k))
    v, dout = v.double(), dout.double()
    gx = g.double().expand(v.shape[:3])
    dq, dk, dv, dg = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(gx)
    first = []
    for i, (row, a, b) in enumerate(spans(cu, v.shape[1], v.shape[0])):
        dS = torch.zeros_like(kept[i][0]) if dstate is None else dstate[i:i + 1].double()
        tail = (dS * kept[i][-1]).sum((-1, -2))
        for t in range(b - 1, a - 1, -1):
            dq[row, t] = scale * (kept[i][t - a + 1] * dout[row, t][..., None, :]).sum(-1)
            dS = dS + scale * q[row, t][..., None] * dout[row, t][..., None, :]
            dk[row, t] = (dS * v[row, t][..., None, :]).sum(-1)
            dv[row, t] = (dS * k[row, t][..., None]).sum(-2)
            dS = dS * gx[row, t].exp()[..., None, None]
            tail = tail + (q[row, t] * dq[row, t]).sum(-1) + (k[row, t] * dk[row, t]).sum(-1)
            dg[row, t] = tail if size else (dS * kept[i][t - a]).sum((-1, -2))
        first.append(dS)
    dq, dk = (x.unflatten(2, (hk, rep)).sum(3) for x in (dq, dk))
    if g.dim() == 1:
        dg = dg.sum((0, 1))
    return dq, dk, dv, dg, torch.cat(first)


def make(lead, hk, hv, dk, dv, dtype, dev, seed=0, gdtype=torch.float32, fixed=False):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*lead, *s, generator=gen)  # noqa: E731
    q, k, v = rand(hk, dk), rand(hk, dk), rand(hv, dv)
    g = -torch.exp(torch.randn(hv, generator=gen) - 2) if fixed else -torch.exp(rand(hv) - 2)
    return [t.to(dev) for t in (q.to(dtype), k.to(dtype), v.to(dtype), g.to(gdtype))]


def sizes(q, k, v, g):
    return q.abs(), k.abs(), v.abs(), g


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,hk,hv,dk,dv", [(1, 1, 1, 1, 1), (3, 2, 4, 128, 128), (2, 1, 3, 64, 100), (2, 2, 2, 130, 36),
                                           (5, 1, 2, 256, 256), (2, 3, 3, 17, 33), (1, 2, 2, 100, 7), (33, 1, 4, 32, 64),
                                           (64, 1, 4, 128, 100), (86, 1, 3, 200, 132)])
def test_update(dev, n, hk, hv, dk, dv, dtype):
    import amd_tuned_torch as P
    for fixed in (False, True):
        q, k, v, g = make((n,), hk, hv, dk, dv, dtype, dev, seed=n + dk, fixed=fixed)
        state = torch.randn(n, hv, dk, dv, generator=torch.Generator().manual_seed(1)).to(dev)
        for scale in (None, 0.5):
            sc = dk ** -0.5 if scale is None else scale
            one = [x[:, None] for x in (q, k, v)] + [g if fixed else g[:, None]]
            want, want_s, _ = forward64(*one, sc, state, None)
            size, size_s, _ = forward64(*sizes(*one), sc, state.abs(), None)
            got = P.linear_attention_update(q, k, v, g, state, scale)      # the second from the state it left
            assert got.dtype == dtype
            close(got, want[:, 0], size[:, 0], dk + 8)
            close(state, want_s, size_s, 8)


@gpu
@pytest.mark.parametrize("dv", [64, 66])
def test_update_slots_strides_and_padding(dev, dv):
    import amd_tuned_torch as P
    n, hk, hv, dk = 4, 2, 4, 96
    q, k, v, g = make((n, 3), hk, hv, dk, dv, torch.bfloat16, dev, gdtype=torch.bfloat16)
    fused = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1)[:, 1]       # one row of a projection
    a, b = hk * dk, 2 * hk * dk
    q, k, v = (fused[:, :a].unflatten(1, (hk, dk)), fused[:, a:b].unflatten(1, (hk, dk)),
               fused[:, b:].unflatten(1, (hv, dv)))
    g = g[:, 1]
    cache = torch.randn(9, 2, hv, dk, dv, device=dev)[:, 1]                        # slots apart
    before = cache.clone()
    slots = torch.tensor([7, -1, 0, 9], dtype=torch.int32, device=dev)
    live = [0, 2]
    one = [x[live][:, None] for x in (q, k, v, g)]
    want, want_s, _ = forward64(*one, dk ** -0.5, before[[7, 0]], None)
    size, size_s, _ = forward64(*sizes(*one), dk ** -0.5, before[[7, 0]].abs(), None)
    out = P.linear_attention_update(q, k, v, g, cache, state_indices=slots)
    close(out[live], want[:, 0], size[:, 0], dk + 8)
    assert out[[1, 3]].eq(0).all()
    close(cache[[7, 0]], want_s, size_s, 8)
    rest = [1, 2, 3, 4, 5, 6, 8]
    assert torch.equal(cache[rest], before[rest])
    twin = before.clone()
    ref = P.linear_attention_ops.linear_attention_update_ref(q, k, v, g, twin, state_indices=slots)
    close(ref[live], want[:, 0], size[:, 0], dk + 8)
    close(twin[[7, 0]], want_s, size_s, 8)
    assert P.linear_attention_update(q[:0], k[:0], v[:0], g[:0], cache, state_indices=slots[:0]).shape == (0, hv, dv)


SHAPES = [(1, 1, 1, 1, 1, 1), (2, 5, 2, 4, 64, 64), (1, 63, 1, 1, 16, 16), (2, 64, 1, 2, 128, 128), (1, 65, 2, 2, 100, 72),
          (3, 37, 2, 2, 128, 128), (1, 200, 1, 3, 130, 36), (1, 300, 1, 1, 256, 264), (2, 700, 1, 2, 64, 100),
          (1, 513, 2, 2, 17, 33), (1, 257, 1, 1, 3, 5), (1, 600, 1, 2, 128, 200)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sequences(dev, shape, dtype):
    import amd_tuned_torch as P
    n, t, hk, hv, dk, dv = shape
    fixed = t % 2 == 1
    args = make((n, t), hk, hv, dk, dv, dtype, dev, seed=t, fixed=fixed)
    state = torch.randn(n, hv, dk, dv, generator=torch.Generator().manual_seed(2)).to(dev)
    steps = t / 4 + dk + dv + 100
    for s in (None, state):
        want, want_s, _ = forward64(*args, dk ** -0.5, s, None)
        size, size_s, _ = forward64(*sizes(*args), dk ** -0.5, None if s is None else s.abs(), None)
        out, final = P.linear_attention(*args, initial_state=s, return_final_state=True)
        assert out.dtype == dtype and final.dtype == torch.float32 and out.is_contiguous() and final.is_contiguous()
        close(out, want, size, steps, "out")
        close(final, want_s, size_s, steps, "state")
        assert torch.equal(P.linear_attention(*args, initial_state=s), out)


PACKED = [(0, 5, 5, 70, 300), (3, 64, 129, 129, 640), (0, 0, 1, 2, 3), (10, 700)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cu", PACKED, ids=str)
@pytest.mark.parametrize("dk,dv", [(64, 100), (128, 128)])
def test_packed(dev, cu, dk, dv, dtype):
    import amd_tuned_torch as P
    hk, hv, t, n = 2, 4, cu[-1] + 9, len(cu) - 1
    args = make((1, t), hk, hv, dk, dv, dtype, dev, seed=t, gdtype=dtype)
    off = torch.tensor(cu, dtype=torch.int32, device=dev)
    state = torch.randn(n, hv, dk, dv, generator=torch.Generator().manual_seed(2)).to(dev)
    steps = t / 4 + dk + dv + 100
    for s in (None, state):
        want, want_s, _ = forward64(*args, 0.3, s, cu)
        size, size_s, _ = forward64(*sizes(*args), 0.3, None if s is None else s.abs(), cu)
        out, final = P.linear_attention(*args, 0.3, initial_state=s, return_final_state=True, cu_seqlens=off)
        close(out, want, size, steps, "out")
        close(final, want_s, size_s, steps, "state")
        assert out[0, :cu[0]].eq(0).all() and out[0, cu[-1]:].eq(0).all()


def run_backward(P, args, scale, state, cu, dout, dstate):
    leaves = [x.detach().clone().requires_grad_() for x in args] + ([] if state is None else [state.detach().clone().requires_grad_()])
    out, final = P.linear_attention(*leaves[:4], scale, initial_state=leaves[4] if state is not None else None,
                                    return_final_state=True, cu_seqlens=cu)
    ends, grads = [out], [dout]
    if dstate is not None:
        ends.append(final)
        grads.append(dstate)
    return out.detach(), torch.autograd.grad(ends, leaves, grads)


def check_backward(P, args, scale, state, cu, dout, dstate, steps):
    q, k, v, g = args
    off = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=q.device)
    out, got = run_backward(P, args, scale, state, off, dout, dstate)
    want = backward64(*args, scale, state, cu, dout, dstate)
    mag = lambda x: None if x is None else x.abs()  # noqa: E731
    size = backward64(*sizes(*args), scale, mag(state), cu, dout.abs(), mag(dstate), size=True)
    for name, a, b, c, x in zip(("dq", "dk", "dv", "dg", "dstate"), got, want, size, (*args, state)):
        assert a.dtype == x.dtype and a.shape == x.shape
        close(a, b, c, 2 * steps, name)
    return out, got


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(dev, shape, dtype):
    import amd_tuned_torch as P
    n, t, hk, hv, dk, dv = shape
    args = make((n, t), hk, hv, dk, dv, dtype, dev, seed=t, fixed=t % 2 == 0)
    gen = torch.Generator().manual_seed(3)
    dout = torch.randn(n, t, hv, dv, generator=gen).to(dev, dtype)
    state, dstate = (torch.randn(n, hv, dk, dv, generator=gen).to(dev) for _ in range(2))
    steps = t / 4 + dk + dv + 100
    check_backward(P, args, 0.4, None, None, dout, None, steps)
    out, got = check_backward(P, args, 0.4, state, None, dout, dstate, steps)
    again, more = run_backward(P, args, 0.4, state, None, dout, dstate)
    assert torch.equal(out, again) and all(torch.equal(a, b) for a, b in zip(got, more))     # same bits


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cu", PACKED, ids=str)
@pytest.mark.parametrize("dk,dv,fixed", [(64, 100, False), (128, 128, True)])
def test_packed_backward(dev, cu, dk, dv, fixed, dtype):
    import amd_tuned_torch as P
    hk, hv, t, n = 2, 4, cu[-1] + 9, len(cu) - 1
    args = make((1, t), hk, hv, dk, dv, dtype, dev, seed=t, gdtype=dtype, fixed=fixed)
    gen = torch.Generator().manual_seed(3)
    dout = torch.randn(1, t, hv, dv, generator=gen).to(dev, dtype)
    state, dstate = (torch.randn(n, hv, dk, dv, generator=gen).to(dev) for _ in range(2))
    check_backward(P, args, 0.3, state, cu, dout, dstate, t / 4 + dk + dv + 100)
