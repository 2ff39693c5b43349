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


# ---------------------------------------------------------------------------------------------
# layouts, values and callers out of the ordinary
# ---------------------------------------------------------------------------------------------
@gpu
def test_strided_and_broadcast_inputs(dev):
    """The same numbers in another layout run through the same kernel: equal bits."""
    import amd_tuned_torch as P
    b, t, hk, hv, dk, dv = 2, 300, 2, 4, 64, 72
    q, k, v, g = make((b, t), hk, hv, dk, dv, torch.bfloat16, dev, gdtype=torch.bfloat16)
    want = P.linear_attention(q, k, v, g)
    fused = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2), v.flatten(2)[..., :3]], -1)  # odd rows
    q1, k1, v1 = fused.split([hk * dk, hk * dk, hv * dv, 3], -1)[:3]
    got = P.linear_attention(q1.unflatten(2, (hk, dk)), k1.unflatten(2, (hk, dk)), v1.unflatten(2, (hv, dv)),
                             g.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(got, want)
    heads_first = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    assert torch.equal(P.linear_attention(*(heads_first(x) for x in (q, k, v, g))), want)
    columns_first = lambda x: x.transpose(2, 3).contiguous().transpose(2, 3)  # noqa: E731
    assert torch.equal(P.linear_attention(columns_first(q), k, columns_first(v), g), want)
    one = k[:, :1].expand(b, t, hk, dk)                                        # a broadcast input, and one decay a head
    fixed = g[0, 0]
    assert torch.equal(P.linear_attention(q, one, v, fixed),
                       P.linear_attention(q, one.contiguous(), v, fixed.expand(b, t, hv).contiguous()))
    # gradients: heads first, an expanded leaf, an output gradient that is not dense
    dout = torch.randn(b, hv, t, dv, device=dev).bfloat16().transpose(1, 2)
    outs = []
    for f in (lambda x: x, heads_first, columns_first):
        leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
        outs.append(torch.autograd.grad(P.linear_attention(*(f(x) for x in leaves), g), leaves, dout if f is heads_first else dout.contiguous()))
    assert all(torch.equal(x, y) for other in outs[1:] for x, y in zip(outs[0], other))
    leaf = k[:, :1].detach().clone().requires_grad_()
    full = k[:, :1].expand(b, t, hk, dk).contiguous().requires_grad_()
    a, = torch.autograd.grad(P.linear_attention(q, leaf.expand(b, t, hk, dk), v, g), leaf, dout)
    c, = torch.autograd.grad(P.linear_attention(q, full, v, g), full, dout)
    # the expanded leaf's gradient is torch's sum of t rounded rows
    assert ((a.double() - c.double().sum(1, keepdim=True)).abs() <= 2.0 ** -7 * c.double().abs().sum(1, keepdim=True)).all()


@gpu
def test_offsets_beyond_32_bits(dev):
    """Rows of a buffer whose elements lie up to 3.3e9 apart, and slots of a state as far apart."""
    import amd_tuned_torch as P
    t, far = 100, 1 << 25
    q, k, v, g = make((1, t), 1, 1, 64, 64, torch.bfloat16, dev)
    buffer = torch.empty(t * far, dtype=torch.bfloat16, device=dev)
    rows = buffer.view(1, t, 1, far)
    for i, x in enumerate((q, k, v)):
        rows[..., i * 64:(i + 1) * 64] = x
    apart = [rows[..., i * 64:(i + 1) * 64] for i in range(3)]
    assert torch.equal(P.linear_attention(*apart, g), P.linear_attention(q, k, v, g))
    big = torch.empty(3, 1 << 30, device=dev)
    state = big.as_strided((3, 1, 64, 64), (1 << 30, 4096, 64, 1))
    state.zero_()
    idx = torch.tensor([2, 0], dtype=torch.int32, device=dev)
    args = [x[0, :2] for x in (q, k, v, g)]
    small = torch.zeros(3, 1, 64, 64, device=dev)
    assert torch.equal(P.linear_attention_update(*args, state, state_indices=idx),
                       P.linear_attention_update(*args, small, state_indices=idx))
    assert torch.equal(state, small)


@gpu
def test_many_tokens(dev):
    """A packed row of 70000 tokens: sequences of one token, of none and of most of it, against each alone."""
    import amd_tuned_torch as P
    t = 70000
    q, k, v, g = make((1, t), 1, 2, 64, 64, torch.bfloat16, dev)
    cu = [0, 1, 1, 2, 66, 69000, 69999, t]
    off = torch.tensor(cu, dtype=torch.int32, device=dev)
    out, final = P.linear_attention(q, k, v, g, cu_seqlens=off, return_final_state=True)
    size, size_s, _ = forward64(*sizes(*(x[:, 66:2066] for x in (q, k, v, g))), 0.125, None, None)
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        alone, state = P.linear_attention(*(x[:, a:b].contiguous() for x in (q, k, v, g)), return_final_state=True)
        # another length of segments: sums in another order, each of 2^-24 of at most `size`, then one rounding
        lim = 2 * 2.0 ** -8 * alone.float().abs() + (2.0 ** -15 + t / 4 * 2.0 ** -24) * size.max()
        assert ((out[:, a:b].float() - alone.float()).abs() <= lim).all(), i
        assert ((final[i] - state[0]).abs() <= t / 4 * 2.0 ** -24 * size_s.max()).all(), i


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decays_at_their_ends(dev, dtype):
    """No decay, all forgotten, hardly anything left, the type's least value, growth, decays that cancel in sums."""
    import amd_tuned_torch as P
    q, k, v, g = make((1, 150), 1, 7, 64, 64, dtype, dev)
    g[:, :, 0] = 0
    g[:, ::7, 1] = float("-inf")
    g[:, :, 2] = -40
    g[:, :, 3] = torch.finfo(torch.float32).min
    g[:, :, 4] = 0.05
    g[:, 20, 5] = -119
    g[:, 21:, 5] = -2.0 ** -12
    g[:, 100, 6] = -1e6
    state = torch.randn(1, 7, 64, 64, device=dev)
    want, want_s, _ = forward64(q, k, v, g, 0.125, state, None)
    size, size_s, _ = forward64(*sizes(q, k, v, g), 0.125, state.abs(), None)
    got, got_s = P.linear_attention(q, k, v, g, initial_state=state, return_final_state=True)
    for h in range(7):
        close(got[:, :, h], want[:, :, h], size[:, :, h], 300, h)
        close(got_s[:, h], want_s[:, h], size_s[:, h], 300, h)
    gen = torch.Generator().manual_seed(0)
    dout = torch.randn(1, 150, 7, 64, generator=gen).to(dev, dtype)
    dstate = torch.randn(1, 7, 64, 64, generator=gen).to(dev)
    _, grads = check_backward(P, (q, k, v, g), 0.125, state, None, dout, dstate, 300)
    assert grads[3][:, ::7, 1].eq(0).all() and grads[3][:, :, 3].eq(0).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite(dev, bad, dtype):
    """They spoil no token before their own, no other head and, in v, no other column."""
    import amd_tuned_torch as P
    t, at = 400, 301                               # in the second segment or later, and inside a chunk
    clean = make((1, t), 1, 2, 64, 72, dtype, dev)
    want, want_s = P.linear_attention(*clean, return_final_state=True)
    for i, name in enumerate("qkvg"):
        args = [x.clone() for x in clean]
        args[i][(0, at, 0, 5) if i < 2 else (0, at, 1, 5) if i == 2 else (0, at, 1)] = bad
        out, final = P.linear_attention(*args, return_final_state=True)
        assert torch.equal(out[:, :at], want[:, :at]), name
        if i == 0:                                 # a query's own token
            assert not out[0, at].isfinite().any() and torch.equal(out[:, at + 1:], want[:, at + 1:]) and torch.equal(final, want_s)
        elif i == 1:
            assert not out[0, at:].isfinite().any() and not final[0, :, 5].isfinite().any()
        elif i == 2:
            assert not out[0, at:, 1, 5].isfinite().any() and not final[0, 1, :, 5].isfinite().any()
            rest = [c for c in range(72) if c != 5]
            assert torch.equal(out[..., rest], want[..., rest]) and torch.equal(out[:, :, 0], want[:, :, 0])
            assert torch.equal(final[..., rest], want_s[..., rest])
        elif bad != -float("inf"):
            assert not out[0, at:, 1].isfinite().any() and torch.equal(out[:, :, 0], want[:, :, 0])
        else:
            assert out.isfinite().all()            # -inf forgets
    # a batch element, or a packed sequence, of its own
    args = [x.expand(2, *x.shape[1:]).clone() for x in clean]
    args[2][0, 3, 0, 0] = bad
    assert torch.equal(P.linear_attention(*args)[1:], want)
    off = torch.tensor([0, 200, t], dtype=torch.int32, device=dev)
    args = [x.clone() for x in clean]
    args[1][0, 199, 0, 0] = bad
    assert torch.equal(P.linear_attention(*args, cu_seqlens=off)[:, 200:], P.linear_attention(*clean, cu_seqlens=off)[:, 200:])


@gpu
def test_offsets_that_no_row_has(dev):
    """Offsets past the row or before it are clamped to it; nothing else is read or written."""
    import amd_tuned_torch as P
    args = make((1, 300), 1, 2, 64, 64, torch.bfloat16, dev)
    cu = torch.tensor([-50, 30, 1000], dtype=torch.int32, device=dev)
    good = torch.tensor([0, 30, 300], dtype=torch.int32, device=dev)
    for a, b in zip(P.linear_attention(*args, return_final_state=True, cu_seqlens=cu),
                    P.linear_attention(*args, return_final_state=True, cu_seqlens=good)):
        assert torch.equal(a, b)


@gpu
def test_continuing_and_decoding_agree_with_one_pass(dev):
    """A prompt in two parts and then token by token gives what one pass gives."""
    import amd_tuned_torch as P
    args = make((2, 150), 2, 4, 128, 64, torch.float32, dev)
    want, want_s = P.linear_attention(*args, return_final_state=True)
    size, size_s, _ = forward64(*sizes(*args), 128 ** -0.5, None, None)
    out, S = P.linear_attention(*(x[:, :80] for x in args), return_final_state=True)
    outs = [out]
    out, S = P.linear_attention(*(x[:, 80:145] for x in args), initial_state=S, return_final_state=True)
    outs.append(out)
    for t in range(145, 150):
        outs.append(P.linear_attention_update(*(x[:, t] for x in args), S)[:, None])
    close(torch.cat(outs, 1), want.double(), size, 600)
    close(S, want_s.double(), size_s, 600)


@gpu
def test_empty_calls(dev):
    import amd_tuned_torch as P
    args = make((2, 70), 1, 2, 64, 64, torch.bfloat16, dev)
    assert P.linear_attention(*(x[:0] for x in args)).shape == (0, 70, 2, 64)
    state = torch.randn(2, 2, 64, 64, device=dev)
    none = [x[:, :0].clone().requires_grad_() for x in args]
    s = state.clone().requires_grad_()
    out, S = P.linear_attention(*none, initial_state=s, return_final_state=True)
    assert out.shape == (2, 0, 2, 64) and torch.equal(S, state)
    grads = torch.autograd.grad(S, [*none, s], torch.ones_like(S), allow_unused=True)
    assert grads[4].eq(1).all() and all(x.shape == y.shape for x, y in zip(grads, none))
    fixed = torch.full((2,), -0.1, device=dev, requires_grad=True)
    _, S = P.linear_attention(*(x[:, :0] for x in args[:3]), fixed, initial_state=state, return_final_state=True)
    assert torch.autograd.grad(S.sum(), fixed)[0].eq(0).all()
    cu = torch.tensor([7], dtype=torch.int32, device=dev)
    out, S = P.linear_attention(*(x[:1] for x in args), cu_seqlens=cu, return_final_state=True)
    assert out.eq(0).all() and S.shape == (0, 2, 64, 64)
    cu = torch.tensor([5, 5, 5], dtype=torch.int32, device=dev)
    leaves = [x[:1].clone().requires_grad_() for x in args]
    out, S = P.linear_attention(*leaves, initial_state=state, cu_seqlens=cu, return_final_state=True)
    assert out.eq(0).all() and torch.equal(S, state)
    assert all(x.eq(0).all() for x in torch.autograd.grad(out.sum(), leaves))


@gpu
def test_gradients_of_some(dev):
    """Only some inputs, only one result, and without the decays' gradient: what all together give."""
    import amd_tuned_torch as P
    args = make((1, 90), 2, 4, 64, 48, torch.bfloat16, dev)
    gen = torch.Generator().manual_seed(3)
    dout = torch.randn(1, 90, 4, 48, generator=gen).to(dev, torch.bfloat16)
    state, dstate = (torch.randn(1, 4, 64, 48, generator=gen).to(dev) for _ in range(2))
    _, full = run_backward(P, args, 0.2, state, None, dout, dstate)
    want = backward64(*args, 0.2, state, None, dout, dstate)
    size = backward64(*sizes(*args), 0.2, state.abs(), None, dout.abs(), dstate.abs(), size=True)
    for wanted in ((0,), (1, 2), (3,), (4,), (0, 1, 2)):
        leaves = [x.detach().clone().requires_grad_(i in wanted) for i, x in enumerate((*args, state))]
        out, S = P.linear_attention(*leaves[:4], 0.2, initial_state=leaves[4], return_final_state=True)
        got = torch.autograd.grad((out, S), [leaves[i] for i in wanted], (dout, dstate))
        for i, x in zip(wanted, got):
            close(x, want[i], size[i], 2 * 300, i)
            if i > 1:
                assert torch.equal(x, full[i])
    leaves = [x.detach().clone().requires_grad_() for x in args]
    _, S = P.linear_attention(*leaves, 0.2, return_final_state=True)
    got = torch.autograd.grad(S, leaves, dstate, allow_unused=True)
    zero = torch.zeros_like(dout)
    want = backward64(*args, 0.2, None, None, zero, dstate)
    size = backward64(*sizes(*args), 0.2, None, None, zero, dstate.abs(), size=True)
    for x, a, b in zip(got, want, size):
        close(x, a, b, 600)


@gpu
def test_gradients_against_differences(dev):
    """The output is linear in each of q, k, v and the state, so L(x + d) - L(x - d) is twice the slope along d but
    for rounding, of 300 2^-24 of the magnitudes; along g a step of e leaves e^2 / 6 of the third derivative,
    which the magnitudes times (sum of |d| over a sequence, 4 at most here)^3 bound."""
    import amd_tuned_torch as P
    args = make((1, 100), 1, 2, 32, 40, torch.float32, dev, seed=4)
    gen = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
    state, dout, dstate = r(1, 2, 32, 40), r(1, 100, 2, 40), r(1, 2, 32, 40)

    def loss(a):
        out, S = P.linear_attention(*a[:4], 0.3, initial_state=a[4], return_final_state=True)
        return (out.double() * dout.double()).sum() + (S.double() * dstate.double()).sum()

    leaves = [*args, state]
    _, grads = run_backward(P, args, 0.3, state, None, dout, dstate)
    for i in range(5):
        d = r(*leaves[i].shape)
        e = 1.0
        if i == 3:
            d, e = d / d.abs().sum(1, keepdim=True) * 4, 2.0 ** -6
        ends = [loss([x + s * e * d if j == i else x for j, x in enumerate(leaves)]) for s in (1, -1)]
        a = [x.abs() + (e * d.abs() if j == i and i != 3 else 0) if j != 3 else x for j, x in enumerate(leaves)]
        if i == 3:
            a[3] = a[3] + e * d.abs()
        o, s, _ = forward64(*a[:4], 0.3, a[4], None)
        size = (o * dout.double().abs()).sum() + (s * dstate.double().abs()).sum()
        slope, want = (ends[0] - ends[1]) / (2 * e), (grads[i].double() * d.double()).sum()
        lim = (2 * 300 * 2.0 ** -24 / e + (e * e / 6 * 64 if i == 3 else 0)) * size
        assert (slope - want).abs() <= lim, (i, slope, want, lim)


@gpu
def test_streams_and_graphs(dev):
    """On another stream, and captured with its backward: replayed with inputs and gradients changed between."""
    import amd_tuned_torch as P
    args = [x.requires_grad_() for x in make((2, 300), 1, 2, 64, 64, torch.bfloat16, dev)]
    dout = torch.randn(2, 300, 2, 64, device=dev).bfloat16()
    call = lambda: (lambda o: (o.detach(), *torch.autograd.grad(o, args, dout)))(P.linear_attention(*args))  # noqa: E731
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(3):
        with torch.no_grad():
            args[2].normal_()
            dout.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, call()))


@gpu
def test_two_graphs_side_by_side(dev):
    """Two captured passes, replayed on two streams at once: each has a workspace of its own."""
    import amd_tuned_torch as P
    sets = []
    for seed in (0, 1):
        args = [x.requires_grad_() for x in make((1, 2000), 2, 4, 64, 64, torch.bfloat16, dev, seed=seed)]
        dout = torch.randn(1, 2000, 4, 64, device=dev).bfloat16()
        want = torch.autograd.grad(P.linear_attention(*args), args, dout)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(P.linear_attention(*args), args, dout)
        sets.append((graph, got, want, args, dout, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, _, _, _, _, stream in sets:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for s in sets for a, b in zip(s[1], s[2]))


@gpu
def test_update_in_a_graph_and_values(dev):
    import amd_tuned_torch as P
    args = make((3,), 2, 4, 128, 128, torch.bfloat16, dev)
    state = torch.randn(3, 4, 128, 128, device=dev)
    eager = state.clone()
    graph = torch.cuda.CUDAGraph()
    P.linear_attention_update(*args, state.clone())
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = P.linear_attention_update(*args, state)
    state.copy_(eager)
    for _ in range(3):
        graph.replay()
        want = P.linear_attention_update(*args, eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(state, eager)
    q, k, v, g = make((2,), 1, 2, 64, 64, torch.float32, dev)
    state = torch.randn(2, 2, 64, 64, device=dev)
    g[0] = float("-inf")
    v[1, 0, 3] = float("nan")
    one = [x[:, None] for x in (q, k, v, g)]
    want, want_s, _ = forward64(*one, 0.125, state, None)
    size, size_s, _ = forward64(*sizes(*one), 0.125, state.abs(), None)
    out = P.linear_attention_update(q, k, v, g, state)
    close(out[0], want[0, 0], size[0, 0], 72)
    close(state[0], want_s[0], size_s[0], 8)
    assert torch.equal(out[1].isnan(), want[1, 0].isnan()) and torch.equal(state[1].isnan(), want_s[1].isnan())


@gpu
def test_second_derivatives_and_transforms(dev):
    import amd_tuned_torch as P
    small = [x.requires_grad_() for x in make((1, 9), 1, 2, 8, 8, torch.float32, dev)]
    twice = []
    for fn in (P.linear_attention, P.linear_attention_ops.linear_attention_ref):
        grads = torch.autograd.grad(fn(*small).square().sum(), small, create_graph=True)
        twice.append(torch.autograd.grad(sum(x.square().sum() for x in grads), small))
    # the statement's own operations but for the first output, 2^-20 apart
    assert all((x - y).abs().max() <= 1e-4 * y.abs().max() for x, y in zip(*twice))
    with torch.no_grad():
        assert not P.linear_attention(*small).requires_grad
        plain = [x.detach() for x in small]
        got, tangent = torch.func.jvp(lambda v: P.linear_attention(plain[0], plain[1], v, plain[3]), (plain[2],), (plain[2],))
        assert (got - tangent).abs().max() <= 1e-5 * got.abs().max()          # linear in v


@gpu
def test_refusals(dev):
    import amd_tuned_torch as P
    q, k, v, g = make((2, 5), 2, 4, 32, 16, torch.bfloat16, dev)
    bad = [(q[0], k, v, g), (q, k[:, :3], v, g), (q, k.half(), v, g), (q, k, v[:, :3], g), (q, k, v[:, :, :3], g[:, :, :3]),
           (q, k, v, g.double()), (q, k, v, g.half()), (q, k, v, g[..., :2]), (q, k, v, g[0]), (q.cpu(), k, v, g), (q, k, v, g.cpu()),
           tuple(x.double() for x in (q, k, v, g))]
    for a in bad:
        with pytest.raises(RuntimeError, match="linear_attention"):
            P.linear_attention(*a)
    cu = torch.tensor([0, 5], dtype=torch.int32, device=dev)
    one = [x[:1] for x in (q, k, v, g)]
    for c, a in ((cu, (q, k, v, g)), (cu.long(), one), (cu.cpu(), one), (cu[:0], one)):
        with pytest.raises(RuntimeError, match="cu_seqlens"):
            P.linear_attention(*a, cu_seqlens=c)
    for s in (torch.zeros(2, 4, 32, 16, device=dev), torch.zeros(1, 4, 32, 16, device=dev).half(), torch.zeros(1, 4, 32, 16)):
        with pytest.raises(RuntimeError, match="initial_state"):
            P.linear_attention(*one, initial_state=s)
    with pytest.raises(RuntimeError, match="256"):
        P.linear_attention(*make((1, 5), 1, 1, 257, 8, torch.bfloat16, dev))
    q, k, v, g = make((2,), 2, 4, 32, 16, torch.bfloat16, dev)
    state = torch.zeros(2, 4, 32, 16, device=dev)
    idx = torch.zeros(2, dtype=torch.int32, device=dev)
    bad = [(q[0], k, v, g, state), (q, k[:1], v, g, state), (q, k.half(), v, g, state), (q, k, v[:, :3], g[:, :3], state[:, :3]),
           (q, k, v, g[:1], state), (q, k, v, g.double(), state), (q, k, v, g, state.bfloat16()), (q, k, v, g, state[:1]),
           (q, k, v, g, state.transpose(2, 3)), (q.cpu(), k, v, g, state), (q, k, v, g, state.cpu())]
    for a in bad:
        with pytest.raises(RuntimeError, match="linear_attention_update"):
            P.linear_attention_update(*a)
    for i in (idx.long(), idx[:1], idx.cpu()):
        with pytest.raises(RuntimeError, match="state_indices"):
            P.linear_attention_update(q, k, v, g, state, state_indices=i)
    with pytest.raises(RuntimeError, match="256"):
        P.linear_attention_update(*make((1,), 1, 1, 257, 8, torch.bfloat16, dev), torch.zeros(1, 1, 257, 8, device=dev))


@gpu
@pytest.mark.parametrize("cu", [(0, 70), (5000, 5064), (0, 0), (19999, 20000)], ids=str)
def test_rows_mostly_outside(dev, cu):
    """A packed row most of which belongs to no sequence: zeros there, written by the call."""
    import amd_tuned_torch as P
    t = 20000
    args = make((1, t), 1, 4, 64, 40, torch.bfloat16, dev)
    off = torch.tensor(cu, dtype=torch.int32, device=dev)
    keep = torch.full((1, t, 4, 40), float("nan"), device=dev, dtype=torch.bfloat16)  # what fresh memory may hold
    dout = keep.nan_to_num(1.0)
    del keep
    leaves = [x.requires_grad_() for x in args]
    out = P.linear_attention(*leaves, cu_seqlens=off)
    grads = torch.autograd.grad(out, leaves, dout)
    a, b = cu
    alone = [x.detach()[:, a:b].clone().requires_grad_() for x in args]
    want = P.linear_attention(*alone)
    want_grads = torch.autograd.grad(want, alone, dout[:, a:b])
    for x, y in zip((out, *grads), (want, *want_grads)):
        assert x[:, :a].eq(0).all() and x[:, b:].eq(0).all()
        assert (x[:, a:b].float() - y.float()).abs().max() <= 2.0 ** -6 * y.float().abs().max() if b > a else True


@gpu
def test_states_that_begin_anywhere(dev):
    """Initial states and their gradients whose first element has no alignment."""
    import amd_tuned_torch as P
    args = make((2, 700), 1, 2, 64, 64, torch.bfloat16, dev)
    n = 2 * 2 * 64 * 64
    base, dbase = torch.randn(n + 1, device=dev), torch.randn(n + 1, device=dev)
    dout = torch.randn(2, 700, 2, 64, device=dev).bfloat16()
    outs = []
    for shift in (lambda x: x[1:].view(2, 2, 64, 64), lambda x: x[1:].clone().view(2, 2, 64, 64)):
        state, dstate = shift(base), shift(dbase)
        outs.append(run_backward(P, args, 0.1, None, None, dout, dstate))
        leaves = [x.detach().requires_grad_() for x in args]
        out, S = P.linear_attention(*leaves, 0.1, initial_state=state, return_final_state=True)
        outs[-1] += (out.detach(), S.detach(), *torch.autograd.grad((out, S), leaves, (dout, dstate)))
    flat = [[y for x in o for y in (x if isinstance(x, tuple) else (x,))] for o in outs]
    assert all(torch.equal(a, b) for a, b in zip(*flat))


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_types_largest_values(dev, dtype):
    """The type's lowest and largest value, as padding may hold them, spoil no token before their own either."""
    import amd_tuned_torch as P
    t, at = 400, 301
    clean = make((1, t), 1, 2, 64, 72, dtype, dev)
    want = P.linear_attention(*clean)
    for x in (torch.finfo(dtype).min, torch.finfo(dtype).max):
        for i in (0, 1, 2):
            args = [y.clone() for y in clean]
            args[i][0, at:] = x
            assert torch.equal(P.linear_attention(*args)[:, :at], want[:, :at]), (i, x)
        args = [y.clone() for y in clean]
        args[2][0, at, 1, 5] = x
        rest = [c for c in range(72) if c != 5]
        assert torch.equal(P.linear_attention(*args)[..., rest], want[..., rest]), x


@gpu
def test_more_heads_than_a_launch(dev):
    """More sequences' heads than a launch has workgroups: every kernel of the backward is launched in parts."""
    import amd_tuned_torch as P
    n, hv, d = 65535, 136, 8                       # 8912760 of them; a launch has 2^23 waves or 2^21 workgroups
    torch.manual_seed(3)
    q, k = (torch.randn(n, 1, 1, d, device=dev).bfloat16().requires_grad_() for _ in range(2))
    v = torch.randn(n, 1, hv, d, device=dev).bfloat16().requires_grad_()
    g = (-torch.rand(n, 1, hv, device=dev)).requires_grad_()
    state, dout = torch.randn(n, hv, d, d, device=dev), torch.randn(n, 1, hv, d, device=dev).bfloat16()
    out = P.linear_attention(q, k, v, g, 1.0, initial_state=state)
    dq, dk, dv, dg = torch.autograd.grad(out, (q, k, v, g), dout)
    steps = 1 + 2 * d + 100 + hv                   # and the sum over the heads of dq and dk
    for at in (slice(0, 40), slice(30000, 30040), slice(n - 40, n)):
        few, s0, do = [x.detach()[at] for x in (q, k, v, g)], state[at], dout[at]
        want, size = forward64(*few, 1.0, s0, None)[0], forward64(*sizes(*few), 1.0, s0.abs(), None)[0]
        close(out.detach()[at], want, size, steps, "out")
        want = backward64(*few, 1.0, s0, None, do, None)
        size = backward64(*sizes(*few), 1.0, s0.abs(), None, do.abs(), None, size=True)
        for got, w, s, name in zip((dq, dk, dv, dg), want, size, ("dq", "dk", "dv", "dg")):
            close(got[at], w, s, 2 * steps, name)


def offsets(lens):
    return torch.tensor([0] + lens).cumsum(0).tolist()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_many_packed_sequences(dev, dtype):
    """More sequences than are looked at together, most of them short, some empty; one of many segments among them,
    one at the end."""
    import amd_tuned_torch as P
    torch.manual_seed(11)
    lens = torch.randint(0, 12, (260,)).tolist()
    lens[131], lens[-1] = 2100, 1500
    cu = offsets(lens)
    t, n = cu[-1] + 3, len(lens)
    args = make((1, t), 1, 2, 64, 40, dtype, dev)
    state, dstate = (torch.randn(n, 2, 64, 40, device=dev) for _ in range(2))
    dout = torch.randn(1, t, 2, 40, device=dev).to(dtype)
    check_backward(P, args, 0.125, state, cu, dout, dstate, max(lens) // 4 + 64 + 40 + 100)


@gpu
def test_packed_states_of_many_heads(dev):
    """So many heads that a workgroup joins more than its share of a state: as each sequence by itself, both within
    their rounding of `size` (here from the kernels, of magnitudes)."""
    import amd_tuned_torch as P
    lens = [4000, 1, 2500, 30, 0, 700, 1100, 64, 5, 200, 3, 90] + [7] * 30
    cu = offsets(lens)
    args = make((1, cu[-1]), 8, 64, 128, 128, torch.float32, dev)
    off = torch.tensor(cu, dtype=torch.int32, device=dev)
    dout, dstate = torch.randn(1, cu[-1], 64, 128, device=dev), torch.randn(len(lens), 64, 128, 128, device=dev)
    out, grads = run_backward(P, args, 0.1, None, off, dout, dstate)
    steps = max(lens) / 4 + 256 + 100
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        part = lambda x: x[:, a:b]  # noqa: E731
        want, _ = run_backward(P, [part(x) for x in args], 0.1, None, None, part(dout), dstate[i:i + 1])
        size = P.linear_attention(*[part(x) for x in sizes(*args)], 0.1)
        close(part(out), want.double(), 2 * size.double(), steps, i)
        if b - a in (1, 2500, 1100):
            _, want = run_backward(P, [part(x) for x in args], 0.1, None, None, part(dout), dstate[i:i + 1])
            _, size = run_backward(P, [part(x) for x in sizes(*args)], 0.1, None, None, part(dout).abs(), dstate[i:i + 1].abs())
            for got, w, m, name in zip(grads[:3], want, size, ("dq", "dk", "dv")):
                close(part(got), w.double(), 2 * m.double(), 2 * steps + 8, (i, name))
