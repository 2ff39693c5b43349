"""Linear attention where fewer bits than an fp32 product's would show: results next to a border between two values
of a 16-bit type, gradients of strong decays, values beyond a part's range."""
from __future__ import annotations

import pytest
import torch

gpu = pytest.mark.gpu


def border(dtype):
    """(a, t): 1 + 2 a is half way between 1 and the next value of dtype, t^2 is too small a part of a to stand beside
    it in 8 bits, and all sums of 1, a and t^2 fit 24 bits."""
    return (2.0 ** -9, 2.0 ** -10) if dtype == torch.bfloat16 else (2.0 ** -12, 2.0 ** -11)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("later", [0, 3, 70])
def test_results_next_to_a_border(dev, later, dtype):
    """Results of 1 + 2 a + t^2, of which fp32 loses nothing, lie just above half way, and are rounded up.  A state
    or a decayed product cut to 16 bits, 1 + a, ends half way, and is rounded down, to even.  `later`: tokens of
    zeros in front, so that the tokens lie elsewhere in their chunk, or in the next one."""
    import amd_tuned_torch as P
    a, t = border(dtype)
    up = 1 + 4 * a

    def rows(*tokens):
        x = torch.zeros(1, later + len(tokens), 1, 16)
        for i, token in enumerate(tokens):
            x[0, later + i, 0, :len(token)] = torch.tensor(token)
        return x.to(dev, dtype)

    zero, one, sum_, part, pick = (0.0,), (1.0,), (1.0, 1.0, t), (1.0, a, t), (0.0, 1.0)   # sum_ . part = 1 + a + t^2
    g = torch.zeros(1, device=dev)
    # outputs: q_1 . k_0 = 1 + a + t^2 and q_1 . k_1 = a
    q, k, v = rows(zero, sum_), rows(part, (0.0, a)), rows(one, one)
    assert P.linear_attention(q, k, v, g, 1.0)[0, -1, 0, 0].item() == up
    # a state of 1 + a + t^2, and a token that adds a
    state = torch.zeros(1, 1, 16, 16, device=dev)
    state[0, 0, 0, 0] = 1 + a + t * t
    q, k, v = rows((1.0, 1.0)), rows(pick), rows((a,))
    assert P.linear_attention(q, k, v, g, 1.0, initial_state=state)[0, -1, 0, 0].item() == up
    # gradients: dq_1 = sum over j of (dO_1 . v_j) k_j, dk_0 = sum over i of (v_0 . dO_i) q_i, dv_0 = sum over i of (k_0 . q_i) dO_i
    for name, (q, k, v, do) in {"q": (rows(one, one), rows(one, one), rows(part, (0.0, a)), rows(zero, sum_)),
                                "k": (rows(one, one), rows(one, one), rows(part, zero), rows(sum_, pick)),
                                "v": (rows(sum_, pick), rows(part, zero), rows(one, one), rows(one, one))}.items():
        leaves = {"q": q, "k": k, "v": v}
        leaf = leaves[name].requires_grad_()
        got, = torch.autograd.grad(P.linear_attention(q, k, v, g, 1.0), leaf, do)
        assert got[0, later + (1 if name == "q" else 0), 0, 0].item() == up, name


TYPES = [torch.bfloat16, torch.float16, torch.float32]


def decays64(q, k, v, g, scale, state, cu, dout, dstate, size=False):
    """The gradient of every token's log decay (1, t, heads) by the formula, exp(g_t) <S_{t-1}, dS_t>, in 64 bits.  With
    `size`, of magnitudes, the sum of what it is the sum of: of each token s from t on, q_s . dq_s and k_s . dk_s
    without the token's product with itself (what they have from other tokens and states, which has decays),
    and the end's inner product without the last token's own term."""
    rep = v.shape[2] // q.shape[2]
    q, k = (x.double().repeat_interleave(rep, dim=2) for x in (q, k))
    v, dout, g = v.double(), dout.double(), g.double().expand(v.shape[:3])
    dg = torch.zeros_like(g)
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        S = torch.zeros(v.shape[2], q.shape[3], v.shape[3], dtype=torch.float64, device=v.device) if state is None else state[i].double()
        seen = []                                                # decayed states, before each token's own term
        for t in range(a, b):
            seen.append(S * g[0, t].exp()[:, None, None])
            S = seen[-1] + k[0, t][..., None] * v[0, t][..., None, :]
        dS = torch.zeros_like(S) if dstate is None else dstate[i].double()
        total = (dS * seen[-1]).sum((-1, -2)) if seen else 0
        for t in range(b - 1, a - 1, -1):
            if size:
                total = total + scale * (q[0, t][..., None] * seen[t - a] * dout[0, t][..., None, :]).sum((-1, -2))
                total = total + ((k[0, t][..., None] * dS * v[0, t][..., None, :]).sum((-1, -2)) if t < b - 1 else 0)
                dg[0, t] = total
            dS = dS + scale * q[0, t][..., None] * dout[0, t][..., None, :]
            if not size:
                dg[0, t] = (dS * seen[t - a]).sum((-1, -2))
            dS = dS * g[0, t].exp()[:, None, None]
    return dg


def decay_case(dev, dtype, cu, hk, hv, dk, dv):
    gen = torch.Generator().manual_seed(len(cu))
    r = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
    t, n = cu[-1], len(cu) - 1
    return [r(1, t, h, d).to(dtype) for h, d in ((hk, dk), (hk, dk), (hv, dv))], r(1, t, hv, dv).to(dtype), r(n, hv, dk, dv), r(n, hv, dk, dv)


def decay_gradient(P, qkv, g, state, cu, dout, dstate):
    g = g.clone().requires_grad_()
    off = torch.tensor(cu, dtype=torch.int32, device=g.device) if len(cu) > 2 else None
    out, S = P.linear_attention(*qkv, g, 0.125, initial_state=state, return_final_state=True, cu_seqlens=off)
    ends, grads = ([out, S], [dout, dstate]) if dstate is not None else ([out], [dout])
    return torch.autograd.grad(ends, g, grads)[0]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("cu,hk,hv,dk,dv", [((0, 256), 2, 2, 64, 64), ((0, 1), 1, 2, 32, 32), ((0, 130, 131, 131, 700), 2, 4, 128, 100),
                                            ((0, 150), 1, 1, 256, 264), ((0, 2100), 1, 2, 64, 128)], ids=str)
def test_gradients_of_strong_decays(dev, cu, hk, hv, dk, dv, dtype):
    """exp(g) is all that is left of a decay's gradient, so it is right by that measure, not by that of products
    without a decay.  Tolerances: the roundings that follow each other, in number as for the other gradients,
    2 (T / 4 + dim_k + dim_v + 100), of 2^-24 of the magnitudes, which have the decays too.  And against its own
    size, in the 2-norm: a dot product of d columns and a chunk's tokens has sqrt(d_k + d_v + 64) roundings of 2^-24 by
    chance, so at most 24 of its own size, which is a token's gradient's; from t on 2 T of these are added, so a
    token's is off by sqrt(2 T) 24 2^-24 of it or less, 2^-13 for T up to 4096; a head's sum is off by as many T
    times over, sqrt(T) more for terms of random sign, and so is up to sqrt(T) 2^-13, at 256 tokens 2^-9."""
    import amd_tuned_torch as P
    qkv, dout, state, dstate = decay_case(dev, dtype, cu, hk, hv, dk, dv)
    t = max(b - a for a, b in zip(cu, cu[1:]))
    steps = 2 * (t / 4 + dk + dv + 100)
    mag = [x.abs() for x in (*qkv, dout, state, dstate)]
    for s0, s1, m0, m1 in ((state, dstate, mag[4], mag[5]), (None, None, None, None)):
        for rate in (-0.1, -2.0, -5.0, -10.0, -20.0, -40.0):
            g = torch.full((1, cu[-1], hv), rate, device=dev)
            want = decays64(*qkv, g, 0.125, s0, cu, dout, s1)
            size = decays64(*mag[:3], g, 0.125, m0, cu, mag[3], m1, size=True)
            for fixed in (False, True):
                got = decay_gradient(P, qkv, g[0, 0] if fixed else g, s0, cu, dout, s1)
                if fixed:
                    want, size = want.sum((0, 1)), size.sum((0, 1))
                assert ((got.double() - want).abs() <= steps * 2.0 ** -24 * size + 1e-37).all(), (rate, fixed)
                if not fixed or t <= 256:
                    near = 2.0 ** (-9 if fixed else -13) * want.norm()
                    assert (got.double() - want).norm() <= near, (rate, fixed, ((got.double() - want).norm() / want.norm()).item())


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gradients_of_decays_of_all_strengths(dev, dtype):
    """Weak and strong decays side by side, tokens that forget everything among them: within the roundings of the
    terms that have decays."""
    import amd_tuned_torch as P
    cu = (0, 500, 770)
    qkv, dout, state, dstate = decay_case(dev, dtype, cu, 1, 4, 64, 64)
    gen = torch.Generator().manual_seed(9)
    g = -40 * torch.rand(1, cu[-1], 4, generator=gen).to(dev) ** 4
    g[:, ::90, 1] = float("-inf")
    g[:, :, 2] = -30
    g[:, 400:, 2] = -0.01
    got = decay_gradient(P, qkv, g, state, cu, dout, dstate)
    want = decays64(*qkv, g, 0.125, state, cu, dout, dstate)
    size = decays64(*[x.abs() for x in qkv], g, 0.125, state.abs(), cu, dout.abs(), dstate.abs(), size=True)
    assert ((got.double() - want).abs() <= 2 * (500 / 4 + 228) * 2.0 ** -24 * size + 1e-37).all()
    assert got[:, ::90, 1].eq(0).all()


@gpu
@pytest.mark.parametrize("large", ["q", "k", "v", "state", "dout", "dstate"])
def test_values_that_bf16_has_not(dev, large):
    """fp32 values from bf16's largest to fp32's, in one tensor, the others so small that no result overflows."""
    from test_gpu_linear_attention import backward64, close, forward64, sizes
    import amd_tuned_torch as P
    gen = torch.Generator().manual_seed(7)
    t, most = 130, torch.finfo(torch.float32).max
    shapes = {"q": (1, t, 1, 16), "k": (1, t, 1, 16), "v": (1, t, 2, 24), "state": (1, 2, 16, 24), "dout": (1, t, 2, 24),
              "dstate": (1, 2, 16, 24)}
    x = {name: torch.randn(*s, generator=gen).to(dev) * 2.0 ** -30 for name, s in shapes.items()}
    x[large] = most * (1 - torch.rand(*shapes[large], generator=gen).to(dev) * 2.0 ** -8) * x[large].sign()
    assert (x[large].abs() > 3.3895e38).any() and x[large].isfinite().all()
    g = torch.full((1, t, 2), -0.1, device=dev)
    leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v")] + [g.clone().requires_grad_(), x["state"].clone().requires_grad_()]
    out, S = P.linear_attention(*leaves[:4], 0.25, initial_state=leaves[4], return_final_state=True)
    grads = torch.autograd.grad((out, S), leaves, (x["dout"], x["dstate"]))
    args = [leaf.detach() for leaf in leaves]
    steps = t / 4 + 16 + 24 + 100
    want, want_s, _ = forward64(*args[:4], 0.25, args[4], None)
    size, size_s, _ = forward64(*sizes(*args[:4]), 0.25, args[4].abs(), None)
    close(out.detach(), want, size, steps, "out")
    close(S.detach(), want_s, size_s, steps, "state")
    want = backward64(*args[:4], 0.25, args[4], None, x["dout"], x["dstate"])
    size = backward64(*sizes(*args[:4]), 0.25, args[4].abs(), None, x["dout"].abs(), x["dstate"].abs(), size=True)
    for name, a, b, c in zip(("dq", "dk", "dv", "dg", "dstate"), grads, want, size):
        close(a, b, c, 2 * steps, name)
