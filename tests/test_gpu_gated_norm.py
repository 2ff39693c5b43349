"""The gated root-mean-square norm against its formulas in 64 bits.

Tolerance: on the way to a result up to 72 additions of squares follow each other (64 of a thread, then the threads'),
the sigmoid's exponential has a relative error of |z| 2^-23 and the reciprocals and products around it a few 2^-24:
with |z| up to 8, below 160 2^-24 < 2^-16 of the sum of the magnitudes that make the result.  The weight's gradient
adds one rounding for each row that is summed after another, at most all of them.  Then one rounding to the type."""
from __future__ import annotations

import pytest
import torch

ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.bfloat16, torch.float16, torch.float32]
gpu = pytest.mark.gpu


def close(got, want, size, extra=0.0, what=""):
    floor = 2.0 ** -24 if got.dtype == torch.float16 else 1e-30
    off = (got.double() - want).abs() - ULP[got.dtype] * want.abs() - (2.0 ** -16 + extra) * size - floor
    assert got.shape == want.shape and (not off.numel() or off.max().item() <= 0), (what, off.max().item())


def formulas(x, z, w, eps, first, act, group, dy):
    """[(value, sum of magnitudes)] of y, dx, dgate and dw."""
    n = x.shape[-1]
    split = lambda t: t.double().unflatten(-1, (-1, group or n))  # noqa: E731
    x, z, dy = split(x), split(z), split(dy)
    w = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w
    w = split(w)
    s = torch.sigmoid(z)
    a, slope = (z * s, s * (1 + z * (1 - s))) if act == "silu" else (s, s * (1 - s))
    u = x * a if first else x
    r = (u.square().mean(-1, keepdim=True) + eps).rsqrt()
    nn = u * r
    t = dy * w if first else dy * w * a
    y = nn * w if first else nn * w * a
    du, du_size = r * (t - nn * (t * nn).mean(-1, keepdim=True)), r * (t.abs() + nn.abs() * (t * nn).abs().mean(-1, keepdim=True))
    each = dy * nn if first else dy * nn * a
    if first:
        got = [(y, y.abs()), (du * a, du_size * a.abs()), (du * x * slope, du_size * (x * slope).abs() + (du * x).abs() * s)]
    else:
        dz = dy * w * nn
        got = [(y, y.abs()), (du, du_size), (dz * slope, dz.abs() * (slope.abs() + s * (1 + z.abs())))]
    got = [(v.flatten(-2), m.flatten(-2)) for v, m in got]
    rows = each.flatten(0, -3) if each.dim() > 2 else each[None]
    return got + [(rows.sum(0).flatten(), rows.abs().sum(0).flatten())]


def inputs(shape, dtype, dev, wtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, z, dy = r(*shape), (1.5 * r(*shape)).clamp(-8, 8), r(*shape)
    w = None if wtype is None else (1 + 0.3 * r(shape[-1])).to(dev, wtype)
    return x.to(dev, dtype), z.to(dev, dtype), w, dy.to(dev, dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("shape,group", [((1, 1), None), ((3, 5), None), ((70, 128), None), ((2, 3, 4, 64), None), ((9, 256), 64),
                                         ((33, 300), 100), ((5, 21), 3), ((1200, 200), None), ((64, 2048), 128), ((3, 2048), None),
                                         ((1100, 1030), None), ((6, 4104), None), ((4, 8192), None), ((600, 96), 32)])
def test_forward_and_gradients(dev, shape, group, first, dtype):
    import amd_tuned_torch as P
    for act, wtype in (("silu", dtype), ("sigmoid", torch.float32), ("silu", None)):
        x, z, w, dy = inputs(shape, dtype, dev, wtype, seed=shape[-1])
        want = formulas(x, z, w, 1e-5, first, act, group, dy)
        y = P.rms_norm_gated(x, z, w, 1e-5, first, act, group)
        assert y.dtype == dtype
        close(y, *want[0], what="y")
        close(P.rms_norm_ops.rms_norm_gated_ref(x, z, w, 1e-5, first, act, group), *want[0], what="statement")
        leaves = [t.requires_grad_() for t in (x, z, w) if t is not None]
        got = P.rms_norm_gated(x, z, w, 1e-5, first, act, group)
        assert torch.equal(got, y)
        grads = torch.autograd.grad(got, leaves, dy)
        rows = y.numel() // shape[-1]
        for name, a, t, b in zip(("dx", "dgate", "dw"), grads, leaves, want[1:]):
            assert a.dtype == t.dtype
            close(a, *b, extra=rows * 2.0 ** -24 if name == "dw" else 0.0, what=name)
        again = torch.autograd.grad(P.rms_norm_gated(x, z, w, 1e-5, first, act, group), leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(grads, again))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_a_projection(dev, dtype):
    """x and the gate as column ranges of wider rows; heads transposed; a broadcast gate and gradient."""
    import amd_tuned_torch as P
    x, z, w, dy = inputs((7, 3 * 97), dtype, dev, dtype)
    n = 97
    wide = torch.cat((x, z), -1)
    for a, b in ((x[:, :n], z[:, n:2 * n]), (wide[:, 5:5 + n], wide[:, 300:300 + n]), (x[::2, :n], z[1::2, :n][:3].repeat(2, 1)[:4]),
                 (x[:, :n], z[:1, :n].expand(7, n))):
        want = formulas(a, b, w[:n], 1e-6, False, "silu", None, dy[:a.shape[0], :n])
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        y = P.rms_norm_gated(a, b, w[:n])
        close(y, *want[0])
        da, db = torch.autograd.grad(y, (a, b), dy[:a.shape[0], :n])
        close(da, *want[1])
        close(db, *want[2])
    h = torch.randn(2, 4, 5, 64, device=dev).to(dtype)
    y = P.rms_norm_gated(h.transpose(1, 2), h.transpose(1, 2), None)
    close(y, *formulas(h.transpose(1, 2), h.transpose(1, 2), None, 1e-6, False, "silu", None, h.transpose(1, 2))[0])
    t = h.clone().requires_grad_()
    g, = torch.autograd.grad(P.rms_norm_gated(t, t, None).sum(), t)            # an expanded gradient; the input twice
    want = formulas(h, h, None, 1e-6, False, "silu", None, torch.ones_like(h))
    # (two gradients, each rounded to the type, are added and rounded again)
    off = (g.double() - want[1][0] - want[2][0]).abs()
    lim = ULP[dtype] * (want[1][0].abs() + want[2][0].abs() + g.double().abs()) * 1.01 + 2.0 ** -16 * (want[1][1] + want[2][1])
    assert (off <= lim).all()


@gpu
def test_edges(dev):
    import amd_tuned_torch as P
    e = torch.zeros(0, 8, device=dev)
    assert P.rms_norm_gated(e, e).shape == (0, 8)
    assert P.rms_norm_gated(torch.zeros(3, 0, device=dev), torch.zeros(3, 0, device=dev)).shape == (3, 0)
    w = torch.ones(8, device=dev, requires_grad=True)
    P.rms_norm_gated(e.clone().requires_grad_(), e, w).sum().backward()
    assert w.grad.eq(0).all()
    x = torch.randn(4, 64, device=dev)
    z = torch.randn(4, 64, device=dev)
    x[1, 3] = float("nan")                     # its row alone
    z[2, 5] = float("inf")
    y = P.rms_norm_gated(x, z)
    assert y[0].isfinite().all() and y[3].isfinite().all() and y[1].isnan().all()
    assert y[2, 5].isinf() and y[2, [0, 63]].isfinite().all()
    x, z = torch.zeros(2, 64, device=dev), torch.full((2, 64), -200.0, device=dev)
    assert P.rms_norm_gated(x, z).eq(0).all() and P.rms_norm_gated(x + 1, z).abs().max() == 0
    x.requires_grad_()
    assert torch.autograd.grad(P.rms_norm_gated(x, z).sum(), x)[0].isfinite().all()


@gpu
def test_refusals(dev):
    import amd_tuned_torch as P
    x = torch.randn(3, 64, device=dev)
    for args, kw in (((x, x.half()), {}), ((x, x[:2]), {}), ((x, x.cpu()), {}), ((x.double(), x.double()), {}),
                     ((x, x, x[0, :32]), {}), ((x, x, x[0].half()), {}), ((x, x), {"activation": "gelu"}),
                     ((x, x), {"group_size": 24}), ((x, x), {"group_size": -64}), ((x.cpu(), x.cpu()), {})):
        with pytest.raises(RuntimeError):
            P.rms_norm_gated(*args, **kw)
    wide = torch.zeros(1, 8200, device=dev)
    with pytest.raises(RuntimeError):
        P.rms_norm_gated(wide, wide)
    assert P.rms_norm_gated(wide, wide, group_size=4100).shape == wide.shape


@gpu
def test_graph_and_second_order(dev):
    import amd_tuned_torch as P
    x, z, w, dy = inputs((40, 96), torch.float32, dev, torch.float32)
    x.requires_grad_()
    z.requires_grad_()
    w.requires_grad_()
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.autograd.grad(P.rms_norm_gated(x, z, w), (x, z, w), dy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = P.rms_norm_gated(x, z, w)
        got = torch.autograd.grad(y, (x, z, w), dy)
    for _ in range(3):
        dy.normal_()
        with torch.no_grad():
            x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(P.rms_norm_gated(x, z, w), (x, z, w), dy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a second derivative is the one of the statement in torch operations
    outs = []
    for fn in (P.rms_norm_gated, P.rms_norm_ops.rms_norm_gated_ref):
        g, = torch.autograd.grad(fn(x, z, w).square().sum(), x, create_graph=True)
        outs.append(torch.autograd.grad(g.square().sum(), (x, z, w)))
    # batched gradients
    y = P.rms_norm_gated(x, z, w)
    both = torch.autograd.grad(y, (x, z, w), torch.stack((dy, 2 * dy)), is_grads_batched=True, retain_graph=True)
    for a, b, (_, size) in zip(both, torch.autograd.grad(y, (x, z, w), dy),
                               formulas(x.detach(), z.detach(), w.detach(), 1e-6, False, "silu", None, dy)[1:]):
        assert ((a[0] - b).abs() <= (2.0 ** -15 + 40 * 2.0 ** -24) * size).all()
    # the same operations but for the first output, which enters with a few 2^-24
    assert all((a - b).abs().max() <= 2.0 ** -14 * b.abs().max() for a, b in zip(*outs))


def test_statement_on_the_cpu():
    from amd_tuned_torch.rms_norm_ops import rms_norm_gated_ref
    gen = torch.Generator().manual_seed(0)
    x, z, dy = (torch.randn(3, 12, generator=gen, dtype=torch.float64) for _ in range(3))
    w = torch.randn(12, generator=gen, dtype=torch.float64)
    for first in (False, True):
        for act in ("silu", "sigmoid"):
            for group in (None, 4):
                want = formulas(x, z, w, 1e-5, first, act, group, dy)
                leaves = [t.clone().requires_grad_() for t in (x, z, w)]
                y = rms_norm_gated_ref(*leaves, 1e-5, first, act, group)
                for a, (b, _) in zip((y, *torch.autograd.grad(y, leaves, dy)), want):
                    assert (a - b).abs().max() <= 1e-13
                assert torch.autograd.gradcheck(lambda *a: rms_norm_gated_ref(*a, 1e-5, first, act, group), leaves)
