"""Root-mean-square norm (residual's addition, 8-bit outputs, gradients) against the formula in 64
bits.

Tolerances.  A result is rounded once to its type (relative 2^-8 for bf16, 2^-11 for fp16: half a
last place at most) after fp32 arithmetic, whose sums run over a few dozen additions in a row per
thread and then a tree: 64 roundings of 2^-24 of the magnitude that was summed."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

ULP = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32 = 64 * 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def close(got, want, dtype, mag):
    """|got - want| <= one rounding of want, and fp32 arithmetic on numbers of size mag."""
    off = (got.double() - want).abs() - ULP[dtype] * want.abs() - F32 * mag
    assert off.max().item() <= 0 if off.numel() else True, off.max().item()


def inputs(shape, dtype, dev, seed=0, wdtype=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g).to(dtype).to(dev)
    r = (2 * torch.randn(shape, generator=g)).to(dtype).to(dev)
    w = (1 + 0.3 * torch.randn(shape[-1], generator=g)).to(wdtype or dtype).to(dev)
    return x, r, w


def formula(h, w, eps=1e-6):
    h = h.double()
    y = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    return y if w is None else y * w.double()


WIDTHS = [1, 7, 8, 100, 128, 129, 257, 512, 1021, 1024, 2048, 2050, 4099, 8192, 8200, 16384, 32768]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", WIDTHS)
def test_forward(dev, n, dtype):
    import amd_tuned_torch as P
    for m in (1, 5, 17):
        x, r, w = inputs((m, n), dtype, dev, seed=n + m)
        want = formula(x, w)
        close(P.rms_norm(x, w, 1e-6), want, dtype, want.abs() + 1)
        y, h = P.rms_norm(x, w, 1e-6, residual=r)
        assert torch.equal(h, (x.float() + r.float()).to(dtype))
        want = formula(h, w)
        close(y, want, dtype, want.abs() + 1)


def test_widest_rows(dev):
    import amd_tuned_torch as P
    x, r, w = inputs((3, 65536), torch.bfloat16, dev)
    want = formula(x, w)
    close(P.rms_norm(x, w), want, torch.bfloat16, want.abs() + 1)
    with pytest.raises(RuntimeError, match="columns"):
        P.rms_norm(torch.zeros(1, 65537, device=dev, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="columns"):
        P.rms_norm(torch.zeros(1, 32769, device=dev))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_shapes_and_strides(dev, dtype):
    import amd_tuned_torch as P
    x, r, w = inputs((2, 3, 130), dtype, dev, wdtype=torch.float32)
    want = formula(x, w)
    close(P.rms_norm(x, w), want, dtype, want.abs() + 1)
    close(P.rms_norm(x), formula(x, None), dtype, 4.0)
    wide = torch.randn(6, 300, device=dev).to(dtype)
    part = wide[:, 31:161]                       # rows apart, and of no alignment
    close(P.rms_norm(part, w), formula(part, w), dtype, formula(part, w).abs() + 1)
    turned = x.transpose(0, 1)
    close(P.rms_norm(turned, w), formula(turned, w), dtype, want.abs().max() + 1)
    y, h = P.rms_norm(part, w, residual=wide[:, :130])
    assert torch.equal(h, (part.float() + wide[:, :130].float()).to(dtype))
    close(y, formula(h, w), dtype, formula(h, w).abs() + 1)
    for empty in ((0, 128), (2, 0, 64)):
        assert P.rms_norm(torch.empty(empty, device=dev, dtype=dtype)).shape == empty
    ones = torch.full((4, 128), float("inf"), device=dev, dtype=dtype)
    assert P.rms_norm(ones).isnan().all()        # inf / inf, as the formula
    assert P.rms_norm(torch.zeros(4, 128, device=dev, dtype=dtype)).eq(0).all()


def check_quant(q, scales, y, dtype, group):
    """q * scales stands for y within half a step: of 1 for int8, of 2^-3 of the value (or 2^-9, the least
    step) for fp8; the scale is max|y| / top to fp32 arithmetic."""
    n = y.shape[-1]
    width = group or n
    top = 448.0 if dtype == torch.float8_e4m3fn else 127.0
    for i, a in enumerate(range(0, n, width)):
        part, s = y[..., a:a + width], scales[..., i:i + 1].double()
        want = part.abs().amax(-1, keepdim=True) / top
        assert ((s - want.clamp_min(2.0 ** -126)).abs() <= 2 * F32 * want).all()
        v = part / s
        half = 0.5 if dtype == torch.int8 else torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10))
        got = q[..., a:a + width].float().double()
        assert ((got - v).abs() <= half + 4 * F32 * v.abs()).all()
        assert got.abs().max() <= top


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 31, 64, 128, 129, 257, 1021, 2048, 4100, 8200])
def test_eight_bits(dev, n, dtype, out):
    import amd_tuned_torch as P
    for m, group in ((1, None), (5, None), (5, 16), (18, 32), (3, 128), (3, 256)):
        x, r, w = inputs((m, n), dtype, dev, seed=n + m)
        x[0] = 0 if m > 1 else x[0]
        q, s = P.rms_norm_quant(x, w, 1e-6, dtype=out, group_size=group)
        assert q.dtype == out and s.dtype == torch.float32 and s.shape == (m, -(-n // group) if group else 1)
        check_quant(q, s, formula(x, w), out, group)
        q, s, h = P.rms_norm_quant(x, w, 1e-6, residual=r, dtype=out, group_size=group)
        assert torch.equal(h, (x.float() + r.float()).to(dtype))
        check_quant(q, s, formula(h, w), out, group)


def test_eight_bits_of_nothing_and_nan(dev):
    import amd_tuned_torch as P
    q, s = P.rms_norm_quant(torch.zeros(3, 200, device=dev), None, 0.0, dtype=torch.float8_e4m3fn, group_size=64)
    assert q.float().isnan().all()               # 0 / 0 without an eps, as the formula
    q, s = P.rms_norm_quant(torch.zeros(3, 200, device=dev), None, 1e-6, dtype=torch.int8)
    assert q.eq(0).all() and s.gt(0).all()
    x = torch.randn(3, 200, device=dev)
    x[1, 7] = float("nan")
    q, s = P.rms_norm_quant(x, None, 1e-6)
    assert q[1].float().isnan().all() and not q[[0, 2]].float().isnan().any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(1, 1), (3, 7), (33, 100), (70, 128), (5, 257), (129, 1021), (9, 2048), (2100, 136),
                                 (3, 4099), (2, 16384), (2, 32768)])
def test_gradients(dev, m, n, dtype):
    import amd_tuned_torch as P
    for wdtype in (dtype, torch.float32):
        x, r, w = inputs((m, n), dtype, dev, seed=m + n, wdtype=wdtype)
        dy, dh, _ = inputs((m, n), dtype, dev, seed=m + n + 1)
        for residual in (False, True):
            a = [t.detach().clone().requires_grad_() for t in ((x, w, r) if residual else (x, w))]
            if residual:
                y, h = P.rms_norm(a[0], a[1], 1e-6, residual=a[2])
                grads = torch.autograd.grad((y, h), a, (dy, dh))
                assert torch.equal(grads[0], grads[2])
            else:
                grads = torch.autograd.grad(P.rms_norm(a[0], a[1], 1e-6), a, dy)
                h = x
            h, g, wd = h.detach().double(), dy.double(), w.double()
            rstd = (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
            inner = (wd * g * h).mean(-1, keepdim=True)
            want = rstd * (wd * g - h * rstd * rstd * inner) + (dh.double() if residual else 0)
            mag = rstd * ((wd * g).abs() + h.abs() * rstd * rstd * (wd * g * h).abs().mean(-1, keepdim=True)) + 3
            close(grads[0], want, dtype, mag)
            close(grads[1], (g * h * rstd).sum(0), wdtype, (g * h * rstd).abs().sum(0))


def test_gradient_against_differences(dev):
    """(L(x + e d) - L(x - e d)) / 2e of the kernel's own fp32 forward, e = 2^-6: the cubic term is below
    e^2 of the derivative's own size, and rounding below 2^-24 / e of L's terms."""
    import amd_tuned_torch as P
    x, r, w = (t.requires_grad_() for t in inputs((6, 100), torch.float32, dev, seed=5))
    dy, dh, _ = inputs((6, 100), torch.float32, dev, seed=6)

    def loss(x, w, r):
        y, h = P.rms_norm(x, w, 1e-6, residual=r)
        return (y.double() * dy.double()).sum() + (h.double() * dh.double()).sum()

    grads = torch.autograd.grad(loss(x, w, r), (x, w, r))
    e = 2.0 ** -6
    for i, at in enumerate((x, w, r)):
        d = torch.randn(at.shape, generator=torch.Generator().manual_seed(i)).to(dev)
        ends = []
        for sign in (1, -1):
            a = [t.detach() for t in (x, w, r)]
            a[i] = a[i] + sign * e * d
            ends.append(loss(*a))
        slope = ((ends[0] - ends[1]) / (2 * e)).item()
        want = (grads[i].double() * d.double()).sum().item()
        size = (grads[i].double().norm() * d.double().norm()).item()
        assert abs(slope - want) <= 4 * e * e * size + 1e-4 * size, (i, slope, want)


def test_second_derivatives_and_partial_gradients(dev):
    import amd_tuned_torch as P
    x, r, w = (t.requires_grad_() for t in inputs((3, 40), torch.float32, dev, seed=9))
    for fn in (P.rms_norm, P.rms_norm_ops.rms_norm_ref):
        y, h = fn(x, w, 1e-6, residual=r)
        g, = torch.autograd.grad((y * y).sum() + h.sum(), x, create_graph=True)
        got = torch.autograd.grad((g * g).sum(), (x, w, r))
        if fn is P.rms_norm:
            kept = got
    for a, b in zip(kept, got):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max()
    y, h = P.rms_norm(x, w, 1e-6, residual=r)
    assert torch.equal(torch.autograd.grad(h.sum(), r)[0], torch.ones_like(r))   # only the stream is used
    y, h = P.rms_norm(x.detach(), w, 1e-6, residual=r.detach())
    assert torch.autograd.grad(y.sum(), w)[0].shape == w.shape
    with torch.no_grad():
        assert not P.rms_norm(x, w).requires_grad
    tangent = torch.func.jvp(lambda t: P.rms_norm(t, w.detach()), (x.detach(),), (torch.ones_like(x),))[1]
    assert tangent.shape == x.shape


def test_fixed_order_and_streams(dev):
    import amd_tuned_torch as P
    x, r, w = (t.requires_grad_() for t in inputs((5000, 128), torch.bfloat16, dev))
    dy = torch.randn(5000, 128, device=dev).bfloat16()
    first = torch.autograd.grad(P.rms_norm(x, w), (x, w), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = torch.autograd.grad(P.rms_norm(x, w), (x, w), dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_refusals(dev):
    import amd_tuned_torch as P
    x = torch.randn(4, 64, device=dev)
    for call in (lambda: P.rms_norm(x.cpu()), lambda: P.rms_norm(x.double()), lambda: P.rms_norm(x, x[0, :32]),
                 lambda: P.rms_norm(x, x[0].half()), lambda: P.rms_norm(x, residual=x[:2]),
                 lambda: P.rms_norm(x, residual=x.half()), lambda: P.rms_norm(torch.tensor(1.0, device=dev)),
                 lambda: P.rms_norm_quant(x, dtype=torch.uint8), lambda: P.rms_norm_quant(x, dtype=None),
                 lambda: P.rms_norm_quant(x, group_size=24), lambda: P.rms_norm_quant(x, group_size=512),
                 lambda: P.rms_norm_quant(x, group_size=-16)):
        with pytest.raises(RuntimeError, match="rms_norm"):
            call()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 3, 4, 5, 9, 15, 63, 127, 511, 513, 1023, 1025, 2047, 2049, 8191, 8193, 16383, 16385,
                               32767])
def test_rows_that_end_inside_a_vector(dev, n, dtype):
    """Rows amid NaN, from an odd element on, with an fp32 weight: nothing beyond a row is taken for part
    of it, and nothing beyond the output is written."""
    import amd_tuned_torch as P
    m = 3
    x, r, w = inputs((m, n), dtype, dev, seed=n, wdtype=torch.float32)
    wide = [torch.full((m, n + 4), float("nan"), dtype=dtype, device=dev) for _ in range(2)]
    for b, t in zip(wide, (x, r)):
        b[:, 1:n + 1] = t
    xv, rv = (b[:, 1:n + 1] for b in wide)
    y, h = P.rms_norm(xv, w, 1e-6, residual=rv)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    want = formula(h, w)
    close(y, want, dtype, want.abs() + 1)
    xv, wg = xv.detach().requires_grad_(), w.detach().requires_grad_()
    dy = wide[1][:, 1:n + 1]
    dx, dw = torch.autograd.grad(P.rms_norm(xv, wg, 1e-6), (xv, wg), dy)
    x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
    ex, ew = torch.autograd.grad(formula(x64, w64), (x64, w64), r.double())
    # dx: a term of the row's mean besides its own; dw: a sum over the rows
    rstd = (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    g = (r.double() * w.double()).abs()
    close(dx, ex, dtype, rstd * (g + (x.double() * rstd).abs() * (g * (x.double() * rstd).abs()).mean(-1, keepdim=True)))
    close(dw, ew, torch.float32, (r.double() * x.double() * rstd).abs().sum(0))
