"""The root-mean-square norm and the gated delta rule where layouts, values and callers are unusual.

Where a call only differs from another in its layout, the same kernel runs on the same numbers, so the
results have equal bits.  Other tolerances stand at their tests."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def turned(dev, dtype, n, seed):
    """Layouts with an axis of length 1 and a stride there that is not the rows'."""
    x = torch.randn(12 * n, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)
    return [x.view(1, 12, n).transpose(0, 1), x.view(3, 1, 4, n).transpose(1, 2),
            x.as_strided((12, 1, n), (n, 0, 1)), x.as_strided((12, 1, n), (n, 1, 1))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [8, 128, 130])
def test_rms_norm_of_axes_of_one(dev, n, dtype):
    """x, residual, dy and dh in such layouts, each against the same rows in a dense matrix."""
    import amd_tuned_torch as P
    w = (1 + 0.3 * torch.randn(n, generator=torch.Generator().manual_seed(9))).to(dtype).to(dev)
    for x, r, dy, dh in zip(*(turned(dev, dtype, n, i) for i in range(4))):
        X, R, DY, DH = (t.reshape(12, n).clone() for t in (x, r, dy, dh))
        assert torch.equal(P.rms_norm(x, w).reshape(12, n), P.rms_norm(X, w))
        for got, want in zip(P.rms_norm(x, w, residual=r), P.rms_norm(X, w, residual=R)):
            assert got.shape == x.shape and torch.equal(got.reshape(12, n), want)
        assert torch.equal(P.rms_norm(X, w, residual=R)[1], (X.float() + R.float()).to(dtype))
        for got, want in zip(P.rms_norm_quant(x, w, residual=r, dtype=torch.int8),
                             P.rms_norm_quant(X, w, residual=R, dtype=torch.int8)):
            assert torch.equal(got.flatten(0, -2), want)
        grads = []
        for a, b, c, d in ((x, r, dy, dh), (X, R, DY, DH)):
            leaves = [t.detach().requires_grad_() for t in (a, b, w)]
            y, h = P.rms_norm(leaves[0], leaves[2], residual=leaves[1])
            grads.append(torch.autograd.grad((y, h), leaves, (c, d)))
            grads[-1] += torch.autograd.grad(P.rms_norm(leaves[0], leaves[2]), (leaves[0], leaves[2]), c)  # h is x itself
        for got, want in zip(*grads):
            assert torch.equal(got.reshape(want.shape), want)


def test_weight_gradients_of_graphs_that_run_side_by_side(dev):
    """Two captured backward passes, replayed on two streams at once: each has scratch of its own."""
    import amd_tuned_torch as P
    from amd_tuned_torch import _native
    before = set(_native.workspace_keys())
    sets, graphs = [], []
    for seed in (0, 1):
        gen = torch.Generator().manual_seed(seed)
        x, dy = (torch.randn(4096, 512, generator=gen).bfloat16().to(dev) for _ in range(2))
        w = torch.ones(512, dtype=torch.bfloat16, device=dev)
        _, _, rstd, _ = _native.rms_norm(x, w, 1e-6, want_rstd=True)
        want = _native.rms_norm_backward(x, dy, None, w, rstd)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _native.rms_norm_backward(x, dy, None, w, rstd)
        sets.append((got, want, (x, dy, w, rstd)))  # (a graph reads its inputs where they were)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for got, _, _ in sets:
            for t in got:
                t.zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for got, want, _ in sets:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not [k for k in set(_native.workspace_keys()) - before if "rms" in k[2]]


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [5, 100, 200, 1021, 2048, 4100, 20000])
def test_eight_bits_keep_nan(dev, n, dtype, out):
    """A scale is NaN where its row or group holds one, and there alone, so the values it stands for are."""
    import amd_tuned_torch as P
    x = torch.randn(6, n, generator=torch.Generator().manual_seed(n)).to(dtype).to(dev)
    x[1, n // 2] = float("nan")
    x[3, n - 1] = float("inf")        # the row's own value is inf / inf, the others are 0
    x[4] = 0
    w = torch.ones(n, dtype=dtype, device=dev)
    spoilt = w.clone()
    spoilt[n // 3] = float("nan")     # a column of every row
    for weight in (None, w, spoilt):
        for group in (None, 16, 64, 256):
            q, s = P.rms_norm_quant(x, weight, 1e-6, dtype=out, group_size=group)
            h = x.double()
            y = h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * (1 if weight is None else weight.double())
            width = group or n
            bad = torch.stack([y[:, a:a + width].isnan().any(-1) for a in range(0, n, width)], -1)
            assert torch.equal(s.isnan(), bad) and (s[~bad] >= 2.0 ** -126).all() and s[~bad].isfinite().all()
            wide = s.repeat_interleave(width, -1)[:, :n] if group else s
            assert torch.equal((q.float() * wide).isnan(), bad.repeat_interleave(width, -1)[:, :n])
            assert q[4].float()[~bad.repeat_interleave(width, -1)[4, :n]].eq(0).all()


def test_eight_bits_of_no_columns(dev):
    import amd_tuned_torch as P
    torch.full((4096,), float("nan"), device=dev)  # what a fresh tensor may hold
    q, s = P.rms_norm_quant(torch.empty(4096, 0, device=dev))
    assert q.shape == (4096, 0) and s.shape == (4096, 1) and s.eq(2.0 ** -126).all()
    q, s, h = P.rms_norm_quant(torch.empty(3, 0, device=dev), residual=torch.empty(3, 0, device=dev), group_size=32)
    assert s.shape == (3, 0) and h.shape == (3, 0)


@pytest.mark.parametrize("m,n", [((1 << 26) + 3, 130), ((1 << 28) + 5, 12)])
def test_rows_beyond_2_to_the_32_threads(dev, m, n):
    """More rows than one launch has threads for: the rows around the seam and at the ends, against the
    same rows alone."""
    import amd_tuned_torch as P
    if torch.cuda.mem_get_info(dev)[0] < 5 * m * n * 2:
        pytest.skip("not enough memory")
    x = torch.empty(m, n, dtype=torch.bfloat16, device=dev)
    part = torch.randn(1 << 20, n, device=dev).bfloat16()
    for at in range(0, m, 1 << 20):
        x[at:at + (1 << 20)] = part[:m - at]
        part = part.roll(1, 0)
    seam = 1 << 25 if n > 128 else 1 << 27
    y = P.rms_norm(x)
    for rows in (slice(0, 9), slice(seam - 9, seam + 9), slice(2 * seam - 9, 2 * seam + 2), slice(m - 3, m)):
        assert torch.equal(y[rows], P.rms_norm(x[rows])), rows
    del y
    q, s, h = P.rms_norm_quant(x, residual=x, dtype=torch.int8)
    for rows in (slice(seam - 9, seam + 9), slice(m - 3, m)):
        for got, want in zip((q, s, h), P.rms_norm_quant(x[rows], residual=x[rows], dtype=torch.int8)):
            assert torch.equal(got[rows], want), rows
    del x, q, s, h, got
    torch.cuda.empty_cache()


def test_update_of_one_head(dev):
    """A cache of one value head that was laid out heads first: equal bits to the same states copied."""
    import amd_tuned_torch as P
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
    q, k, v, g, beta = r(3, 1, 64) / 8, r(3, 1, 64) / 8, r(3, 1, 36), -r(3, 1).abs(), r(3, 1).sigmoid()
    state = r(1, 5, 64, 36).transpose(0, 1)
    copy = state.reshape(5, 64 * 36).clone().view(5, 1, 64, 36)
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device=dev)
    got, want = (P.gated_delta_rule_update(q, k, v, g, beta, s, state_indices=slots) for s in (state, copy))
    assert torch.equal(got, want) and torch.equal(state, copy)


@pytest.mark.parametrize("n,hv,gradients", [(64, 64, False), (64, 34, True)])
def test_chains_beyond_one_launch(dev, n, hv, gradients):
    """More heads, sequences and value tiles than one launch has threads for.  A value column depends on no
    other, so columns from here and there have equal bits to a call on them alone."""
    import amd_tuned_torch as P
    t, dk, dv = 11, 16, 32768
    if torch.cuda.mem_get_info(dev)[0] < (200 << 30):
        pytest.skip("not enough memory")
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, k = (torch.nn.functional.normalize(r(n, t, 1, dk), dim=-1).bfloat16().to(dev) for _ in range(2))
    g, beta = -r(n, t, hv).abs().to(dev), r(n, t, hv).sigmoid().bfloat16().to(dev)
    v = torch.empty(n, t, hv, dv, dtype=torch.bfloat16, device=dev)
    for i in range(n):
        v[i].normal_(generator=torch.Generator(device=dev).manual_seed(i))
    parts = [slice(0, 64), slice(16384, 16448), slice(dv - 64, dv)]
    if not gradients:
        out = P.gated_delta_rule(q, k, v, g, beta)
        for at in parts:
            assert torch.equal(out[..., at], P.gated_delta_rule(q, k, v[..., at], g, beta)), at
    else:
        dout = torch.empty_like(v)
        for i in range(n):
            dout[i].normal_(generator=torch.Generator(device=dev).manual_seed(n + i))
        v.requires_grad_()
        dv_all, = torch.autograd.grad(P.gated_delta_rule(q, k, v, g, beta), v, dout)
        for at in parts:
            some = v.detach()[..., at].clone().requires_grad_()
            want, = torch.autograd.grad(P.gated_delta_rule(q, k, some, g, beta), some, dout[..., at])
            assert torch.equal(dv_all[..., at], want), at
        del dout, dv_all
    del v
    torch.cuda.empty_cache()


def programs(dev):
    """(operator, inputs, other inputs), the others of another length."""
    import amd_tuned_torch as P
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
    seqs = lambda t: (r(1, t, 1, 32) / 6, r(1, t, 1, 32) / 6, r(1, t, 2, 36), -r(1, t, 2).abs(), r(1, t, 2).sigmoid())  # noqa: E731
    token = lambda: (r(2, 1, 32) / 6, r(2, 1, 32) / 6, r(2, 2, 36), -r(2, 2).abs(), r(2, 2).sigmoid(), r(2, 2, 32, 36))  # noqa: E731
    rows = lambda m: (r(m, 140), r(140), r(m, 140))  # noqa: E731
    return [(lambda *a: P.gated_delta_rule(*a), seqs(70), seqs(133)),
            (lambda *a: P.gated_delta_rule(*a, return_final_state=True), seqs(5), seqs(80)),
            (lambda *a: P.gated_delta_rule_update(*a), token(), token()),
            (lambda x, w, h: P.rms_norm(x, w, residual=h), rows(3), rows(5)),
            (lambda x, w, h: P.rms_norm(x, w), rows(3), rows(5)),
            (lambda x, w, h: P.rms_norm_quant(x, w, residual=h, dtype=torch.int8), rows(3), rows(5))]


def check_program(fn, recorded, inputs):
    """Outputs, and the state that a step overwrites, as the call's own: fp32 sums in another order at most,
    64 roundings of 2^-24 of the largest value; 8-bit values a step apart at most."""
    with torch.no_grad():
        a, b = [x.clone() for x in inputs], [x.clone() for x in inputs]
        want, got = fn(*a), recorded(*b)
    want, got = (list(x) if isinstance(x, tuple) else [x] for x in (want, got))
    for x, y in zip(got + b, want + a):
        assert x.dtype == y.dtype and x.shape == y.shape
        off = (x.double() - y.double()).abs().max()
        assert off <= (1 if x.dtype == torch.int8 else 64 * 2.0 ** -24 * y.double().abs().max())


def test_traces_on_the_device(dev):
    for fn, first, other in programs(dev):
        with torch.no_grad():
            traced = torch.jit.trace(fn, tuple(x.clone() for x in first), check_trace=False)
        check_program(fn, traced, first)
        check_program(fn, traced, other)


def test_compiled_functions(dev):
    """Inside torch.compile the operators run as they are, between graphs."""
    for fn, first, other in programs(dev):
        torch._dynamo.reset()
        compiled = torch.compile(lambda *a, fn=fn: fn(*[x + 0 for x in a[:5]], *a[5:]), backend="eager")
        check_program(fn, compiled, first)
        check_program(fn, compiled, other)
    torch._dynamo.reset()
