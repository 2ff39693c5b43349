"""What the package does on the host for the root-mean-square norm and the gated delta rule, without a
GPU: the layouts it hands to the C entries, sizes and refusals, and gradients in torch operations."""
from __future__ import annotations

import pytest
import torch


@pytest.fixture(scope="module")
def nat():
    from amd_tuned_torch import _native
    _native.load()
    return _native


def one_long_axes():
    """Tensors with an axis of length 1, whose stride there says nothing about the rows."""
    base = torch.arange(2 * 5 * 8.0)
    return {
        "sequence first, batch of one": base[:32].view(1, 4, 8).transpose(0, 1),
        "one token, batch first": base[:32].view(1, 4, 8).transpose(0, 1).contiguous().as_strided((4, 1, 8), (8, 1, 1)),
        "one head, heads first": base.view(2, 1, 5, 8).transpose(1, 2),
        "expanded axis": base.as_strided((4, 1, 8), (8, 0, 1)),
        "one row": base.as_strided((1, 8), (3, 1)),
        "rows apart": base.view(5, 16)[:, 3:11].unsqueeze(1),
        "heads of a projection": base.view(5, 16)[:, None, :8],
        "one row of each": base.view(2, 5, 8)[:, 2:3],
        "rows of one column": base.as_strided((6, 1), (8, 5)),
        "one axis": base.as_strided((7,), (2,)),
    }


@pytest.mark.parametrize("name", list(one_long_axes()))
def test_row_strides(nat, name):
    """Rows lie where the kernels look for them, and inside the tensor's storage."""
    t = one_long_axes()[name]
    rows = nat._rows(t)
    stride, n = nat._row_stride(rows), t.shape[-1]
    m = t.numel() // n
    held = rows.untyped_storage().nbytes() // 4
    assert rows.storage_offset() + (m - 1) * stride + n <= held
    flat = torch.empty(0).set_(rows.untyped_storage(), 0, (held,), (1,))
    seen = torch.stack([flat[rows.storage_offset() + i * stride:][:n] for i in range(m)])
    assert torch.equal(seen, t.reshape(m, n))


def dependent_inputs(name, leaf):
    """(q, k, v, g, beta, state) in 64 bits, computed from one leaf in part."""
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    q, k, v, g, beta, state = leaf, r(1, 5, 2, 4), r(1, 5, 2, 4), -r(1, 5, 2).abs(), r(1, 5, 2).sigmoid(), r(1, 2, 4, 4)
    if name == "v from q":
        v = 2 * q
    elif name == "q is k":
        k = q
    elif name == "gates and state from q":
        g, beta, state = -q.square().sum(-1), q.sum(-1).sigmoid(), q[:, 0, :, :, None] * k[:, 1, :, None]
    return q, k, v, g, beta, state


def statement(gd):
    """The operator as an autograd function whose backward is the one in torch operations."""
    class Statement(torch.autograd.Function):
        @staticmethod
        def forward(ctx, *inputs):
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(*inputs)
            return gd.gated_delta_rule_ref(*inputs[:5], 0.3, inputs[5], True)

        @staticmethod
        def backward(ctx, dout, dstate):
            return tuple(gd._backward_ops(ctx.saved_tensors, 0.3, None, dout, dstate, list(ctx.needs_input_grad)))
    return Statement


@pytest.mark.parametrize("name", ["v from q", "q is k", "gates and state from q"])
def test_gradients_in_torch_operations_of_dependent_inputs(name):
    """The backward that is taken for a second derivative, inside autograd, against autograd of the
    statement itself: both are the same operations in 64 bits, so 1e-12 is thousands of roundings."""
    from amd_tuned_torch import gated_delta as gd
    leaf = torch.randn(1, 5, 2, 4, generator=torch.Generator().manual_seed(0), dtype=torch.float64).requires_grad_()
    got = []
    for fn in (statement(gd).apply, lambda *a: gd.gated_delta_rule_ref(*a[:5], 0.3, a[5], True)):
        out, state = fn(*dependent_inputs(name, leaf))
        first, = torch.autograd.grad(out.square().sum() + state.square().sum(), leaf, create_graph=True)
        second, = torch.autograd.grad(first.pow(3).sum(), leaf)
        got.append((first.detach(), second))
    for a, b in zip(*got):
        assert (a - b).abs().max() <= 1e-12 * b.abs().max()


def test_gradients_in_torch_operations_of_q_alone():
    """The final state takes no part of q: asked for its gradient, the backward has zeros, or nothing."""
    from amd_tuned_torch import gated_delta as gd
    leaf = torch.randn(1, 5, 2, 4, generator=torch.Generator().manual_seed(0), dtype=torch.float64).requires_grad_()
    inputs = dependent_inputs("apart", leaf)
    out, state = statement(gd).apply(*inputs)
    got, = torch.autograd.grad(out.square().sum() + state.square().sum(), leaf, create_graph=True)
    want, = torch.autograd.grad(gd.gated_delta_rule_ref(*inputs[:5], 0.3, inputs[5]).square().sum(), leaf)
    assert (got - want).abs().max() <= 1e-12 * want.abs().max()
    out, state = statement(gd).apply(*inputs)
    assert torch.autograd.grad(state.square().sum(), leaf, create_graph=True, allow_unused=True)[0] is None


class OnDevice:
    """A CPU tensor that says it is on the GPU: for the checks, which look at sizes and strides alone."""

    def __init__(self, t):
        self.t, self.is_cuda, self.device = t, True, torch.device("cuda", 0)

    def __getattr__(self, name):
        return getattr(self.t, name)

    def __getitem__(self, at):
        return OnDevice(self.t[at])


def test_states_with_an_axis_of_one(nat):
    """Slots that are contiguous pass, whatever strides their axes of length 1 state; others do not."""
    def check(state, n=2):
        hv, dk, dv = state.shape[1:]
        r = lambda *s: OnDevice(torch.zeros(s))  # noqa: E731
        nat._delta_update_check(r(n, 1, dk), r(n, 1, dk), r(n, hv, dv), r(n, hv), r(n, hv), OnDevice(state),
                                OnDevice(torch.zeros(n, dtype=torch.int32)))

    base = torch.zeros(4096)
    for state in (base[:768].view(3, 4, 8, 8).contiguous(), base[:192].view(1, 3, 8, 8).transpose(0, 1),  # one head
                  base.view(8, 8, 8, 8)[:, 2:3], base.as_strided((3, 1, 8, 8), (64, 5, 8, 1)),
                  base.as_strided((3, 2, 1, 8), (16, 8, 3, 1)), base.as_strided((3, 2, 8, 1), (16, 8, 1, 9)),
                  base.as_strided((1, 2, 8, 8), (7, 64, 8, 1)), base.view(2, 2, 4, 16, 16)[:, 1]):
        check(state)
    for state in (base.view(1, 8, 8, 64)[..., :8], base[:256].view(2, 2, 8, 8).transpose(2, 3),
                  base.view(8, 8, 8, 8).transpose(1, 2), base.as_strided((3, 1, 8, 8), (32, 64, 8, 1)),
                  base.as_strided((3, 2, 8, 8), (0, 64, 8, 1))):
        with pytest.raises(RuntimeError, match="contiguous"):
            check(state)


P = 1 << 20  # a pointer that no refusal may follow


def sequences(nat, fn, **kw):
    import ctypes
    a = nat._DeltaArgs()
    for f in ("q", "k", "v", "g", "beta", "out"):
        setattr(a, f, P)
    a.N, a.T, a.Hk, a.Hv, a.K, a.V, a.dtype = 2, 100, 2, 4, 64, 64, nat.ATK_BF16
    for name, value in kw.items():
        setattr(a, name, value)
    return fn(ctypes.addressof(a))


def test_gates_of_a_type_that_the_kernels_do_not_read(nat):
    import ctypes
    lib = nat.lib()
    bwd = lambda p: lib.atk_gated_delta_bwd(p, P, None, P, P, P, P, P, None)  # noqa: E731
    pairs = [(nat.ATK_BF16, nat.ATK_F16), (nat.ATK_F16, nat.ATK_BF16), (nat.ATK_F32, nat.ATK_F16),
             (nat.ATK_F32, nat.ATK_BF16)]
    for dtype, gate in pairs:
        for name, other in (("g_dtype", "beta_dtype"), ("beta_dtype", "g_dtype")):
            kw = {"dtype": dtype, name: gate, other: dtype}
            for size in (lib.atk_gated_delta_workspace_bytes, lib.atk_gated_delta_bwd_workspace_bytes):
                assert sequences(nat, size, **kw) == 0, kw
            for fn in (lib.atk_gated_delta_fwd, bwd):
                assert sequences(nat, fn, workspace=P, workspace_bytes=1 << 40, **kw) == nat.ATK_EINVAL, kw
            a = nat._DeltaUpdateArgs()
            for f in ("q", "k", "v", "g", "beta", "state", "out"):
                setattr(a, f, P)
            a.N, a.slots, a.Hk, a.Hv, a.K, a.V = 2, 2, 2, 4, 64, 64
            for f, value in kw.items():
                setattr(a, f, value)
            assert lib.atk_gated_delta_update(ctypes.addressof(a)) == nat.ATK_EINVAL, kw


def test_short_calls_need_no_workspace(nat):
    """Ten tokens go one after the other with the state in registers; the backward has chunks all the same."""
    lib = nat.lib()
    size, size_b = lib.atk_gated_delta_workspace_bytes, lib.atk_gated_delta_bwd_workspace_bytes
    for n in (1, 1024):
        for t in (0, 1, 10):
            assert sequences(nat, size, N=n, T=t) == 0
            assert sequences(nat, size, N=n, T=t, cu_seqlens=P) == 0
        assert sequences(nat, size, N=n, T=11) > 0 and sequences(nat, size_b, N=n, T=10) > 0


def test_states_that_32_bits_cannot_index(nat):
    lib = nat.lib()
    bwd = lambda p: lib.atk_gated_delta_bwd(p, P, None, P, P, P, P, P, None)  # noqa: E731
    size, size_b = lib.atk_gated_delta_workspace_bytes, lib.atk_gated_delta_bwd_workspace_bytes
    for k, v in ((129, 1 << 23), (256, (1 << 23) - 31), (128, 1 << 24)):
        kw = dict(N=1, Hk=1, Hv=1, K=k, V=v, workspace=P, workspace_bytes=1 << 60)
        assert sequences(nat, bwd, **kw) == nat.ATK_UNSUPPORTED and sequences(nat, size_b, **kw) == 0
        assert sequences(nat, size, **kw) > 0    # the forward has no such index
    for k, v in ((256, (1 << 23) - 32), (64, 1 << 24)):
        assert sequences(nat, size_b, N=1, Hk=1, Hv=1, K=k, V=v) > 0


def test_many_sequences_in_one_long_row(nat):
    """A packed row has a chunk for each 64 tokens and one a sequence, not the row's for every sequence."""
    size = nat.lib().atk_gated_delta_workspace_bytes
    chunk = sequences(nat, size, N=2, T=64) - sequences(nat, size, N=1, T=64)
    base = sequences(nat, size, N=1, T=64) - chunk
    for n, t in ((40000, 1 << 22), (65535, (1 << 31) - 128)):
        assert sequences(nat, size, N=n, T=t, cu_seqlens=P) == base + chunk * (t // 64 + n)
    assert sequences(nat, nat.lib().atk_gated_delta_fwd, N=40000, T=1 << 22) == nat.ATK_UNSUPPORTED


def test_statement_clamps_offsets():
    """As the kernels do: what offsets beyond the row leave of it, in the result and the gradients."""
    from amd_tuned_torch import gated_delta as gd
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    args = r(1, 9, 1, 4), r(1, 9, 1, 4), r(1, 9, 2, 3), -r(1, 9, 2).abs(), r(1, 9, 2).sigmoid()
    for bad, good in (([-5, 3, 40], [0, 3, 9]), ([2, 4, 12], [2, 4, 9]), ([11, 12], [9, 9])):
        got, want = (gd.gated_delta_rule_ref(*args, 0.3, None, True, torch.tensor(cu, dtype=torch.int32)) for cu in (bad, good))
        assert got[0].shape == args[2].shape and all(torch.equal(a, b) for a, b in zip(got, want))


def test_decode_step_has_no_gradient_and_says_so(nat, monkeypatch):
    """With the torch statement, under no_grad as a kernel is, in the kernel's place."""
    from amd_tuned_torch import gated_delta as gd

    def kernel(*a):
        with torch.no_grad():
            return gd.gated_delta_rule_update_ref(*a)

    monkeypatch.setattr(nat, "gated_delta_update", kernel)
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    args = [r(2, 1, 4), r(2, 1, 4), r(2, 2, 3), -r(2, 2).abs(), r(2, 2).sigmoid(), r(2, 2, 4, 3)]
    plain = gd.gated_delta_rule_update(*(x.clone() for x in args))
    assert not plain.requires_grad
    for i in range(6):
        a = [x.clone() for x in args]
        with torch.no_grad():
            assert not gd.gated_delta_rule_update(*a[:i], a[i].requires_grad_(), *a[i + 1:]).requires_grad
        a = [x.clone().requires_grad_(j == i) for j, x in enumerate(args)]
        out = gd.gated_delta_rule_update(*a)
        assert torch.equal(out, plain)
        with pytest.raises(RuntimeError, match="no gradient"):
            out.sum().backward()
    for i in range(5):
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda x: gd.gated_delta_rule_update(*args[:i], x, *args[i + 1:]), (args[i],), (args[i],))
        with pytest.raises(RuntimeError):
            with torch.autograd.forward_ad.dual_level():
                a = list(args)
                a[i] = torch.autograd.forward_ad.make_dual(a[i], a[i])
                gd.gated_delta_rule_update(*a)


def unrecorded(fn):
    """`fn` as a kernel is to autograd and to traces: its results appear in fresh memory."""
    def kernel(*a, **kw):
        arrays = [x.detach().numpy() if isinstance(x, torch.Tensor) else x for x in a]
        out = []

        def work():
            with torch.no_grad():
                out.append(fn(*[torch.from_numpy(x) if hasattr(x, "ctypes") else x for x in arrays], **kw))

        import threading
        thread = threading.Thread(target=work)     # (a trace records its own thread)
        thread.start()
        thread.join()
        got = out[0] if isinstance(out[0], tuple) else (out[0],)
        fresh = [None if x is None else torch.empty(x.shape, dtype=x.dtype) for x in got]
        for to, x in zip(fresh, got):
            if x is not None:
                import ctypes
                ctypes.memmove(to.data_ptr(), x.contiguous().data_ptr(), x.numel() * x.element_size())
        return tuple(fresh) if isinstance(out[0], tuple) else fresh[0]
    return kernel


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_traces(nat, monkeypatch):
    """What torch.jit.trace records computes the operators on other inputs, of other lengths too."""
    import amd_tuned_torch as att
    from amd_tuned_torch import gated_delta as gd

    def rule(q, k, v, g, beta, scale, initial_state=None, cu_seqlens=None, want_state=False):
        out, state = gd.gated_delta_rule_ref(q, k, v, g, beta, scale, initial_state, True, cu_seqlens)
        return out, state if want_state else None

    monkeypatch.setattr(nat, "gated_delta", unrecorded(rule))
    monkeypatch.setattr(nat, "gated_delta_update", unrecorded(gd.gated_delta_rule_update_ref))
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    seqs = lambda t: (r(1, t, 1, 4), r(1, t, 1, 4), r(1, t, 2, 3), -r(1, t, 2).abs(), r(1, t, 2).sigmoid())  # noqa: E731
    token = lambda: (r(2, 1, 4), r(2, 1, 4), r(2, 2, 3), -r(2, 2).abs(), r(2, 2).sigmoid(), r(2, 2, 4, 3))  # noqa: E731
    rows = lambda m: (r(m, 40), r(40), r(m, 40))  # noqa: E731
    cases = [(lambda *a: att.gated_delta_rule(*a), seqs(5), seqs(7)),
             (lambda *a: att.gated_delta_rule(*a, return_final_state=True), seqs(5), seqs(3)),
             (lambda *a: att.gated_delta_rule_update(*a), token(), token()),
             (lambda x, w, h: att.rms_norm(x, w, residual=h), rows(3), rows(5)),
             (lambda x, w, h: att.rms_norm(x, w), rows(3), rows(5)),
             (lambda x, w, h: att.rms_norm_quant(x, w, residual=h), rows(3), rows(5)),
             (lambda x, w, h: att.rms_norm_quant(x, w, dtype=torch.int8, group_size=16), rows(3), rows(5))]
    refs = {"rms_norm": att.rms_norm_ops.rms_norm_ref, "rms_norm_quant": att.rms_norm_ops.rms_norm_quant_ref}
    for i, (fn, first, other) in enumerate(cases):
        with torch.no_grad():
            traced = torch.jit.trace(fn, tuple(x.clone() for x in first), check_trace=False)
            got = traced(*(x.clone() for x in other))
            with monkeypatch.context() as m:
                for name, ref in refs.items():
                    m.setattr(att, name, ref)
                want = fn(*(x.clone() for x in other))
        for a, b in zip(*(x if isinstance(x, tuple) else (x,) for x in (got, want))):
            assert torch.equal(a.float(), b.float()), i


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("n,group", [(0, None), (1, None), (40, None), (40, 16), (64, 32), (7, 16)])
def test_statement_in_8_bits(n, group, out):
    """Half a step of int8 or of fp8's 3 bits, and the scales of the definition; a NaN spoils its run."""
    from amd_tuned_torch.rms_norm_ops import rms_norm_quant_ref
    gen = torch.Generator().manual_seed(n)
    x, w, res = (torch.randn(*s, generator=gen) for s in ((3, n), (n,), (3, n)))
    top = 448.0 if out == torch.float8_e4m3fn else 127.0
    q, s, h = rms_norm_quant_ref(x, w, 1e-6, res, out, group)
    assert torch.equal(h, x + res) and q.dtype == out and q.shape == x.shape
    assert s.shape == (3, -(-n // group) if group else 1)
    y = h.double() / (h.double().square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    wide = (s.repeat_interleave(group, -1)[:, :n] if group else s).double()
    if n:
        v = y / wide
        half = 0.5 if out == torch.int8 else torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10))
        assert ((q.double() - v).abs() <= half + 1e-4).all() and q.float().abs().max() <= top
        x[1, 0] = float("nan")
        q, s = rms_norm_quant_ref(x, w, 1e-6, None, out, group)
        assert s[1].isnan().all() and s[[0, 2]].isfinite().all()
    else:
        assert s.eq(2.0 ** -126).all()


def test_heads_without_columns_are_refused(nat):
    """By the operators' own checks, with the default scale too."""
    import amd_tuned_torch as att
    z = lambda *s: torch.zeros(s)  # noqa: E731
    for dk, dv in ((0, 4), (4, 0)):
        with pytest.raises(RuntimeError, match="no head empty"):
            att.gated_delta_rule(z(1, 3, 1, dk), z(1, 3, 1, dk), z(1, 3, 2, dv), z(1, 3, 2), z(1, 3, 2))
        with pytest.raises(RuntimeError, match="no head empty"):
            att.gated_delta_rule_update(z(1, 1, dk), z(1, 1, dk), z(1, 2, dv), z(1, 2), z(1, 2), z(1, 2, dk, dv))
