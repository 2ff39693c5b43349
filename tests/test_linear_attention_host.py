"""Linear attention, rotary positions and the gated norm without a GPU: struct layouts against the header,
sizes and refusals of the C entries that come before any device work, layouts that the package hands to them,
the torch statements and their gradients, and traces."""
from __future__ import annotations

import ctypes
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "amd_tuned_torch_hip.h")
P = 1 << 20  # a pointer that no refusal may follow


@pytest.fixture(scope="module")
def nat():
    from amd_tuned_torch import _native
    _native.load()
    return _native


def test_struct_layouts_match_the_header(nat, tmp_path):
    blocks = {"atk_rms_norm_gated_args": nat._GatedArgs, "atk_rotary_args": nat._RotaryArgs,
              "atk_linear_attn_update_args": nat._LinearUpdateArgs, "atk_linear_attn_args": nat._LinearArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    want = []
    for cname, cls in blocks.items():
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({cname}, {f}));')
            want.append(getattr(cls, f).offset)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-O0", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE, text=True).stdout.split()
    assert [int(x) for x in out] == want


def filled(cls, base, kw):
    a = cls()
    for name, value in {**base, **kw}.items():
        field = getattr(a, name)
        if isinstance(value, tuple):
            field[:] = value
        else:
            setattr(a, name, value)
    return a


def called(fn, a, *more):
    """fn(address of the struct, ...), which lives until the call returns."""
    return fn(ctypes.addressof(a), *more)


def test_gated_norm_refusals(nat):
    lib = nat.lib()
    base = dict(x=P, gate=P, y=P, M=2, N=64, group=32, x_stride=64, gate_stride=64, eps=1e-6, dtype=nat.ATK_BF16, w_dtype=nat.ATK_BF16)
    fwd = lambda **kw: called(lib.atk_rms_norm_gated_fwd, filled(nat._GatedArgs, base, kw))  # noqa: E731
    bwd = lambda dy=P, dx=P, dz=P, dw=None, ws=None, size=0, **kw: called(  # noqa: E731
        lib.atk_rms_norm_gated_bwd, filled(nat._GatedArgs, base, kw), dy, 64, dx, dz, dw, ws, size)
    assert lib.atk_rms_norm_gated_fwd(None) == nat.ATK_EINVAL
    for fn in (fwd, bwd):
        assert fn(M=0) == nat.ATK_OK and fn(N=0, group=0) == nat.ATK_OK
        for kw in (dict(x=None), dict(gate=None), dict(dtype=7), dict(activation=2), dict(M=-1), dict(group=24), dict(group=0),
                   dict(group=-32), dict(x_stride=63), dict(gate_stride=3), dict(weight=P, w_dtype=nat.ATK_F16)):
            assert fn(**kw) == nat.ATK_EINVAL, kw
        for kw in (dict(N=16385, group=16385, x_stride=16385, gate_stride=16385), dict(M=1 << 31),
                   dict(N=65536, group=1, x_stride=65536, gate_stride=65536),
                   dict(dtype=nat.ATK_F32, N=8193, group=8193, x_stride=8193, gate_stride=8193)):
            assert fn(**kw) == nat.ATK_UNSUPPORTED, kw
    assert fwd(y=None) == nat.ATK_EINVAL
    for kw in (dict(dy=None), dict(dx=None), dict(dz=None), dict(dw=P), dict(dw=P, weight=P), dict(dw=P, weight=P, ws=P, size=255)):
        assert bwd(**kw) == nat.ATK_EINVAL, kw
    size = lib.atk_rms_norm_gated_bwd_workspace_bytes
    assert size(0, 64, 32, 2) == 0 and size(3, 64, 24, 2) == 0 and size(3, 64, 32, 2) >= 64 * 4 and size(3, 64, 32, 2) % 256 == 0


def test_rotary_refusals(nat):
    base = dict(q=P, k=P, q_out=P, k_out=P, inv_freq=P, N=2, T=3, Hq=4, Hk=2, D=64, rot=64, dtype=nat.ATK_BF16, scale=1.0)
    call = lambda **kw: called(nat.lib().atk_rotary, filled(nat._RotaryArgs, base, kw))  # noqa: E731
    assert nat.lib().atk_rotary(None) == nat.ATK_EINVAL
    for kw in (dict(N=0), dict(T=0), dict(D=0, rot=0), dict(Hq=0, Hk=0)):
        assert call(**kw) == nat.ATK_OK, kw
    for kw in (dict(q=None), dict(k_out=None), dict(inv_freq=None), dict(dtype=3), dict(rot=63), dict(rot=66), dict(rot=-2), dict(Hq=-1)):
        assert call(**kw) == nat.ATK_EINVAL, kw
    for kw in (dict(D=4098), dict(Hq=65536), dict(N=1 << 20, T=1 << 20)):
        assert call(**kw) == nat.ATK_UNSUPPORTED, kw


def test_update_refusals(nat):
    base = dict(q=P, k=P, v=P, g=P, state=P, out=P, N=2, slots=2, Hk=2, Hv=4, K=64, V=64, dtype=nat.ATK_BF16)
    call = lambda **kw: called(nat.lib().atk_linear_attn_update, filled(nat._LinearUpdateArgs, base, kw))  # noqa: E731
    assert nat.lib().atk_linear_attn_update(None) == nat.ATK_EINVAL
    assert call(N=0) == nat.ATK_OK
    for kw in (dict(q=None), dict(state=None), dict(out=None), dict(dtype=5), dict(g_dtype=5), dict(g_dtype=nat.ATK_F16), dict(Hk=0),
               dict(Hk=3), dict(K=0), dict(V=0), dict(N=-1), dict(slots=1)):
        assert call(**kw) == nat.ATK_EINVAL, kw
    for kw in (dict(K=257), dict(Hk=65536, Hv=65536), dict(N=70000, slots=70000)):
        assert call(**kw) == nat.ATK_UNSUPPORTED, kw


def sequences(nat, fn, **kw):
    base = dict(q=P, k=P, v=P, g=P, out=P, N=2, T=1000, Hk=2, Hv=4, K=64, V=64, dtype=nat.ATK_BF16)
    return called(fn, filled(nat._LinearArgs, base, kw))


def test_sequence_refusals_and_workspaces(nat):
    lib = nat.lib()
    fwd = lib.atk_linear_attn_fwd
    bwd = lambda p: lib.atk_linear_attn_bwd(p, P, None, P, P, P, P, None)  # noqa: E731
    size, size_b = lib.atk_linear_attn_workspace_bytes, lib.atk_linear_attn_bwd_workspace_bytes
    assert size(None) == 0 and size_b(None) == 0 and fwd(None) == nat.ATK_EINVAL and bwd(None) == nat.ATK_EINVAL
    assert sequences(nat, fwd, N=0) == nat.ATK_OK and sequences(nat, fwd, T=0) == nat.ATK_OK and sequences(nat, bwd, N=0) == nat.ATK_OK
    for fn in (fwd, bwd):
        for kw in (dict(q=None), dict(g=None), dict(dtype=4), dict(g_dtype=9), dict(g_dtype=nat.ATK_F16), dict(Hk=3), dict(K=0),
                   dict(T=-1), dict(), dict(workspace=P + 8, workspace_bytes=1 << 40)):  # no workspace; an unaligned one
            assert sequences(nat, fn, **kw) == nat.ATK_EINVAL, kw
        for kw in (dict(K=257), dict(K=7), dict(V=7), dict(K=3, dtype=nat.ATK_F32, g_dtype=nat.ATK_F32), dict(T=1 << 31), dict(N=65536),
                   dict(K=256, V=1 << 21), dict(q_stride=(0, 1 << 22, 64)), dict(g_stride=(0, 1 << 22, 1)), dict(v_stride=(0, -64, 64)),
                   dict(N=60000, T=1 << 30)):
            assert sequences(nat, fn, **kw) == nat.ATK_UNSUPPORTED, kw
    # sequences of one segment need nothing between segments; the backward's dots it always needs
    assert sequences(nat, size, T=64) == 0 and sequences(nat, size, T=64, N=60000) == 0
    assert sequences(nat, size_b, T=64) >= 2 * 4 * 2 * 64 * 4
    # a state of each head and segment, and a decay
    need = sequences(nat, size, N=1, T=8192)
    assert need > 0 and need % (4 * (64 * 64 * 4 + 4)) == 0
    wide = sequences(nat, size, N=1, T=8192, V=128)    # (segments may be longer)
    assert wide > 0 and wide % (4 * (64 * 128 * 4 + 4)) == 0
    assert sequences(nat, size_b, N=1, T=8192) > 2 * need - 4096


def test_narrow_heads_are_widened(nat):
    """Heads of fewer than 16 bytes are padded with zeros, which change no sum."""
    from amd_tuned_torch.linear_attention_ops import linear_attention_ref
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    q, k, v, g, state = r(1, 9, 1, 3), r(1, 9, 1, 3), r(1, 9, 2, 5), -r(1, 9, 2).abs(), r(1, 2, 3, 5)
    want, want_s = linear_attention_ref(q, k, v, g, 0.3, state, True)
    got, got_s = linear_attention_ref(*nat._widen(8, q, k, v, None)[:3], g, 0.3, nat._widen(8, q, k, v, state)[3], True)
    assert torch.equal(got[..., :5], want) and torch.equal(got_s[:, :, :3, :5], want_s)


def test_statements_agree_on_the_cpu():
    from amd_tuned_torch import linear_attention_ops as la
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    q, k, v, g, state = r(2, 9, 2, 5), r(2, 9, 2, 5), r(2, 9, 4, 3), -r(2, 9, 4).abs(), r(2, 4, 5, 3)
    for gates in (g, g[0, 0]):
        out, final = la.linear_attention_ref(q, k, v, gates, 0.3, state, True)
        S = state.float()
        for t in range(9):
            o = la.linear_attention_update_ref(*(x[:, t] for x in (q, k, v)), gates[:, t] if gates.dim() == 3 else gates, S, 0.3)
            assert (o - out[:, t]).abs().max() <= 1e-5 * out.abs().max()
        assert (S - final).abs().max() <= 1e-5 * final.abs().max()
    out, final = la.linear_attention_ref(q, k, v, g, 0.3, state, True)
    packed = [x.flatten(0, 1)[None] for x in (q, k, v, g)]
    again, final2 = la.linear_attention_ref(*packed, 0.3, state, True, torch.tensor([0, 9, 18], dtype=torch.int32))
    assert torch.equal(again[0], out.flatten(0, 1)) and torch.equal(final2, final)
    # the formula itself, term by term
    i, j = 6, 2
    decay = g[0, j + 1:i + 1, 1].sum().exp()
    base = la.linear_attention_ref(q, k, v, g, 1.0)[0, i, 1]
    v2 = v.clone()
    v2[0, j, 1] += 1
    got = la.linear_attention_ref(q, k, v2, g, 1.0)[0, i, 1] - base
    assert (got - decay * (q[0, i, 0] * k[0, j, 0]).sum()).abs().max() < 1e-12
    leaves = [x[:1, :3].clone().requires_grad_() for x in (q, k, v, g)] + [state[:1].clone().requires_grad_()]
    assert torch.autograd.gradcheck(lambda *a: la.linear_attention_ref(*a[:4], 0.3, a[4], True), leaves)
    for bad, good in (([-5, 3, 40], [0, 3, 18]), ([2, 4, 32], [2, 4, 18]), ([21, 22], [18, 18])):
        a, b = (la.linear_attention_ref(*packed, 0.3, None, True, torch.tensor(cu, dtype=torch.int32)) for cu in (bad, good))
        assert a[0].shape == packed[2].shape and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("name", ["v from q", "q is k", "decays and state from q"])
def test_gradients_in_torch_operations_of_dependent_inputs(name):
    """The backward that is taken for a second derivative, inside autograd, against autograd of the statement:
    the same operations in 64 bits, so 1e-12 is thousands of roundings."""
    from amd_tuned_torch import linear_attention_ops as la

    class Statement(torch.autograd.Function):
        @staticmethod
        def forward(ctx, *inputs):
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(*inputs)
            return la.linear_attention_ref(*inputs[:4], 0.3, inputs[4], True)

        @staticmethod
        def backward(ctx, dout, dstate):
            return tuple(la._backward_ops(ctx.saved_tensors, 0.3, None, dout, dstate, list(ctx.needs_input_grad)))

    def inputs(leaf):
        gen = torch.Generator().manual_seed(1)
        r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
        q, k, v, g, state = leaf, r(1, 5, 2, 4), r(1, 5, 2, 4), -r(1, 5, 2).abs(), r(1, 2, 4, 4)
        if name == "v from q":
            v = 2 * q
        elif name == "q is k":
            k = q
        else:
            g, state = -q.square().sum(-1), q[:, 0, :, :, None] * k[:, 1, :, None]
        return q, k, v, g, state

    leaf = torch.randn(1, 5, 2, 4, generator=torch.Generator().manual_seed(0), dtype=torch.float64).requires_grad_()
    got = []
    for fn in (Statement.apply, lambda *a: la.linear_attention_ref(*a[:4], 0.3, a[4], True)):
        out, state = fn(*inputs(leaf))
        first, = torch.autograd.grad(out.square().sum() + state.square().sum(), leaf, create_graph=True)
        second, = torch.autograd.grad(first.pow(3).sum(), leaf)
        got.append((first.detach(), second))
    for a, b in zip(*got):
        assert (a - b).abs().max() <= 1e-12 * b.abs().max()


def test_calls_without_a_gpu_say_so(nat):
    import amd_tuned_torch as att
    x = torch.randn(2, 5, 2, 8)
    inv = torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU"):
        att.linear_attention(x, x, x, x[..., 0])
    with pytest.raises(RuntimeError, match="GPU"):
        att.linear_attention_update(x[:, 0], x[:, 0], x[:, 0], x[:, 0, :, 0], torch.zeros(2, 2, 8, 8))
    with pytest.raises(RuntimeError, match="GPU"):
        att.rotary_embedding(x, x, inv)
    with pytest.raises(RuntimeError, match="GPU"):
        att.rms_norm_gated(x, x)
    z = lambda *s: torch.zeros(s)  # noqa: E731
    for dk, dv in ((0, 4), (4, 0)):
        with pytest.raises(RuntimeError, match="no head empty"):
            att.linear_attention(z(1, 3, 1, dk), z(1, 3, 1, dk), z(1, 3, 2, dv), z(1, 3, 2))
        with pytest.raises(RuntimeError, match="no head empty"):
            att.linear_attention_update(z(1, 1, dk), z(1, 1, dk), z(1, 2, dv), z(1, 2), z(1, 2, dk, dv))


def test_decode_step_has_no_gradient_and_says_so(nat, monkeypatch):
    """With the torch statement, under no_grad as a kernel is, in the kernel's place."""
    from amd_tuned_torch import linear_attention_ops as la

    def kernel(*a):
        with torch.no_grad():
            return la.linear_attention_update_ref(*a)

    monkeypatch.setattr(nat, "linear_attn_update", kernel)
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    args = [r(2, 1, 4), r(2, 1, 4), r(2, 2, 3), -r(2, 2).abs(), r(2, 2, 4, 3)]
    plain = la.linear_attention_update(*(x.clone() for x in args))
    assert not plain.requires_grad
    for i in range(5):
        a = [x.clone().requires_grad_(j == i) for j, x in enumerate(args)]
        with torch.no_grad():
            assert not la.linear_attention_update(*(x.clone() for x in a)).requires_grad
        out = la.linear_attention_update(*a)
        assert torch.equal(out, plain)
        with pytest.raises(RuntimeError, match="no gradient"):
            out.sum().backward()
        if i < 4:
            with pytest.raises(RuntimeError):
                torch.func.jvp(lambda x: la.linear_attention_update(*args[:i], x, *args[i + 1:]), (args[i],), (args[i],))


def unrecorded(fn):
    """`fn` as a kernel is to traces: its results appear in fresh memory, by another thread."""
    def kernel(*a, **kw):
        import threading
        arrays = [x.detach().numpy() if isinstance(x, torch.Tensor) else x for x in a]
        out = []

        def work():
            with torch.no_grad():
                out.append(fn(*[torch.from_numpy(x) if hasattr(x, "ctypes") else x for x in arrays], **kw))

        thread = threading.Thread(target=work)
        thread.start()
        thread.join()
        got = out[0] if isinstance(out[0], tuple) else (out[0],)
        fresh = [None if x is None else torch.empty(x.shape, dtype=x.dtype) for x in got]
        for to, x in zip(fresh, got):
            if x is not None:
                ctypes.memmove(to.data_ptr(), x.contiguous().data_ptr(), x.numel() * x.element_size())
        return tuple(fresh) if isinstance(out[0], tuple) else fresh[0]
    return kernel


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_traces(nat, monkeypatch):
    """What torch.jit.trace records computes the operators on other inputs, of other lengths too."""
    import amd_tuned_torch as att
    la, ro, rn = att.linear_attention_ops, att.rotary_ops, att.rms_norm_ops

    def attend(q, k, v, g, scale, initial_state=None, cu_seqlens=None, want_state=False):
        out, state = la.linear_attention_ref(q, k, v, g, scale, initial_state, True, cu_seqlens)
        return out, state if want_state else None

    monkeypatch.setattr(nat, "linear_attn", unrecorded(attend))
    monkeypatch.setattr(nat, "linear_attn_update", unrecorded(la.linear_attention_update_ref))
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    seqs = lambda t: (r(1, t, 1, 4), r(1, t, 1, 4), r(1, t, 2, 3), -r(1, t, 2).abs())  # noqa: E731
    token = lambda: (r(2, 1, 4), r(2, 1, 4), r(2, 2, 3), -r(2, 2).abs(), r(2, 2, 4, 3))  # noqa: E731
    inv = torch.tensor([1.0, 0.1], dtype=torch.float64)
    turn = lambda: (r(2, 5, 2, 6), r(2, 5, 1, 6), torch.randint(0, 50, (2, 5), generator=gen))  # noqa: E731
    rows = lambda m: (r(m, 40), r(m, 40), r(40))  # noqa: E731
    cases = [(lambda *a: att.linear_attention(*a), seqs(5), seqs(7)),
             (lambda *a: att.linear_attention(*a, return_final_state=True), seqs(5), seqs(3)),
             (lambda *a: att.linear_attention_update(*a), token(), token()),
             (lambda q, k, p: att.rotary_embedding(q, k, inv, p), turn(), turn()),
             (lambda q, k, p: att.rotary_embedding(q, None, inv, p, True, 1.5), turn(), turn()),
             (lambda x, z, w: att.rms_norm_gated(x, z, w), rows(3), rows(5)),
             (lambda x, z, w: att.rms_norm_gated(x, z, w, gate_first=True, activation="sigmoid", group_size=8), rows(3), rows(5))]
    refs = {"rotary_embedding": ro.rotary_embedding_ref, "rms_norm_gated": rn.rms_norm_gated_ref}
    for i, (fn, first, other) in enumerate(cases):
        with torch.no_grad():
            traced = torch.jit.trace(fn, tuple(x.clone() for x in first), check_trace=False)
            got = traced(*(x.clone() for x in other))
            with monkeypatch.context() as m:
                for name, ref in refs.items():
                    m.setattr(att, name, ref)
                want = fn(*(x.clone() for x in other))
        for a, b in zip(*(x if isinstance(x, tuple) else (x,) for x in (got, want))):
            assert torch.equal(a, b), i


def test_launches_go_to_the_tensors_device(nat, monkeypatch):
    """Where another device is the current one, the call runs with the tensors' made current."""
    seen, current = [], [0]

    class Switch:
        def __init__(self, device):
            self.to = device.index

        def __enter__(self):
            self.back, current[0] = current[0], self.to

        def __exit__(self, *a):
            current[0] = self.back

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", Switch)
    for index in (0, 3):
        assert nat._on(torch.device("cuda", index), lambda x: seen.append((x, current[0])) or x, index) == index
    assert seen == [(0, 0), (3, 3)] and current == [0]
