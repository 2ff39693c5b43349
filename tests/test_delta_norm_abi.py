"""The C entries of the gated delta rule and the root-mean-square norm without a GPU: struct layouts
against the header, sizes, and refusals that come before any device work; and the torch statements of
the rule on the CPU."""
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
    blocks = {"atk_rms_norm_args": nat._RmsArgs, "atk_gated_delta_update_args": nat._DeltaUpdateArgs,
              "atk_gated_delta_args": nat._DeltaArgs}
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


def rms(nat, **kw):
    a = nat._RmsArgs(P, None, None, P, None, None, None, 2, 64, 64, 0, 0, 1e-6, nat.ATK_BF16, nat.ATK_BF16, 0, None)
    for name, value in kw.items():
        setattr(a, name, value)
    return nat.lib().atk_rms_norm_fwd(ctypes.addressof(a))


def test_rms_norm_refusals(nat):
    assert nat.lib().atk_rms_norm_fwd(None) == nat.ATK_EINVAL
    assert rms(nat, M=0) == nat.ATK_OK and rms(nat, N=0, x_stride=0) == nat.ATK_OK
    for kw in (dict(x=None), dict(y=None), dict(dtype=7), dict(quant=3), dict(M=-1), dict(x_stride=63), dict(residual=P),
               dict(quant=1), dict(quant=1, scales=P, group=24), dict(quant=2, scales=P, group=512),
               dict(weight=P, w_dtype=nat.ATK_F16), dict(residual=P, h=P, residual_stride=3)):
        assert rms(nat, **kw) == nat.ATK_EINVAL, kw
    assert rms(nat, N=65537, x_stride=65537) == nat.ATK_UNSUPPORTED
    assert rms(nat, N=32769, x_stride=32769, dtype=nat.ATK_F32, w_dtype=nat.ATK_F32) == nat.ATK_UNSUPPORTED
    lib = nat.lib()
    assert lib.atk_rms_norm_bwd_workspace_bytes(0, 64, 2) == 0
    assert lib.atk_rms_norm_bwd_workspace_bytes(3, 64, 2) % (64 * 4) == 0
    bwd = lambda *a: lib.atk_rms_norm_bwd(*a)  # noqa: E731
    ok = [P, P, None, P, P, P, None, 2, 64, 64, 64, 0, nat.ATK_BF16, nat.ATK_BF16, None, 0, None]
    for i, value in ((0, None), (1, None), (4, None), (5, None), (9, 3), (12, 9), (6, P)):  # dw without scratch
        a = list(ok)
        a[i] = value
        assert bwd(*a) == nat.ATK_EINVAL, i
    a = list(ok)
    a[7] = 0
    assert bwd(*a) == nat.ATK_OK


def update(nat, **kw):
    a = nat._DeltaUpdateArgs()
    for f in ("q", "k", "v", "g", "beta", "state", "out"):
        setattr(a, f, P)
    a.N, a.slots, a.Hk, a.Hv, a.K, a.V, a.dtype = 2, 2, 2, 4, 64, 64, nat.ATK_BF16
    for name, value in kw.items():
        setattr(a, name, value)
    return nat.lib().atk_gated_delta_update(ctypes.addressof(a))


def test_update_refusals(nat):
    assert nat.lib().atk_gated_delta_update(None) == nat.ATK_EINVAL
    assert update(nat, N=0) == nat.ATK_OK
    for kw in (dict(q=None), dict(state=None), dict(out=None), dict(dtype=5), dict(g_dtype=5), dict(Hk=0), dict(Hk=3),
               dict(K=0), dict(V=0), dict(N=-1), dict(slots=1)):
        assert update(nat, **kw) == nat.ATK_EINVAL, kw
    for kw in (dict(K=257), dict(Hk=65536, Hv=65536), dict(N=70000, slots=70000)):
        assert update(nat, **kw) == nat.ATK_UNSUPPORTED, kw


def sequences(nat, fn, **kw):
    a = nat._DeltaArgs()
    for f in ("q", "k", "v", "g", "beta", "out"):
        setattr(a, f, P)
    a.N, a.T, a.Hk, a.Hv, a.K, a.V, a.dtype = 2, 100, 2, 4, 64, 64, nat.ATK_BF16
    for name, value in kw.items():
        setattr(a, name, value)
    return fn(ctypes.addressof(a))


def test_sequence_refusals_and_workspaces(nat):
    lib = nat.lib()
    fwd = lib.atk_gated_delta_fwd
    bwd = lambda p: lib.atk_gated_delta_bwd(p, P, None, P, P, P, P, P, None)  # noqa: E731
    size, size_b = lib.atk_gated_delta_workspace_bytes, lib.atk_gated_delta_bwd_workspace_bytes
    assert size(None) == 0 and size_b(None) == 0 and fwd(None) == nat.ATK_EINVAL
    assert sequences(nat, fwd, N=0) == nat.ATK_OK and sequences(nat, fwd, T=0) == nat.ATK_OK
    assert sequences(nat, bwd, N=0) == nat.ATK_OK
    for fn in (fwd, bwd):
        for kw in (dict(q=None), dict(beta=None), dict(dtype=4), dict(beta_dtype=9), dict(Hk=3), dict(K=0), dict(T=-1),
                   dict(), dict(workspace=P + 8, workspace_bytes=1 << 40)):  # no workspace; an unaligned one
            assert sequences(nat, fn, **kw) == nat.ATK_EINVAL, kw
        for kw in (dict(K=257), dict(T=1 << 31), dict(N=60000, T=1 << 30)):
            assert sequences(nat, fn, **kw) == nat.ATK_UNSUPPORTED, kw
    assert lib.atk_gated_delta_bwd(None, P, None, P, P, P, P, P, None) == nat.ATK_EINVAL
    # a chunk's share: 16 more chunks of each head add 16 times the same, a packed row has one a sequence more
    one, many = sequences(nat, size, N=1, T=64), sequences(nat, size, N=1, T=64 * 17)
    assert one > 0 and many > one and (many - one) % 16 == 0
    assert sequences(nat, size, N=3, T=128, cu_seqlens=P) == sequences(nat, size, N=1, T=64 * 5)
    assert sequences(nat, size_b, N=1, T=64) > 2 * 4 * 64 * 64 * 4      # the states and their gradients


def test_torch_statements_agree_on_the_cpu():
    from amd_tuned_torch import gated_delta as gd
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    q, k, v, g, beta = r(2, 9, 2, 5), r(2, 9, 2, 5), r(2, 9, 4, 3), -r(2, 9, 4).abs(), r(2, 9, 4).sigmoid()
    state = r(2, 4, 5, 3)
    out, final = gd.gated_delta_rule_ref(q, k, v, g, beta, 0.3, state, True)
    S = state.float()
    for t in range(9):
        o = gd.gated_delta_rule_update_ref(*(x[:, t] for x in (q, k, v, g, beta)), S, 0.3)
        assert (o - out[:, t]).abs().max() <= 1e-5 * out.abs().max()
    assert (S - final).abs().max() <= 1e-5 * final.abs().max()
    packed = [x.flatten(0, 1)[None] for x in (q, k, v, g, beta)]
    cu = torch.tensor([0, 9, 18], dtype=torch.int32)
    again, final2 = gd.gated_delta_rule_ref(*packed, 0.3, state, True, cu)
    assert torch.equal(again[0], out.flatten(0, 1)) and torch.equal(final2, final)
    # the gradient of the statement against differences, in 64 bits
    leaves = [x.clone().requires_grad_() for x in (q, k, v, g, beta, state)]
    assert torch.autograd.gradcheck(lambda *a: gd.gated_delta_rule_ref(*a[:5], 0.3, a[5], True),
                                    [x[:1, :3].detach().requires_grad_() if x.dim() != 4 or x.shape[1] == 9 else x[:1].detach().requires_grad_()
                                     for x in leaves])


def test_calls_without_a_gpu_say_so(nat):
    import amd_tuned_torch as att
    x = torch.randn(2, 5, 2, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        att.rms_norm(x)
    with pytest.raises(RuntimeError, match="GPU"):
        att.gated_delta_rule(x, x, x, x[..., 0], x[..., 0])
    with pytest.raises(RuntimeError, match="GPU"):
        att.gated_delta_rule_update(x[:, 0], x[:, 0], x[:, 0], x[:, 0, :, 0], x[:, 0, :, 0], torch.zeros(2, 2, 8, 8))
