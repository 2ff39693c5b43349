"""Layouts that calls of linear attention may have: axes of length 1, whose strides say nothing."""
from __future__ import annotations

import ctypes

import pytest
import torch

gpu = pytest.mark.gpu


def one_token(b, hk, hv, dk, dv, dtype, dev="cpu"):
    """q, k, v, g of one token of b sequences, sequence after sequence along the second axis of the memory: the
    stride of the token axis is that of all sequences, more than 2^22 elements.  They are contiguous, so a copy has
    the same strides."""
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(1, b, *s, generator=gen).to(dev)  # noqa: E731
    q, k, v = (r(h, d).to(dtype).transpose(0, 1) for h, d in ((hk, dk), (hk, dk), (hv, dv)))
    g = (-r(hv).abs()).transpose(0, 1).as_strided((b, 1, hv), (hv, 1 << 23, 1))
    assert all(x.shape[1] == 1 and x.stride(1) >= 1 << 22 and x.contiguous().stride(1) >= 1 << 22 for x in (q, k, v, g))
    return q, k, v, g


def test_one_token_has_no_stride(monkeypatch):
    """What the package hands over for it is within what the C entries take; they look at no stride of one token."""
    from amd_tuned_torch import _native as nat
    nat.load()
    q, k, v, g = one_token(1024, 32, 32, 128, 128, torch.bfloat16)
    monkeypatch.setattr(nat, "_linear_check", lambda q, *a: q.shape[0])
    monkeypatch.setattr(nat, "_on", lambda device, fn, *a: fn(*a))
    monkeypatch.setattr(nat, "_stream", lambda t: None)
    blk = nat._linear_block(q, k, v, g, 1.0, None, None)
    a = blk[0]
    assert blk[6] is None                                                    # nothing was copied
    assert all(abs(s[1]) < 1 << 22 for s in (a.q_stride, a.k_stride, a.v_stride, a.g_stride))
    assert list(a.q_stride)[::2] == [32 * 128, 128] and list(a.g_stride)[::2] == [32, 1]
    assert blk[5] > 0                                                        # the backward has a workspace for it
    nat._tls.la = None
    P = 1 << 20
    a = nat._LinearArgs(k=P, v=P, g=P, out=P, N=2, T=1, Hk=2, Hv=4, K=64, V=64, dtype=nat.ATK_BF16, g_dtype=nat.ATK_BF16)
    for far in (1 << 22, 1 << 40, -64):
        for s in (a.q_stride, a.k_stride, a.v_stride, a.g_stride):
            s[1] = far
        assert nat.lib().atk_linear_attn_fwd(ctypes.addressof(a)) == nat.ATK_EINVAL   # (q is null)
        a.T = 2
        assert nat.lib().atk_linear_attn_fwd(ctypes.addressof(a)) == nat.ATK_UNSUPPORTED
        a.T = 1


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_one_token_of_many_sequences(dev, dtype):
    """The same numbers in another layout: equal bits, forward and backward."""
    import amd_tuned_torch as P
    b, h, d = 1024, 32, 128
    args = one_token(b, h, h, d, d, dtype, dev)
    dense = [x.flatten().clone().view(b, 1, *x.shape[2:]) for x in args]
    dout = torch.randn(b, 1, h, d, device=dev).to(dtype)
    got = []
    for a in (args, dense):
        leaves = [x.detach().requires_grad_() for x in a]
        out = P.linear_attention(*leaves)
        got.append((out.detach(), *torch.autograd.grad(out, leaves, dout)))
    assert all(torch.equal(x, y) for x, y in zip(*got))


@gpu
@pytest.mark.parametrize("dv", [64, 66])
def test_a_cache_without_slots(dev, dv):
    """Every sequence is a row of padding: outputs of zeros."""
    import amd_tuned_torch as P
    r = lambda *s: torch.randn(*s, device=dev)  # noqa: E731
    out = P.linear_attention_update(r(3, 1, 64), r(3, 1, 64), r(3, 2, dv), -r(3, 2).abs(), torch.zeros(0, 2, 64, dv, device=dev),
                                    state_indices=torch.tensor([-1, 0, 7], dtype=torch.int32, device=dev))
    assert out.shape == (3, 2, dv) and out.eq(0).all()


def test_null_states_of_slots_are_refused():
    from amd_tuned_torch import _native as nat
    nat.load()
    P = 1 << 20
    a = nat._LinearUpdateArgs(q=P, k=P, v=P, g=P, out=P, state_indices=P, N=2, slots=1, Hk=2, Hv=4, K=64, V=64, dtype=nat.ATK_BF16,
                              g_dtype=nat.ATK_BF16)
    assert nat.lib().atk_linear_attn_update(ctypes.addressof(a)) == nat.ATK_EINVAL
    a.slots, a.state_indices = 0, None
    assert nat.lib().atk_linear_attn_update(ctypes.addressof(a)) == nat.ATK_EINVAL   # fewer slots than sequences
