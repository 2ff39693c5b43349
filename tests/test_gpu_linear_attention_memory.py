"""What linear attention leaves in memory that held something else, and its widest heads: rows of no sequence, and
states whose rows and columns take several tiles, in the launch that makes all gradients."""
from __future__ import annotations

import ctypes

import pytest
import torch

from test_gpu_linear_attention import TYPES, check_backward, make

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 300, 1, 2, 256, 256), (1, 150, 1, 1, 256, 512), (1, 200, 1, 1, 192, 160),
                                   (2, 1100, 2, 2, 256, 256), (1, 900, 1, 1, 200, 450)], ids=str)
def test_widest_heads(dev, shape, dtype):
    """More than 128 rows of a state, and as many tiles of its columns for dv as for dq and dk: one launch, also where
    the rows of dO and v take two tiles of their own; of one segment and of several."""
    import amd_tuned_torch as P
    n, t, hk, hv, dk, dv = shape
    args = make((n, t), hk, hv, dk, dv, dtype, dev, seed=t, fixed=t % 4 == 0)
    gen = torch.Generator().manual_seed(3)
    dout = torch.randn(n, t, hv, dv, generator=gen).to(dev, dtype)
    state, dstate = (torch.randn(n, hv, dk, dv, generator=gen).to(dev) for _ in range(2))
    check_backward(P, args, 0.4, state, None, dout, dstate, t / 4 + dk + dv + 100)
    check_backward(P, args, 0.4, None, None, dout, None, t / 4 + dk + dv + 100)


@gpu
@pytest.mark.parametrize("dtype,code", [(torch.bfloat16, 2), (torch.float32, 0)], ids=["bf16", "fp32"])
@pytest.mark.parametrize("cu", [(0, 70), (5000, 5064), (3000, 3000), (19999, 20000), (7, 2000, 9000)], ids=str)
@pytest.mark.parametrize("hk,hv", [(1, 1), (1, 4)])
@pytest.mark.parametrize("fixed", [False, True])
def test_rows_of_no_sequence_are_written(dev, cu, hk, hv, fixed, dtype, code):
    """Through the C entries, results and workspace full of NaN beforehand: zeros outside the sequences, values inside."""
    from amd_tuned_torch import _native as nat
    L = nat.lib()
    assert code == nat._DTYPE_CODE[dtype]
    t, dk, dv, n = 20000, 64, 40, len(cu) - 1
    q, k, v, g = make((1, t), hk, hv, dk, dv, dtype, dev, fixed=fixed)
    off = torch.tensor(cu, dtype=torch.int32, device=dev)
    dout = torch.ones_like(v)
    full = lambda x: torch.full_like(x, float("nan"))  # noqa: E731
    a = nat._LinearArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), g=g.data_ptr(), cu_seqlens=off.data_ptr(), N=n, T=t, Hk=hk,
                        Hv=hv, K=dk, V=dv, dtype=code, g_dtype=nat.ATK_F32, fixed_decay=int(fixed), scale=0.125,
                        stream=torch.cuda.current_stream().cuda_stream)
    for s, x in ((a.q_stride, q), (a.k_stride, k), (a.v_stride, v)):
        s[:] = x.stride()[:3]
    a.g_stride[:] = (0, 0, 1) if fixed else g.stride()
    at = ctypes.addressof(a)

    def with_workspace(size):
        ws = torch.full((size // 4 + 4,), float("nan"), device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), size
        return ws

    out, states = full(v), torch.full((n, hv, dk, dv), float("nan"), device=dev)
    a.out, a.final_state = out.data_ptr(), states.data_ptr()
    ws = with_workspace(L.atk_linear_attn_workspace_bytes(at))
    assert L.atk_linear_attn_fwd(at) == nat.ATK_OK
    grads = [full(x) for x in (q, k, v, g)]
    ws2 = with_workspace(L.atk_linear_attn_bwd_workspace_bytes(at))
    assert L.atk_linear_attn_bwd(at, dout.data_ptr(), None, *[x.data_ptr() for x in grads], None) == nat.ATK_OK
    torch.cuda.synchronize()
    assert ws is not None and ws2 is not None and states.isfinite().all()
    for name, x in zip(("out", "dq", "dk", "dv", "dg"), (out, *grads)):
        assert x.isfinite().all(), name
        if x.dim() > 1:
            assert x[:, :cu[0]].eq(0).all() and x[:, cu[-1]:].eq(0).all(), name
            # (a first token's decay has no state to act on: its gradient is 0)
            assert cu[-1] - cu[0] <= (name == "dg") or x[:, cu[0]:cu[-1]].ne(0).any(), name
