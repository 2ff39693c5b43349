"""Linear attention where fewer bits than an fp32 product's would show: results next to a border between two values
of a 16-bit type."""
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
