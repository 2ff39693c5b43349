"""Angles of rotary positions, near and far, against their product in 100 digits."""
from __future__ import annotations

import decimal
import math

import pytest
import torch

gpu = pytest.mark.gpu

PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798")
FAR = [0, 1, -1, 2047, 2048, 4095, 10 ** 6 + 1, 10 ** 9, -(1 << 36) - 7, (1 << 40) + 12345, -(1 << 40), (1 << 45) - 3, (1 << 53) + 1,
       10 ** 17 + 1, -(1 << 60) - 1025, (1 << 62) - 1]


def turns100(position: int, freq: float) -> float:
    """position * freq, without whole turns, from -1/2 to 1/2 of one."""
    with decimal.localcontext() as c:
        c.prec = 100
        t = decimal.Decimal(position) * decimal.Decimal(freq) / (2 * PI)
        return float(t - t.to_integral_value())


def freqs():
    return 10000.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64) / 32)


def exact(positions, inv_freq):
    angle = torch.tensor([[2 * math.pi * turns100(p, f) for f in inv_freq.tolist()] for p in positions], dtype=torch.float64)
    return angle.cos(), angle.sin()


def test_statement_at_far_positions():
    """2^-40 of a turn, and 2^-52 of fp64's own."""
    from amd_tuned_torch import rotary_ops as R
    inv = freqs()
    q = torch.cat((torch.ones(len(FAR), 1, 16), torch.zeros(len(FAR), 1, 16)), -1).double()
    got = R.rotary_embedding_ref(q, None, inv, torch.tensor(FAR))[:, 0]
    cos, sin = exact(FAR, inv)
    assert (got - torch.cat((cos, sin), -1)).abs().max() <= 2 * math.pi * 2.0 ** -40


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_far_positions(dev, dtype):
    """As near ones: 2^-20 (here of 1), the angle's part of a turn in fp32 and its sine and cosine, and one rounding."""
    import amd_tuned_torch as P
    inv = freqs()
    q = torch.cat((torch.ones(len(FAR), 1, 16), torch.zeros(len(FAR), 1, 16)), -1).to(dev, dtype)
    cos, sin = exact(FAR, inv)
    want = torch.cat((cos, sin), -1)
    lim = 2.0 ** -20 + (2.0 ** -8 * want.abs() if dtype == torch.bfloat16 else 0)
    got = P.rotary_embedding(q, None, inv.to(dev), torch.tensor(FAR, device=dev))[:, 0]
    assert ((got.cpu().double() - want).abs() <= lim).all()
    back = P.rotary_embedding(q, None, inv.to(dev), -torch.tensor(FAR, device=dev))[:, 0].cpu().double()
    assert ((back - torch.cat((cos, -sin), -1)).abs() <= lim).all()
    for p, c, s in zip(FAR, cos, sin):                                      # the same as an offset
        if -(1 << 62) <= p:
            got = P.rotary_embedding(q[:1], None, inv.to(dev), p)[0, 0].cpu().double()
            assert ((got - torch.cat((c, s))).abs() <= 2.0 ** -20 + (2.0 ** -8 if dtype == torch.bfloat16 else 0)).all(), p


@gpu
def test_sine_and_cosine_are_rounded_once(dev):
    """A pair of (1, 0) becomes (scale cos, scale sin), whose products with 1 and 0 are exact in fp32: within half a
    step of fp32, 2^-24 of the value, and 2 pi 2^-40 of scale where the value is small."""
    import amd_tuned_torch as P
    inv = freqs()
    positions = list(range(0, 4000, 37)) + [10 ** 6 + i for i in range(50)] + FAR
    q = torch.cat((torch.ones(len(positions), 1, 16), torch.zeros(len(positions), 1, 16)), -1).to(dev)
    want = torch.cat(exact(positions, inv), -1)
    for scale in (1.0, 1.25):                                               # (both exact in fp32)
        got = P.rotary_embedding(q, None, inv.to(dev), torch.tensor(positions, device=dev), scale=scale)[:, 0].cpu().double()
        off = (got - scale * want).abs() - 2.0 ** -24 * scale * want.abs() - scale * 2 * math.pi * 2.0 ** -40
        assert off.max() <= 0, off.max().item()
