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
