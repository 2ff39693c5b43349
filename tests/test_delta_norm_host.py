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
