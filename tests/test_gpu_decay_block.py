"""The example block (examples/decay_block.py): norms, rotary positions, linear attention and projections
together, in training, prefill, packed rows and decoding."""
from __future__ import annotations

import importlib.util
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


def load():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decay_block.py")
    spec = importlib.util.spec_from_file_location("decay_block", path)
    block = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(block)
    return block


def test_block_trains_prefills_and_decodes(dev):
    got = load().main()
    assert math.isfinite(got["loss"]) and all(math.isfinite(v) and v > 0 for v in got["gradients"].values()), got
    # bf16 activations between the operators: a few roundings of 2^-9 each, in another order
    assert got["steps against the whole"] <= 8 * 2.0 ** -8, got
    assert got["packed against the batch"] <= 8 * 2.0 ** -8, got


def test_block_gradients(dev, monkeypatch):
    """In fp32 against the block of the operators' statements in torch operations: the same formulas, so what
    differs is the order of sums of up to a few hundred terms, 2^-24 each, through five operators: 1e-4 of a
    parameter's largest gradient is over a thousand of those."""
    import amd_tuned_torch as att
    module = load()
    torch.manual_seed(1)
    block = module.DecayBlock(width=96, heads_k=2, heads_v=4, dim_k=32, dim_v=40, stretch=4.0, dtype=torch.float32)
    x, r = (torch.randn(2, 83, 96, device=dev) for _ in range(2))
    x.requires_grad_()

    def grads():
        out, h = block(x, r)
        loss = (out * torch.arange(96, device=dev).sin()).sum() + h.square().sum()
        return out.detach(), torch.autograd.grad(loss, [x, *block.parameters()])

    out, got = grads()
    ref = {"rms_norm": lambda x, w, residual: att.rms_norm_ops.rms_norm_ref(x, w, residual=residual),
           "rotary_embedding": att.rotary_ops.rotary_embedding_ref,
           "linear_attention": att.linear_attention_ops.linear_attention_ref,
           "rms_norm_gated": att.rms_norm_ops.rms_norm_gated_ref}
    for name, fn in ref.items():
        monkeypatch.setattr(module.att, name, fn)
    want_out, want = grads()
    assert (out - want_out).abs().max() <= 1e-4 * want_out.abs().max()
    for a, b in zip(got, want):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max()
