"""The example block (examples/delta_block.py): norms, causal conv, gated delta rule and projections
together, in training, prefill and decoding."""
from __future__ import annotations

import importlib.util
import math
import os

import pytest

pytestmark = pytest.mark.gpu


def test_block_trains_prefills_and_decodes(dev):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "delta_block.py")
    spec = importlib.util.spec_from_file_location("delta_block", path)
    block = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(block)
    got = block.main()
    assert math.isfinite(got["loss"]) and all(math.isfinite(v) and v > 0 for v in got["gradients"].values()), got
    # bf16 activations between the operators: a few roundings of 2^-9 each, in another order
    assert got["steps against the whole"] <= 8 * 2.0 ** -8, got
    # e4m3 rows and weights: 2^-4 at most for each factor, about 2^-5.5 of a product on the mean
    assert got["fp8 projection"] <= 2.0 ** -3, got
