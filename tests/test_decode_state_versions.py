"""Decode steps write a cache of states in place.  A state that a backward still needs is then gone, and autograd
has to say so, as it does after an operation of torch's in place."""
from __future__ import annotations

import pytest
import torch

gpu = pytest.mark.gpu


def linear(P, dev):
    r = lambda *s: torch.randn(*s, device=dev)  # noqa: E731
    token = [r(2, 1, 16), r(2, 1, 16), r(2, 2, 16), -r(2, 2).abs()]
    return (lambda cache: P.linear_attention(*[x[:, None] for x in token[:2]], token[2][:, None].requires_grad_(), token[3][:, None],
                                             initial_state=cache),
            lambda cache: P.linear_attention_update(*token, cache), r(2, 2, 16, 16))


def delta(P, dev):
    r = lambda *s: torch.randn(*s, device=dev)  # noqa: E731
    token = [r(2, 1, 16), torch.nn.functional.normalize(r(2, 1, 16), dim=-1), r(2, 2, 16), -r(2, 2).abs(), r(2, 2).sigmoid()]
    return (lambda cache: P.gated_delta_rule(*[x[:, None] for x in token[:2]], token[2][:, None].requires_grad_(),
                                             *[x[:, None] for x in token[3:]], initial_state=cache),
            lambda cache: P.gated_delta_rule_update(*token, cache), r(2, 2, 16, 16))


OPERATORS = {"linear attention": (linear, "_linear_update_check"), "gated delta rule": (delta, "_delta_update_check")}


class Launches:
    """A library of which every call succeeds and does nothing."""

    def __getattr__(self, name):
        return lambda *a: 0


@pytest.mark.parametrize("name", OPERATORS)
def test_a_step_counts_as_an_operation_in_place(name, monkeypatch):
    """Without a GPU: the call with the launch left out.  A tensor of inference mode has no version."""
    import amd_tuned_torch as P
    from amd_tuned_torch import _native as nat
    make, check = OPERATORS[name]
    monkeypatch.setattr(nat, check, lambda *a: None)
    monkeypatch.setattr(nat, "lib", Launches)
    monkeypatch.setattr(nat, "_on", lambda device, fn, *a: 0)
    monkeypatch.setattr(nat, "_stream", lambda t: None)
    _, step, cache = make(P, "cpu")
    view, before = cache[:1], cache._version
    with torch.no_grad():
        step(cache)
        assert cache._version > before and view._version == cache._version
    with torch.inference_mode():
        _, step, cache = make(P, "cpu")
        step(cache)


@gpu
@pytest.mark.parametrize("name", OPERATORS)
def test_a_backward_whose_state_was_stepped_on(dev, name):
    import amd_tuned_torch as P
    whole, step, cache = OPERATORS[name][0](P, dev)
    out = whole(cache)
    with torch.no_grad():
        step(cache)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    out = whole(cache)
    out.sum().backward()                                                     # nothing came between
    with torch.inference_mode():
        step(cache.clone())
