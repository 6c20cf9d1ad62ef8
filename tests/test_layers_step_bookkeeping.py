"""The single-token step updates its states in place behind autograd's back: what it owes to autograd, on the CPU with the launch
left out."""
import pytest
import torch
from torch.autograd import forward_ad

import linrec_amd
from linrec_amd import _layers


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    monkeypatch.setattr(_layers, "_call", lambda *_: None)
    monkeypatch.setattr(_layers, "_check_device", lambda *_: None)
    monkeypatch.setattr(_layers._memory, "table", {}, raising=False)


def inputs(batch=2, channels=4):
    return [torch.randn(batch, channels) for _ in range(3)] + [torch.randn(channels)]


@pytest.mark.parametrize("slots", [None, torch.tensor([2, 0], dtype=torch.int32)])
def test_a_step_counts_as_a_change_of_the_states(slots):
    cache = torch.randn(3, 8)
    state = cache[:, 2:6] if slots is not None else cache[:2, 2:6]
    before = state._version
    for n in range(1, 4):
        linrec_amd.gated_linrec_step(*inputs(), state, slots=slots)
        assert state._version == before + n and cache._version == state._version
    wrong = inputs(batch=3)
    with pytest.raises(RuntimeError):
        linrec_amd.gated_linrec_step(*wrong, state[:, :3], slots=slots)
    assert state._version == before + 3


def test_a_backward_that_needs_the_states_as_they_were_refuses():
    x, gate_a, gate_x, rate = inputs()
    state = torch.randn(2, 4)
    leaf = x[:, None].clone().requires_grad_()
    h = linrec_amd.gated_linrec(leaf, gate_a[:, None], gate_x[:, None], rate, h0=state)
    linrec_amd.gated_linrec_step(x, gate_a, gate_x, rate, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


def test_states_made_in_inference_mode():
    with torch.inference_mode():
        state = torch.randn(2, 4)
        linrec_amd.gated_linrec_step(*inputs(), state)
    with torch.no_grad():
        linrec_amd.gated_linrec_step(*inputs(), state)  # (has no version to count)


@pytest.mark.parametrize("which", range(5))
def test_a_tangent_is_refused(which):
    tensors = inputs() + [torch.randn(2, 4)]
    with forward_ad.dual_level():
        linrec_amd.gated_linrec_step(*tensors)  # (a level alone is no reason)
        dual = list(tensors)
        dual[which] = forward_ad.make_dual(tensors[which], torch.ones_like(tensors[which]))
        with pytest.raises(RuntimeError, match="records no gradient"):
            linrec_amd.gated_linrec_step(*dual)
    # no mode that leaves gradients out changes that: the tangent would be lost all the same
    with forward_ad.dual_level(), torch.no_grad():
        dual = list(tensors)
        dual[which] = forward_ad.make_dual(tensors[which], torch.ones_like(tensors[which]))
        with pytest.raises(RuntimeError, match="records no gradient"):
            linrec_amd.gated_linrec_step(*dual)
