"""Forward-mode differentiation of the layer operators is refused, in dual levels and under torch.func.jvp: a tangent is never dropped."""
import pytest
import torch
from torch.autograd import forward_ad

import linrec_amd


def calls():
    g = torch.Generator().manual_seed(0)
    x, rate, h0, tokens = torch.randn((2, 3, 4), generator=g), torch.randn(4, generator=g), torch.randn((2, 4), generator=g), torch.tensor([0, 1])
    return {
        "gated x": (lambda t: linrec_amd.gated_linrec(t, x, x, rate), x), "gated gate": (lambda t: linrec_amd.gated_linrec(x, x, t, rate), x),
        "gated rate": (lambda t: linrec_amd.gated_linrec(x, x, x, t, h0=h0), rate),
        "gated h0": (lambda t: linrec_amd.gated_linrec(x, x, x, rate, h0=t, return_state=True)[1], h0),
        "step": (lambda t: linrec_amd.gated_linrec_step(t, h0, h0, rate, h0.clone()), h0),
        "norm x": (lambda t: linrec_amd.group_norm_act(t, 2), x), "norm bias": (lambda t: linrec_amd.group_norm_act(x, 2, rate, t), rate),
        "embedding": (lambda t: linrec_amd.embedding(tokens, t), h0)}


@pytest.mark.parametrize("name", calls())
def test_a_tangent_is_refused(name):
    call, t = calls()[name]
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="jvp"):
        call(forward_ad.make_dual(t, torch.ones_like(t)))
    with forward_ad.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
        call(forward_ad.make_dual(t, torch.ones_like(t)))
    with pytest.raises(RuntimeError, match="jvp"):
        torch.func.jvp(call, (t,), (torch.ones_like(t),))
    # without a tangent the level does not matter: the next refusal is that of host tensors
    with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError), match="needs device tensors"):
        call(t)
