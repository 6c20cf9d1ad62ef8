"""Group norm with relu where channels are switched off by a bias of minus infinity: they are zero and take no part in any gradient."""
import pytest
import torch

import linrec_amd

from .test_gpu_group_norm import away_from_zero, make

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((40, 64), 4), ((2, 30, 64), 4), ((1, 9000, 16), 1)])
def test_a_bias_of_minus_infinity(shape, groups, dtype):
    x, d_y, weight, bias = make(shape, dtype, seed=9)
    x = away_from_zero(x, weight, bias, groups)
    off = torch.arange(shape[-1]) % 5 == 2
    masked = torch.where(off, torch.full_like(bias, -float("inf")), bias)
    leaves = [t.to(DEV).requires_grad_() for t in (x, weight, masked)]
    y = linrec_amd.group_norm_act(leaves[0], groups, *leaves[1:], act="relu")
    d_x, d_weight, d_bias = torch.autograd.grad(y, leaves, d_y.to(DEV))
    assert not y[..., off].any() and not d_weight[off].any() and not d_bias[off].any()
    # the same with the channels' incoming gradient taken out, which no bias can hide
    leaves = [t.to(DEV).requires_grad_() for t in (x, weight, bias)]
    y2 = linrec_amd.group_norm_act(leaves[0], groups, *leaves[1:], act="relu")
    want = torch.autograd.grad(y2, leaves, torch.where(off, torch.zeros_like(d_y), d_y).to(DEV))
    assert torch.equal(y[..., ~off], y2[..., ~off])
    assert all(torch.equal(a, b) for a, b in zip((d_x, d_weight, d_bias), want))


def test_what_is_not_a_number_stays():
    x, d_y, weight, bias = make((4, 32), torch.float32, seed=10)
    bias[3] = float("nan")
    leaves = [t.to(DEV).requires_grad_() for t in (x, weight, bias)]
    y = linrec_amd.group_norm_act(leaves[0], 2, *leaves[1:], act="relu")
    d_x, _, d_bias = torch.autograd.grad(y, leaves, d_y.to(DEV))
    assert torch.isnan(y[:, 3]).all() and torch.isnan(d_bias[3]) and torch.isnan(d_x[:, :16]).all() and torch.isfinite(d_x[:, 16:]).all()
