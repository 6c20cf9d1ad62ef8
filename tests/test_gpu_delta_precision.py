"""What the gated delta rule gives in float32 beside 16-bit inputs (states, gradients of the gates and of h0) has float32's accuracy.

The unit is e = 2^-24, float32's half step.  An operand that is not an input is three numbers of 8 bits (or two of 11 beside fp16), off by e
at most.  A sum of up to 256 products is taken 32 of them at a time, for up to six pairs of such numbers: 48 roundings of a running sum, each
of at most e of it, e / sqrt(3) on average, while the sum grows to its size as a random walk: e sqrt(48 / 3 / 2) = 2.8 e of it.  A result
passes about eight such sums a chunk, in independent directions: 8 e.  Chunks that a state remembers add up like independent numbers, as do the
first chunk's initial state and decays: sqrt(2 + chunks).  A gradient passes the forward and the backward: twice that."""
import pytest
import torch

import linrec_amd

from . import delta_reference as ref
from .test_gpu_delta import DEV, NAMES, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lead,heads,dims", [((1, 128), (1, 2), (24, 128)), ((2, 150), (1, 2), (64, 64)), ((1, 128), (2, 2), (128, 128)),
                                             ((1, 100), (1, 2), (100, 33)), ((1, 128), (1, 1), (200, 64)), ((1, 192), (1, 3), (128, 20))])
def test_results_in_float32_have_its_accuracy(lead, heads, dims, dtype):
    *inputs, d_o, d_state = make(lead, heads, dims, dtype, seed=11)
    leaves = [t.double().requires_grad_() for t in inputs]
    o, state = ref.gated_delta(*leaves)
    want = torch.autograd.grad((o * d_o.double()).sum() + (state * d_state.double()).sum(), leaves)
    leaves = [t.to(DEV).requires_grad_() for t in inputs]
    got_o, got_state = linrec_amd.gated_delta(*leaves[:5], h0=leaves[5], return_state=True)
    got = torch.autograd.grad([got_o, got_state], leaves, [d_o.to(DEV), d_state.to(DEV)])
    share = 8 * 2.0 ** -24 * (2 + lead[1] / 64) ** 0.5
    ref.assert_near(got_state, state, share, "state")
    for name, value, true in list(zip(NAMES, got, want))[3:]:
        ref.assert_near(value, true, 2 * share, name, (dims[0] * dims[1]) ** 0.5 if name == "d_log_decay" else 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lead,heads,dims", [((16, 128), (2, 2), (128, 128)), ((16, 128), (1, 4), (48, 64)), ((8, 100), (1, 2), (200, 160))])
def test_results_in_16_bits_are_roundings_of_such_results(lead, heads, dims, dtype):
    """Beside the true result's rounding: a value is rounded to the other side with the probability |error| / step, and is a step off then.  The squares of
    these add up to sum |error| step, at most |error| |step| in norm, with a step of 2^-7 (2^-10 in fp16) of a value at most."""
    q, k, v, log_decay, beta, h0, *_ = make(lead, heads, dims, dtype, seed=12)
    want, _ = ref.gated_delta(q, k, v, log_decay, beta, h0)
    got = linrec_amd.gated_delta(*(t.to(DEV) for t in (q, k, v, log_decay, beta)), h0=h0.to(DEV))
    rounded = want.to(dtype).double()
    share = 8 * 2.0 ** -24 * (2 + lead[1] / 64) ** 0.5
    off = float((got.double().cpu() - rounded).norm() / rounded.norm())
    assert off <= (share * 2 * ref.HALF_STEP[dtype]) ** 0.5, off
