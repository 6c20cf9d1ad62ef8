"""Value heads that share a key head: what belongs to one of them does not depend on the others.

The gradients of q and k are sums over the heads of a group; everything else (o, the states, the gradients of v, the gates and h0) is
made of a head's own numbers and of q and k, by the same operations in the same order whatever the other heads hold and wherever the
head stands in its group.  So it has the same bits when they change, which needs no tolerance."""
import pytest
import torch

import linrec_amd

from . import delta_reference as ref
from .test_gpu_delta import DEV, DTYPES, make

pytestmark = pytest.mark.gpu
# (key heads, value heads), (key_dim, value_dim): widths of 64, 128 and, in two turns, 256 channels
SIZES = [((1, 2), (24, 40)), ((1, 4), (100, 72)), ((2, 6), (64, 64)), ((1, 3), (200, 33)), ((2, 4), (128, 128)), ((1, 2), (256, 8))]
LEAD = {"batch": ((2, 150), None), "packed": ((230,), [0, 70, 70, 199, 230]), "segments": ((1, 1100), None)}


def run(data, bounds):
    """{name: result on the device}, every head's own ones with the heads in front."""
    inputs = [t.to(DEV).requires_grad_() for t in data[:6]]
    d_o, d_state = (t.to(DEV) for t in data[6:])
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=DEV)
    o, state = linrec_amd.gated_delta(*inputs[:5], h0=inputs[5], cu_seqlens=cu, return_state=True)
    d_q, d_k, d_v, d_log_decay, d_beta, d_h0 = torch.autograd.grad([o, state], inputs, [d_o, d_state])
    own = {"o": o.detach().movedim(-2, 0), "state": state.detach().movedim(1, 0), "d_v": d_v.movedim(-2, 0),
           "d_log_decay": d_log_decay.movedim(-1, 0), "d_beta": d_beta.movedim(-1, 0), "d_h0": d_h0.movedim(1, 0)}
    return own, {"d_q": d_q, "d_k": d_k}


def parts(data, head):
    """What a head has alone: v, log_decay, beta, h0, d_o and d_state."""
    _, _, v, log_decay, beta, h0, d_o, d_state = data
    return {"v": v[..., head, :], "log_decay": log_decay[..., head], "beta": beta[..., head], "h0": h0[:, head], "d_o": d_o[..., head, :],
            "d_state": d_state[:, head]}


def data_of(lead, heads, dims, dtype, seed):
    lead, bounds = LEAD[lead]
    return [t.clone() for t in make(lead, heads, dims, dtype, seed=seed, sequences=None if bounds is None else len(bounds) - 1)], bounds


@pytest.mark.parametrize("lead", LEAD)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,dims", SIZES)
def test_a_head_has_the_same_bits_whatever_the_other_heads_hold(heads, dims, dtype, lead):
    data, bounds = data_of(lead, heads, dims, dtype, seed=3)
    want, _ = run(data, bounds)
    first = heads[1] // heads[0] * (heads[0] - 1)  # of the last key head's
    others = [h for h in range(heads[1]) if h != first]
    assert all(torch.isfinite(t).all() for t in want.values())
    for names, change in ((("v", "h0", "d_o", "d_state"), lambda t: t.mul_(128)), (("v",), lambda t: t.fill_(float("nan"))),
                          (("d_o",), lambda t: t.fill_(float("inf"))), (("h0", "d_state"), lambda t: t.fill_(float("nan"))),
                          (("log_decay",), lambda t: t.fill_(float("nan"))), (("beta",), lambda t: t.fill_(float("inf")))):
        changed = [t.clone() for t in data]
        for name in names:
            change(parts(changed, first)[name])
        got, _ = run(changed, bounds)
        for name in want:
            assert torch.equal(got[name][others], want[name][others]), (name, names)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,dims", SIZES)
def test_a_head_has_the_same_bits_at_every_place_of_its_group(heads, dims, dtype):
    data, bounds = data_of("batch", heads, dims, dtype, seed=4)
    want, _ = run(data, bounds)
    shared = heads[1] // heads[0]
    order = [g * shared + h for g in range(heads[0]) for h in reversed(range(shared))]
    q, k, v, log_decay, beta, h0, d_o, d_state = data
    got, _ = run([q, k, v[..., order, :], log_decay[..., order], beta[..., order], h0[:, order], d_o[..., order, :], d_state[:, order]], bounds)
    for name in want:
        assert torch.equal(got[name], want[name][order]), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,dims", SIZES)
@pytest.mark.parametrize("lead", ["batch", "packed"])
def test_heads_of_different_sizes_against_float64(heads, dims, dtype, lead):
    """Every head within the bound of its own size, beside one whose gradients of the gates are 2^14 times as large (2^10 in fp16, which d_q
    would leave); d_q and d_k, sums over heads, within that of the largest."""
    data, bounds = data_of(lead, heads, dims, dtype, seed=5)
    large, factor = parts(data, 0), 32.0 if dtype == torch.float16 else 128.0
    for name in ("v", "h0", "d_o", "d_state"):
        large[name].mul_(factor)
    *inputs, d_o, d_state = data
    leaves = [t.double().requires_grad_() for t in inputs]
    o, state = ref.gated_delta(*leaves, bounds)
    grads = torch.autograd.grad((o * d_o.double()).sum() + (state * d_state.double()).sum(), leaves)
    want = {"o": o.detach().movedim(-2, 0), "state": state.detach().movedim(1, 0), "d_v": grads[2].movedim(-2, 0),
            "d_log_decay": grads[3].movedim(-1, 0), "d_beta": grads[4].movedim(-1, 0), "d_h0": grads[5].movedim(1, 0)}
    got, sums = run(data, bounds)
    time = inputs[0].shape[-3]
    for name, values in want.items():
        kind, times = got[name].dtype, 1 if name in ("o", "state") else 2
        for head in range(heads[1]):
            by = factor if head == 0 else 1.0
            size = by * by * (dims[0] * dims[1]) ** 0.5 if name == "d_log_decay" else by * by if name == "d_beta" else by
            ref.assert_near(got[name][head], values[head], times * ref.bound(kind, dtype, time), f"{name} of head {head}", size)
    for name, true in (("d_q", grads[0]), ("d_k", grads[1])):
        ref.assert_near(sums[name], true, 2 * ref.bound(dtype, dtype, time), name, factor * factor)
