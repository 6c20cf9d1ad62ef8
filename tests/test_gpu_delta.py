"""Gated delta rule on the device, forward and backward, against the loop over positions in float64."""
import pytest
import torch

import linrec_amd
from linrec_amd import _delta

from . import delta_reference as ref
from .layers_reference import same_bits_in_a_graph

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def unit(*shape, g):
    rows = torch.randn(shape, generator=g)
    return rows / rows.norm(dim=-1, keepdim=True)


def make(lead, heads, dims, dtype, seed=0, sequences=None, pace=0.2):
    """q, k, v, log_decay, beta, h0 and output gradients on the CPU, q, k, v and d_o rounded to `dtype`."""
    g = torch.Generator().manual_seed(seed)
    (key_heads, heads), (key_dim, value_dim) = heads, dims
    q, k = (unit(*lead, key_heads, key_dim, g=g).to(dtype) for _ in range(2))
    v, d_o = (torch.randn((*lead, heads, value_dim), generator=g).to(dtype) for _ in range(2))
    log_decay = -pace * torch.rand((*lead, heads), generator=g)
    beta = torch.rand((*lead, heads), generator=g)
    n = lead[0] if sequences is None else sequences
    h0, d_state = (torch.randn((n, heads, key_dim, value_dim), generator=g) for _ in range(2))
    return q, k, v, log_decay, beta, h0, d_o, d_state


NAMES = ("d_q", "d_k", "d_v", "d_log_decay", "d_beta", "d_h0")


def check(data, bounds=None, with_state=True, scale=None, on_device=None):
    """Outputs and gradients of one call against the float64 loop and its derivative."""
    *inputs, h0, d_o, d_state = data
    dtype = inputs[2].dtype
    inputs = inputs + ([h0] if with_state else [])
    leaves = [t.double().requires_grad_() for t in inputs]
    o_t, state_t = ref.gated_delta(*leaves[:5], leaves[5] if with_state else None, bounds, scale)
    loss = (o_t * d_o.double()).sum() + ((state_t * d_state.double()).sum() if with_state else 0.0)
    grads_t = torch.autograd.grad(loss, leaves, materialize_grads=True)

    leaves = [t.to(DEV) for t in inputs] if on_device is None else on_device
    leaves = [t.detach().requires_grad_() for t in leaves]
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=DEV)
    o, state = linrec_amd.gated_delta(*leaves[:5], h0=leaves[5] if with_state else None, cu_seqlens=cu, scale=scale, return_state=True)
    assert o.dtype == dtype and state.dtype == torch.float32 and o.is_contiguous()
    outputs, d_outputs = ([o, state], [d_o.to(DEV), d_state.to(DEV)]) if with_state else ([o], [d_o.to(DEV)])
    grads = torch.autograd.grad(outputs, leaves, d_outputs)
    time, q_dim, v_dim = inputs[0].shape[-3], inputs[0].shape[-1], inputs[2].shape[-1]
    ref.assert_near(o, o_t, ref.bound(dtype, dtype, time), "o")
    ref.assert_near(state, state_t, ref.bound(torch.float32, dtype, time), "state")
    for name, leaf, got, want in zip(NAMES, leaves, grads, grads_t):
        assert got.dtype == leaf.dtype and got.shape == leaf.shape
        size = (q_dim * v_dim) ** 0.5 if name == "d_log_decay" else 1.0
        ref.assert_near(got, want, 2 * ref.bound(leaf.dtype, dtype, time), name, size)
    with torch.no_grad():  # without a gradient the same bits
        plain = linrec_amd.gated_delta(*leaves[:5], h0=leaves[5] if with_state else None, cu_seqlens=cu, scale=scale)
    assert torch.equal(plain, o)
    return o, state, grads


CASES = [
    ((1, 1), (1, 1), (1, 1)), ((2, 1), (1, 2), (16, 16)), ((1, 2), (1, 1), (64, 64)), ((1, 63), (2, 2), (32, 16)), ((2, 64), (1, 1), (20, 12)),
    ((1, 65), (1, 3), (128, 128)), ((2, 130), (2, 4), (100, 72)), ((1, 200), (1, 1), (256, 40)), ((1, 129), (1, 2), (200, 33)),
    ((3, 127), (2, 2), (7, 130)), ((1, 300), (1, 1), (128, 64)), ((1, 257), (1, 1), (64, 256)),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,heads,dims", CASES)
def test_against_the_loop(lead, heads, dims, dtype):
    check(make(lead, heads, dims, dtype, seed=sum(lead) + sum(dims)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_a_state_and_with_a_scale(dtype):
    check(make((2, 100), (1, 2), (48, 40), dtype, seed=1), with_state=False)
    check(make((2, 70), (2, 2), (128, 32), dtype, seed=2), scale=0.25)


BOUNDS = [
    [0, 1], [0, 0, 5], [0, 5, 5], [0, 0, 0, 1, 1], [0, 16, 32, 48], [0, 15, 17, 63, 64, 65, 127, 128, 129, 200],
    [0, 64, 128, 256], [0, 200, 200, 200, 201, 300], [0, 1, 2, 3, 4, 5, 6, 7, 8, 100],
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bounds", BOUNDS, ids=lambda b: "-".join(map(str, b)))
def test_packed_sequences(bounds, dtype):
    check(make((bounds[-1],), (1, 2), (36, 24), dtype, seed=len(bounds), sequences=len(bounds) - 1), bounds)


def test_packed_sequences_many_of_them():
    g = torch.Generator().manual_seed(5)
    bounds = [0] + sorted(torch.randint(0, 401, (300,), generator=g).tolist()) + [400]
    check(make((400,), (1, 1), (16, 8), torch.float32, seed=1, sequences=len(bounds) - 1), bounds)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_of_one_projection(dtype):
    q, k, v, log_decay, beta, h0, d_o, d_state = make((2, 90), (2, 4), (40, 24), dtype, seed=9)
    whole = torch.cat([t.flatten(-2) for t in (q, k, v)], -1).to(DEV)
    views = [t.unflatten(-1, (n, -1)) for t, n in zip(whole.split([80, 80, 96], -1), (2, 2, 4))]
    gates = torch.stack([log_decay, beta], -1).to(DEV)
    data = (q, k, v, log_decay, beta, h0, d_o, d_state)
    check(data, on_device=views + [gates[..., 0], gates[..., 1], h0.to(DEV)])
    # heads before time, and channels that are not adjacent
    turned = [t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, log_decay, beta)]
    check(data, on_device=turned + [h0.to(DEV)])
    apart = [t.to(DEV).transpose(-1, -2).contiguous().transpose(-1, -2) for t in (q, k, v)]
    check(data, on_device=apart + [log_decay.to(DEV), beta.to(DEV), h0.to(DEV).transpose(-1, -2).contiguous().transpose(-1, -2)])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strong_decays_and_gates_at_their_ends(dtype):
    data = list(make((1, 150), (1, 2), (32, 32), dtype, seed=4, pace=8.0))
    data[3][0, 10:14] = -300.0
    data[3][0, 80, 0] = -1e5  # forgets everything
    data[3][0, 90] = 0.0
    data[4][0, 20:25] = 0.0
    data[4][0, 30:60] = 1.0
    data[4][0, 100:110] = 2.0
    check(tuple(data))
    forgets = data[3].clone()
    forgets[0, 80, 0] = -float("inf")
    o = [linrec_amd.gated_delta(*(t.to(DEV) for t in (*data[:3], d, data[4]))) for d in (data[3], forgets)]
    assert torch.equal(*o)


def test_alike_keys():
    """Keys that are all the same make the largest inverses."""
    data = list(make((1, 128), (1, 1), (64, 32), torch.float32, seed=6, pace=0.0))
    data[1][:] = data[1][:, :1]
    data[4][:] = 1.0
    check(tuple(data))


def test_the_same_bits_every_time_and_in_a_graph():
    for dtype in DTYPES:
        data = [t.to(DEV) for t in make((2, 200), (2, 4), (128, 96), dtype, seed=3)]
        q, k, v, log_decay, beta, h0, d_o, d_state = data

        def run():
            o, state, _ = _delta.delta_fwd(q, k, v, log_decay, beta, h0, None, 0.1)
            return [o, state, *_delta.delta_bwd(d_o, d_state, q, k, v, log_decay, beta, h0, None, 0.1)]
        same_bits_in_a_graph(run)


def test_no_positions_at_all():
    z = torch.empty((2, 0, 1, 8), device=DEV, requires_grad=True)
    gate = torch.empty((2, 0, 1), device=DEV, requires_grad=True)
    h0 = torch.randn((2, 1, 8, 8), device=DEV, requires_grad=True)
    o, state = linrec_amd.gated_delta(z, z, z, gate, gate, h0=h0, return_state=True)
    assert o.shape == z.shape and torch.equal(state, h0)
    d_z, d_h0 = torch.autograd.grad(state, (z, h0), torch.ones_like(state), allow_unused=True)
    assert torch.equal(d_h0, torch.ones_like(h0)) and d_z.shape == z.shape
    _, state = linrec_amd.gated_delta(z[0], z[0], z[0], gate[0], gate[0], cu_seqlens=torch.zeros(3, dtype=torch.int32, device=DEV), return_state=True)
    assert torch.equal(state, torch.zeros((2, 1, 8, 8), device=DEV))
    z = torch.empty((0, 5, 1, 8), device=DEV)
    assert linrec_amd.gated_delta(z, z, z, z[..., 0], z[..., 0]).shape == z.shape


def test_a_sequence_does_not_see_its_neighbours():
    data = make((192,), (1, 2), (32, 16), torch.float32, seed=8, sequences=3)
    q, k, v, log_decay, beta, _, d_o, _ = (t.to(DEV) for t in data)
    bounds = [0, 70, 100, 192]
    cu = torch.tensor(bounds, dtype=torch.int32, device=DEV)

    def run(v):
        leaf = v.clone().requires_grad_()
        o = linrec_amd.gated_delta(q, k, leaf, log_decay, beta, cu_seqlens=cu)
        return o.detach(), torch.autograd.grad(o, leaf, d_o)[0]
    o, d_v = run(v)
    for bad in (float("nan"), float("inf")):
        spoiled = v.clone()
        spoiled[70:100] = bad
        spoiled[:, 1] = bad
        o2, d_v2 = run(spoiled)
        for sl in (slice(0, 70), slice(100, 192)):
            assert torch.equal(o[sl, 0], o2[sl, 0]) and torch.equal(d_v[sl, 0], d_v2[sl, 0])


def test_bounds_that_are_wrong_stay_inside():
    """Bounds that do not ascend or leave the tensor: what comes out is not specified, nothing else changes."""
    room = torch.full((3, 64, 2, 16), 7.0, device=DEV)
    x = room[1]
    gate = torch.zeros((64, 2), device=DEV)
    for bounds in ([0, 200], [-5, 64], [0, 40, 20, 64], [64, 0, 64], [10, 20], [2 ** 31 - 1, -2 ** 31, 64]):
        cu = torch.tensor(bounds, dtype=torch.int32, device=DEV)
        leaf = x.clone().requires_grad_()
        o, state = linrec_amd.gated_delta(leaf, leaf, leaf, gate, gate, cu_seqlens=cu, return_state=True)
        torch.autograd.grad(o, leaf, torch.ones_like(o))
        torch.cuda.synchronize()
        assert o.shape == x.shape and state.shape == (len(bounds) - 1, 2, 16, 16)
    assert torch.equal(room, torch.full_like(room, 7.0))
