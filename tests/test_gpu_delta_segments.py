"""Gated delta rule over long sequences with few heads, which are cut into segments that run side by side."""
import ctypes

import pytest
import torch

from linrec_amd import _delta

from . import delta_reference as ref
from . import test_gpu_delta as delta
from .layers_reference import same_bits_in_a_graph
from .test_gpu_delta import DEV, DTYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,heads,dims", [((1, 1700), (1, 1), (64, 32)), ((2, 1601), (1, 2), (24, 40)), ((1, 2049), (1, 1), (128, 72)),
                                             ((1, 1540), (1, 1), (200, 16))])
def test_against_the_loop(lead, heads, dims, dtype):
    delta.check(delta.make(lead, heads, dims, dtype, seed=sum(lead), pace=0.02))


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_sequences(dtype):
    bounds = [0, 0, 1900, 1901, 4000, 4000, 4030]
    delta.check(delta.make((bounds[-1],), (1, 1), (32, 16), dtype, seed=2, sequences=len(bounds) - 1, pace=0.02), bounds)


def test_without_a_state_and_with_strong_decays():
    delta.check(delta.make((1, 1800), (1, 1), (40, 24), torch.bfloat16, seed=5), with_state=False)
    data = list(delta.make((1, 1800), (1, 1), (40, 24), torch.float32, seed=6, pace=4.0))
    data[3][0, 600:620] = -1e5
    delta.check(tuple(data))


def test_the_same_bits_every_time_and_in_a_graph():
    q, k, v, log_decay, beta, h0, d_o, d_state = (t.to(DEV) for t in delta.make((1, 3000), (1, 2), (128, 64), torch.bfloat16, seed=3))

    def run():
        o, state, _ = _delta.delta_fwd(q, k, v, log_decay, beta, h0, None, 0.1)
        return [o, state, *_delta.delta_bwd(d_o, d_state, q, k, v, log_decay, beta, h0, None, 0.1)]
    same_bits_in_a_graph(run)


def test_bounds_that_are_wrong_stay_inside():
    x = torch.zeros((4096, 1, 16), device=DEV)
    gate = torch.zeros((4096, 1), device=DEV)
    for bounds in ([0, 5000], [-5, 4096], [0, 4000, 20, 4096], [4096, 0, 4096], [10, 2000], [2 ** 31 - 1, -2 ** 31, 4096], [4096] * 3, [0, 4096, 0, 4096]):
        cu = torch.tensor(bounds, dtype=torch.int32, device=DEV)
        o, state, _ = _delta.delta_fwd(x, x, x, gate, gate, None, cu, 1.0)
        grads = _delta.delta_bwd(x, state, x, x, x, gate, gate, None, cu, 1.0)
        torch.cuda.synchronize()
        assert o.shape == x.shape and grads[0].shape == x.shape


def test_these_sizes_are_cut():
    """(by the scratch that they ask for: that of the segments comes on top of what a chunk and head takes)"""
    def need(batch, time, heads):
        a = _delta.Delta(dtype=0, key_heads=heads, heads=heads, key_dim=64, value_dim=32, batch=batch, time=time, sequences=batch)
        return _delta._lib.linrec_delta_scratch_bytes(ctypes.byref(a), 0)
    each = need(64, 64, 4) // 256
    # 27 chunks in segments of 8: 4 of (columns + key channels) x key channels of what they make, and columns x key channels of what enters
    assert need(1, 1700, 1) >= 27 * each + 4 * ((32 + 64) * 64 + 32 * 64) * 4 and need(64, 1728, 4) <= 64 * 27 * 4 * each + 3 * 256
