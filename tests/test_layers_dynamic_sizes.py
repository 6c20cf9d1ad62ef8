"""Fake functions of the layer operators keep symbolic sizes symbolic: a compiled program is not compiled again for every length."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext

import linrec_amd
from linrec_amd import _layers


def symbolic(mode, t):
    return mode.from_tensor(t, symbolic_context=StatelessSymbolicContext(dynamic_sizes=[DimDynamic.DYNAMIC] * t.dim()))


@pytest.mark.parametrize("packed", [False, True])
def test_gated_linrec(packed):
    mode = FakeTensorMode(shape_env=ShapeEnv())
    x, rate, cu = (symbolic(mode, t) for t in (torch.randn(2, 300, 6), torch.randn(6), torch.zeros(5, dtype=torch.int32)))
    with mode:
        if packed:
            x = x[0]
        x.requires_grad_()
        h, state = linrec_amd.gated_linrec(x, x, x, rate, cu_seqlens=cu if packed else None, return_state=True)
        d_x, = torch.autograd.grad(h, x, h.detach())
    assert not [n for t in (h, d_x, state) for n in t.shape if isinstance(n, int)], (h.shape, d_x.shape, state.shape)


def test_the_others():
    mode = FakeTensorMode(shape_env=ShapeEnv())
    x, rate, state, weight, tokens = (symbolic(mode, t) for t in (torch.randn(2, 300, 6), torch.randn(6), torch.randn(300, 6), torch.randn(9, 6),
                                                                  torch.zeros((4, 5), dtype=torch.long)))
    with mode:
        results = [linrec_amd.gated_linrec_step(x[0], x[0], x[0], rate, state), linrec_amd.embedding(tokens, weight, padding_idx=3),
                   linrec_amd.group_norm_act(x, 3)]
    assert not [n for t in results for n in t.shape if isinstance(n, int)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_sizes_of_saved_values_are_the_library_s(dtype):
    for batch, time, channels in [(0, 5, 5), (1, 0, 4), (2, 3, 0), (1, 1, 1), (3, 63, 7), (2, 64, 7), (2, 65, 130), (8, 4096, 2048), (1, 100001, 250),
                                  (1, 2147479551, 3)]:
        assert _layers.gated_saved_numel(dtype, batch, time, channels) == _layers._lib.linrec_gated_saved_floats(_layers.DTYPES[dtype], batch, time,
                                                                                                                  channels)
