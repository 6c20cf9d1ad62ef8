"""Statistics of large groups whose data hold values far from the others, where sums of differences to one of those would cancel."""
import pytest
import torch

from linrec_amd import _layers

from . import layers_reference as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")

# (batch, positions, channels) in groups, each lane of which goes through 1024 to 8192 values of 4 or 8 channels at a time
SHAPES = [((1, 65536, 1032), 1, torch.bfloat16), ((1, 262144, 1032), 1, torch.bfloat16), ((1, 131072, 516), 1, torch.float32),
          ((4, 70001, 264), 1, torch.float16), ((2, 66000, 774), 3, torch.float32)]


@pytest.mark.parametrize("far", [1.0, 100.0, 1000.0])
@pytest.mark.parametrize("where", ["one position", "every 256th position", "the first of them and one channel of eight", "nowhere, but a mean"])
@pytest.mark.parametrize("shape,groups,dtype", SHAPES, ids=str)
def test_statistics(shape, groups, dtype, where, far):
    x = torch.randn(shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    if where == "one position":
        x[:, 0] = far
    elif where == "every 256th position":
        x[:, ::256] += far
    elif where == "nowhere, but a mean":
        x += far
    else:
        x[:, ::256, ::8] = far
        x[:, 0] = -far
    x = x.to(dtype)
    y, stats, _ = _layers.norm_fwd(x, groups, None, None, 1e-5, "none")
    v = x.double().view(shape[0], shape[1], groups, -1)
    var, mean = torch.var_mean(v, (1, 3), correction=0)
    # a lane adds up at most 8 times 32 differences to a value that takes no more than nine times the sum of squares that
    # remains, in two levels of 32 and 8 terms; a few dozen merges of lanes and chunks follow
    off = (9 * 40 + 64) * ref.U32
    size = v.abs().mean((1, 3)) + var.sqrt()
    ref.assert_within(stats[0], mean.cpu(), 64 * ref.U32 * size.cpu(), "mean")
    # (what the mean is off goes into the sum of squares once more)
    ref.assert_within(stats[1], (1 / torch.sqrt(var + 1e-5)).cpu(), (off / 2 + 64 * ref.U32 * (size / var.sqrt()).cpu()) / var.sqrt().cpu(), "rstd")
    want = ((v - mean[:, None, :, None]) / torch.sqrt(var + 1e-5)[:, None, :, None]).view(shape)
    worst = ((y.double() - want).abs() - ref.UNIT[dtype] * want.abs()).max()
    assert float(worst) <= (off + 128 * ref.U32 * float((size / var.sqrt()).max())) * max(1.0, float(want.abs().max()))


@pytest.mark.parametrize("value", [0.1, 0.7, 1.0 / 3.0])
@pytest.mark.parametrize("positions,channels", [(1048576, 131), (262144, 516)])
def test_sums_of_one_gradient_again_and_again(positions, channels, value):
    """The gradient of a mean: every rounding of a sum that adds the same value goes the same way."""
    x = torch.randn((1, positions, channels), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    d_y = torch.full_like(x, value)
    weight, bias = torch.ones(channels, device=DEV), torch.zeros(channels, device=DEV)
    _, stats, _ = _layers.norm_fwd(x, 1, weight, bias, 1e-5, "none")
    _, d_weight, d_bias = _layers.norm_bwd(d_y, x, 1, weight, bias, stats, 1e-5, "none")
    # two levels of 64 terms each in a lane, those of the workgroups in a tree of at most 40
    want = torch.full((channels,), positions * float(d_y[0, 0, 0]), dtype=torch.float64)
    ref.assert_within(d_bias, want, (64 + 64 + 40) * ref.U32 * want, "d_bias")
    xh = (x[0].double() - stats[0].double()) * stats[1].double()
    # (the normalised values carry three roundings each; sums of them in any order are off by what their sizes allow)
    ref.assert_within(d_weight, (float(d_y[0, 0, 0]) * xh.sum(0)).cpu(), (64 + 64 + 44) * ref.U32 * value * xh.abs().sum(0).cpu(), "d_weight")
