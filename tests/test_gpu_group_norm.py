"""Group norm with an activation on the device, against its definition in float64."""
import pytest
import torch

import linrec_amd
from linrec_amd import _layers

from . import layers_reference as ref
from .layers_reference import same_bits_in_a_graph

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "silu", "gelu"]

# (batch, positions ..., channels), groups
SHAPES = [((1, 1), 1), ((3, 64), 4), ((5, 100), 10), ((7, 1000), 8), ((2, 7, 6), 3), ((2, 33, 222), 6), ((1, 1000, 32), 32),
          ((4, 129, 96), 1), ((2, 5000, 64), 8), ((3, 16384), 2), ((2000, 128), 2), ((2, 9, 11, 40), 5), ((1, 3000, 333), 9),
          ((2, 2, 8192), 1), ((300, 2, 24), 24), ((1, 40000, 16), 2)]


def make(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, d_y = (torch.randn(shape, generator=g) for _ in range(2))
    weight, bias = 1.0 + 0.2 * torch.randn(shape[-1], generator=g), 0.2 * torch.randn(shape[-1], generator=g)
    return (x + 0.5).to(dtype), d_y.to(dtype), weight, bias


def check(x, d_y, weight, bias, groups, act, eps=1e-5, device_x=None, device_d_y=None):
    dtype = x.dtype
    leaves = [x.double().requires_grad_()] + ([] if weight is None else [weight.double().requires_grad_(), bias.double().requires_grad_()])
    y_t = ref.group_norm_act(leaves[0], groups, *(leaves[1:] or (None, None)), eps, act)
    grads_t = torch.autograd.grad(y_t, leaves, d_y.double())
    inputs = [x.to(DEV) if device_x is None else device_x] + ([] if weight is None else [weight.to(DEV), bias.to(DEV)])
    inputs = [t.detach().requires_grad_() for t in inputs]
    y = linrec_amd.group_norm_act(inputs[0], groups, *(inputs[1:] or (None, None)), eps=eps, act=act)
    assert y.dtype == dtype
    grads = torch.autograd.grad(y, inputs, d_y.to(DEV) if device_d_y is None else device_d_y)
    # a normalised value: the mean, the difference and the deviation carry a few roundings of the data's size each, the
    # activation a few more (an fp32 sum in a tree of n terms: log2 n)
    v = x.double().reshape(x.shape[0], -1, groups, x.shape[-1] // groups)
    var, mean = torch.var_mean(v, (1, 3), correction=0, keepdim=True)
    depth = 8 + float(torch.tensor(float(v.shape[1] * v.shape[3])).log2())
    rstd = 1 / torch.sqrt(var + eps)
    off = depth * ref.U32 * (ref.largest((v - mean) * rstd) + 1 + ref.largest(mean * rstd)) * 2
    wide = 1.0 if weight is None else ref.largest(weight) + ref.largest(bias)
    ref.assert_within(y, y_t, ref.UNIT[dtype] * y_t.detach().abs() + off * max(1.0, wide), "y")
    reach = off * 4 * ref.largest(d_y) * max(1.0, wide) * (1 + ref.largest((v - mean) * rstd))
    d_x = grads_t[0]
    ref.assert_within(grads[0], d_x, ref.UNIT[dtype] * d_x.abs() + reach * max(1.0, ref.largest(rstd)), "d_x")
    if weight is not None:
        rows = x.numel() // x.shape[-1]
        for got, want, name, of in zip(grads[1:], grads_t[1:], ("d_weight", "d_bias"), (weight, bias)):
            assert got.dtype == of.dtype
            ref.assert_within(got, want, ref.UNIT[of.dtype] * want.abs() + reach * rows ** 0.5 * 4, name)


def away_from_zero(x, weight, bias, groups):
    """Data whose normalised values keep clear of the corner of relu, where a rounding would change its slope."""
    for seed in range(1, 20):
        z = ref.group_norm_act(x, groups, weight, bias, 1e-5, "none")
        near = z.abs() < 1e-3
        if not near.any():
            return x
        x = torch.where(near, (x.double() + 0.05 * seed).to(x.dtype), x)
    return x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_against_the_definition(shape, groups, dtype):
    x, d_y, weight, bias = make(shape, dtype, seed=sum(shape))
    check(x, d_y, weight, bias, groups, ("silu", "gelu", "none")[sum(shape) % 3])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape,groups", [((6, 96), 3), ((2, 40, 48), 4)])
def test_activations_and_types_of_the_weight(shape, groups, act):
    x, d_y, weight, bias = make(shape, torch.bfloat16, seed=1)
    if act == "relu":
        x = away_from_zero(x, weight, bias, groups)
    check(x, d_y, weight, bias, groups, act)
    if act != "relu":
        check(x, d_y, weight.bfloat16(), bias.bfloat16(), groups, act)
        check(x, d_y, None, None, groups, act)


@pytest.mark.parametrize("shape,groups", [((4, 64), 2), ((2, 50, 32), 4), ((1, 20000, 32), 4)])
def test_values_all_alike_and_far_from_zero(shape, groups):
    x, d_y, weight, bias = make(shape, torch.float32, seed=2)
    check(x + 3000.0, d_y, weight, bias, groups, "silu")
    same = torch.full(shape, 0.75)
    y = linrec_amd.group_norm_act(same.to(DEV), groups, weight.to(DEV), bias.to(DEV), act="none")
    assert torch.equal(y.cpu(), bias.expand(shape))


@pytest.mark.parametrize("shape,groups", [((4, 64), 2), ((3, 50, 32), 4), ((2, 20000, 32), 4)])
def test_what_is_not_finite_stays_in_its_group(shape, groups):
    x, d_y, weight, bias = make(shape, torch.float32, seed=3)
    spoiled = x.clone()
    spoiled.view(shape[0], -1, shape[-1])[1, 0, 0] = float("nan")
    spoiled.view(shape[0], -1, shape[-1])[0, -1, -1] = float("inf")
    run = []
    for t in (x, spoiled):
        t = t.to(DEV).requires_grad_()
        y = linrec_amd.group_norm_act(t, groups, weight.to(DEV), bias.to(DEV))
        run.append((y, torch.autograd.grad(y, t, d_y.to(DEV))[0]))
    width = shape[-1] // groups
    bad = torch.zeros(shape, dtype=torch.bool)
    bad.view(shape[0], -1, shape[-1])[1, :, :width] = True
    bad.view(shape[0], -1, shape[-1])[0, :, -width:] = True
    for good, got in zip(*run):
        assert torch.equal(good[~bad], got[~bad]) and torch.isnan(got[bad]).all()


def test_strides():
    x, d_y, weight, bias = make((2, 30, 24), torch.float32, seed=4)
    wide = torch.zeros((2, 30, 51), device=DEV)
    wide[..., 1:25] = x.to(DEV)
    gradient = d_y.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    check(x, d_y, weight, bias, 3, "silu", device_x=wide[..., 1:25], device_d_y=gradient)
    check(x, d_y, weight, bias, 3, "silu", device_x=x.to(DEV).transpose(1, 2).contiguous().transpose(1, 2))
    check(x, torch.ones_like(d_y), weight, bias, 3, "silu", device_d_y=torch.ones((), device=DEV).expand(2, 30, 24))


def test_images_in_channels_last_memory():
    g = torch.Generator().manual_seed(5)
    image = torch.randn((2, 12, 5, 7), generator=g).to(DEV).to(memory_format=torch.channels_last)
    y = linrec_amd.group_norm_act(image.permute(0, 2, 3, 1), 4, act="none")
    want = torch.nn.functional.group_norm(image.double().cpu(), 4).permute(0, 2, 3, 1)
    ref.assert_within(y, want, 40 * ref.U32 * 5, "image")


def test_differences():
    x, d_y, weight, bias = (t.to(DEV) for t in make((2, 60, 32), torch.float32, seed=6))
    leaves = [x, weight, bias]

    def loss(values):
        return float((linrec_amd.group_norm_act(values[0], 4, *values[1:], act="gelu").double() * d_y).sum())
    tracked = [t.clone().requires_grad_() for t in leaves]
    grads = torch.autograd.grad(linrec_amd.group_norm_act(tracked[0], 4, *tracked[1:], act="gelu"), tracked, d_y)
    g = torch.Generator(device=DEV).manual_seed(1)
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        v = torch.randn(leaf.shape, generator=g, device=DEV)
        step = 2.0 ** -7
        up, down = (loss([t + s * step * v if j == i else t for j, t in enumerate(leaves)]) for s in (1, -1))
        got, want = float((grad.double() * v).sum()), (up - down) / (2 * step)
        assert abs(got - want) <= 1e-3 * float(grad.double().norm() * v.double().norm()) + 1e-3 * abs(want), (i, got, want)


def test_empty_tensors():
    for shape in ((0, 8), (0, 3, 8), (2, 0, 8)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        weight, bias = (torch.ones(8, device=DEV, requires_grad=True) for _ in range(2))
        y = linrec_amd.group_norm_act(x, 2, weight, bias)
        grads = torch.autograd.grad(y, (x, weight, bias), torch.empty_like(y))
        assert y.shape == shape and all(torch.equal(g, torch.zeros_like(g)) for g in grads)


@pytest.mark.parametrize("shape,groups", [((700, 256), 8), ((3, 2500, 64), 8), ((2, 300, 64), 2)])
def test_the_same_bits_every_time_and_in_a_graph(shape, groups):
    x, d_y, weight, bias = (t.to(DEV) for t in make(shape, torch.bfloat16, seed=7))

    def run():
        y, stats, _ = _layers.norm_fwd(x, groups, weight, bias, 1e-5, "silu")
        return (y, stats, *_layers.norm_bwd(d_y, x, groups, weight, bias, stats, 1e-5, "silu"))
    same_bits_in_a_graph(run)


def test_traced_calls_are_the_same_operator():
    x, d_y, weight, bias = (t.to(DEV) for t in make((3, 5, 12), torch.float32, seed=8))
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    args = (x, 3, weight, bias, 1e-5, "silu")
    torch.library.opcheck(linrec_amd.layers.group_norm_act_fwd, args, test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    y, y2 = linrec_amd.layers.group_norm_act_fwd(*args)[0], linrec_amd.group_norm_act(x, 3, weight, bias)
    assert torch.equal(y, y2)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, d_y), torch.autograd.grad(y2, leaves, d_y)))


def test_refusals():
    x, _, weight, bias = (t.to(DEV) for t in make((2, 5, 8), torch.bfloat16))
    call = linrec_amd.group_norm_act
    for args, kw, text in [
            ((x, 3), {}, "groups"), ((x, 0), {}, "groups"), ((x[0, 0], 2), {}, "dimensions"), ((x, 2), {"act": "tanh"}, "act must be"),
            ((x, 2, weight), {}, "go together"), ((x, 2, weight[:4], bias[:4]), {}, "weight has size"),
            ((x, 2, weight.half(), bias.half()), {}, "must both be"), ((x, 2, weight, bias.bfloat16()), {}, "must both be"),
            ((x, 2, weight.cpu(), bias.cpu()), {}, "weight is on"), ((x.double(), 2), {}, "float32, float16 or bfloat16")]:
        with pytest.raises(RuntimeError, match=text):
            call(*args, **kw)
