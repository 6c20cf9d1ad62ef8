"""Root-mean-square norm with a residual and with an output in 8 bits, on the device, against float64.

A row's sum of squares, root and products are at most 64 dependent fp32 roundings (a lane adds up to 32 values, ten joins of lanes, at
most 16 of waves, and the rest), so values are 64 * 2^-24 of the terms off that they consist of, and half a step of their type more."""
import pytest
import torch

import linrec_amd
from linrec_amd import _layers

from .delta_reference import HALF_STEP
from .layers_reference import U32, assert_within, same_bits_in_a_graph

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-6
FEW = 64 * U32


def make(shape, dtype, seed=0, weight_dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x, residual, d_y, d_total = (torch.randn(shape, generator=g).to(dtype) for _ in range(4))
    weight = (1.0 + 0.3 * torch.randn(shape[-1:], generator=g)).to(weight_dtype)
    return x, residual, d_y, d_total, weight


def plain(total, weight):
    """(h, rstd) in float64"""
    total = total.double()
    rstd = 1.0 / torch.sqrt((total * total).mean(-1, keepdim=True) + EPS)
    return total * rstd, rstd


def check(x, residual, d_y, d_total, weight, on_device=None):
    dtype = x.dtype
    total = x if residual is None else (x.float() + residual.float()).to(dtype)  # rounded once: the same bits everywhere
    w = torch.ones(x.shape[-1], dtype=torch.float64) if weight is None else weight.double()
    h, rstd = plain(total, weight)
    y_t = h * w
    g = d_y.double() * w
    mean, mean_abs = (g * h).mean(-1, keepdim=True), (g * h).abs().mean(-1, keepdim=True)
    more = 0.0 if residual is None else d_total.double()
    dx_t = rstd * (g - h * mean) + more
    dx_terms = rstd * (g.abs() + h.abs() * mean_abs) + (0.0 if residual is None else d_total.double().abs())

    tensors = [x, residual, weight] if on_device is None else on_device
    x_d, r_d, w_d = (None if t is None else t.to(DEV).detach().requires_grad_() for t in tensors)
    out = linrec_amd.rms_norm(x_d, w_d, residual=r_d, eps=EPS)
    y, total_d = (out, None) if residual is None else out
    assert y.dtype == dtype and y.is_contiguous()
    if residual is not None:
        assert torch.equal(total_d.cpu(), total)
    assert_within(y, y_t, (HALF_STEP[dtype] + FEW) * y_t.abs() + 1e-30 + (2.0 ** -25 if dtype == torch.float16 else 0.0), "y")
    leaves = [t for t in (x_d, r_d, w_d) if t is not None]
    outputs = [y] if residual is None else [y, total_d]
    grads = torch.autograd.grad(outputs, leaves, [t.to(DEV) for t in (d_y, d_total)[:len(outputs)]])
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    assert grads[0].shape == x.shape and grads[0].dtype == dtype
    assert_within(grads[0], dx_t, HALF_STEP[dtype] * dx_t.abs() + FEW * dx_terms + tiny, "d_x")
    if residual is not None:
        assert torch.equal(grads[0], grads[1])
    if weight is not None:
        terms = d_y.double() * h
        dw_t, dw_abs = terms.flatten(0, -2).sum(0), terms.flatten(0, -2).abs().sum(0)
        rows = x.numel() // x.shape[-1]
        bound = HALF_STEP[weight.dtype] * dw_t.abs() + (64 + rows / 16) * U32 * dw_abs + 1e-30
        assert grads[-1].dtype == weight.dtype
        assert_within(grads[-1], dw_t, bound + (2.0 ** -25 if weight.dtype == torch.float16 else 0.0), "d_weight")
    with torch.no_grad():
        again = linrec_amd.rms_norm(x_d, w_d, residual=r_d, eps=EPS)
    assert torch.equal(again if residual is None else again[0], y)


SHAPES = [(1, 1), (3, 2), (5, 7), (4, 8), (2, 3, 9), (17, 64), (33, 100), (7, 222), (9, 512), (5, 1000), (3, 2048), (300, 130), (2, 4099),
          (1, 8192), (2, 16384), (1, 16383), (2000, 16), (70000, 3), (3000, 1024), (2600, 600)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_float64(shape, dtype):
    x, residual, d_y, d_total, weight = make(shape, dtype, seed=sum(shape), weight_dtype=dtype if sum(shape) % 2 else torch.float32)
    check(x, residual, d_y, d_total, weight)
    check(x, None, d_y, None, weight if sum(shape) % 3 else None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_long_rows(dtype):
    """So many rows that a wave holds a whole one, and more rows than workgroups."""
    for shape in ((5000, 4096), (9000, 1024), (1500, 8200)):
        x, residual, d_y, d_total, weight = make(shape, dtype, seed=1)
        check(x, residual, d_y, d_total, weight)


@pytest.mark.parametrize("dtype", DTYPES)
def test_heads_of_a_projection(dtype):
    """Rows that lie where a projection put them: two strides, or none that a kernel could follow."""
    g = torch.Generator().manual_seed(0)
    whole = torch.randn((2, 30, 3 * 4 * 24), generator=g).to(dtype)
    part = whole[..., 96:192].unflatten(-1, (4, 24))
    x, residual, d_y, d_total, weight = make((2, 30, 4, 24), dtype, seed=3)
    check(part, None, d_y, None, weight, [whole.to(DEV)[..., 96:192].unflatten(-1, (4, 24)), None, weight])
    check(part, residual, d_y, d_total, weight, [whole.to(DEV)[..., 96:192].unflatten(-1, (4, 24)), residual, weight])
    check(part, residual, d_y, d_total, weight, [whole.to(DEV)[..., 96:192].unflatten(-1, (4, 24)), residual.to(DEV).transpose(0, 2).contiguous().transpose(0, 2), weight])
    turned = x.to(DEV).transpose(-1, -2).contiguous().transpose(-1, -2)
    check(x, None, d_y, None, weight, [turned, None, weight])
    every = x.to(DEV)[:, :, :1].expand(-1, -1, 4, -1)
    check(x[:, :, :1].expand(-1, -1, 4, -1), None, d_y, None, weight, [every, None, weight])


def test_one_of_the_gradients_alone():
    x, residual, d_y, d_total, weight = make((6, 40), torch.float32)
    leaves = [t.to(DEV).requires_grad_() for t in (x, residual, weight)]
    y, total = linrec_amd.rms_norm(leaves[0], leaves[2], residual=leaves[1])
    d_x, d_r, d_w = torch.autograd.grad(total, leaves, d_total.to(DEV), retain_graph=True)
    assert torch.equal(d_x.cpu(), d_total) and torch.equal(d_r, d_x) and torch.equal(d_w, torch.zeros_like(d_w))
    d_x, d_w = torch.autograd.grad(y, (leaves[0], leaves[2]), d_y.to(DEV).expand(6, 40))
    both = torch.autograd.grad((linrec_amd.rms_norm(leaves[0], leaves[2], residual=leaves[1])[0]).sum(), leaves[0])[0]
    assert d_x.shape == both.shape
    # against differences, in float32 of a function that is linear enough at this step
    e = 1e-2
    with torch.no_grad():
        direction = torch.randn(6, 40, generator=torch.Generator().manual_seed(2)).to(DEV)
        up, down = (linrec_amd.rms_norm(leaves[0] + s * e * direction, leaves[2], residual=leaves[1])[0] for s in (1, -1))
        slope = float(((up - down) / (2 * e) * d_y.to(DEV)).sum())
    assert abs(slope - float((d_x * direction).sum())) <= 1e-2 * max(1.0, float((d_x * direction).abs().sum()) ** 0.5)


def test_rows_of_zeros_and_of_what_is_not_finite():
    x = torch.randn(5, 64)
    x[1] = 0.0
    x[2, 3] = float("nan")
    x[3, 60] = float("inf")
    y = linrec_amd.rms_norm(x.to(DEV)).cpu()
    h, _ = plain(x, None)
    assert torch.equal(y[1], torch.zeros(64)) and torch.isnan(y[2]).all() and torch.isnan(y[3, 60]) and torch.equal(y[3, :60], torch.zeros(60))
    assert_within(y[[0, 4]], h[[0, 4]], FEW * h[[0, 4]].abs(), "others")
    for kind in (torch.int8, torch.float8_e4m3fn):
        q, scales = linrec_amd.rms_norm_quantize(x.to(DEV), dtype=kind)
        assert float(scales[1]) == 0.0 and torch.isnan(scales[2]) and torch.isnan(scales[3])
        assert torch.equal(q[1:4].float(), torch.zeros((3, 64), device=DEV)) and float(q[0].float().abs().max()) == (127 if kind == torch.int8 else 448)


@pytest.mark.parametrize("kind,most", [(torch.int8, 127.0), (torch.float8_e4m3fn, 448.0)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (2, 3, 8), (17, 222), (64, 4096), (3, 16384), (2500, 96), (40, 1003), (9000, 512)])
def test_quantized(shape, dtype, kind, most):
    x, residual, _, _, weight = make(shape, dtype, seed=sum(shape))
    for r in (residual, None):
        total = x if r is None else (x.float() + r.float()).to(dtype)
        h, _ = plain(total, weight)
        y = h * weight.double()
        out = linrec_amd.rms_norm_quantize(x.to(DEV), weight.to(DEV), residual=None if r is None else r.to(DEV), eps=EPS, dtype=kind)
        q, scales = out[:2]
        assert q.dtype == kind and q.shape == x.shape and scales.shape == x.shape[:-1] and scales.dtype == torch.float32
        if r is not None:
            assert torch.equal(out[2].cpu(), total)
        scales_t = y.abs().amax(-1) / most
        assert_within(scales, scales_t, FEW * scales_t + 1e-38, "scales")
        units = (y / scales_t.clamp(min=1e-300)[..., None]).abs()
        step = torch.ones_like(units) if kind == torch.int8 else torch.exp2(torch.floor(torch.log2(units.clamp(min=2.0 ** -6))) - 3)
        assert_within(q.float(), y / scales_t.clamp(min=1e-300)[..., None], step / 2 + 2 * FEW * units, "q")


def test_scales_whose_reciprocal_is_infinite():
    x = torch.randn(4, 64)
    weight = torch.full((64,), 1e-39)
    q, scales = linrec_amd.rms_norm_quantize(x.to(DEV), weight.to(DEV))
    h, _ = plain(x, None)
    want = h * float(weight[0])
    # (scales are denormal: a step of 2^-149)
    assert_within(scales, want.abs().amax(-1) / 127, 2.0 ** -148, "scales")
    assert int(q.abs().max()) >= 100


def test_empty_and_refused():
    w = torch.ones(8, device=DEV, requires_grad=True)
    x = torch.empty((0, 8), device=DEV, requires_grad=True)
    y = linrec_amd.rms_norm(x, w)
    d_x, d_w = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == x.shape and d_x.shape == x.shape and torch.equal(d_w, torch.zeros_like(w))
    q, scales = linrec_amd.rms_norm_quantize(x.detach(), w.detach())
    assert q.shape == (0, 8) and scales.shape == (0,)
    with pytest.raises(RuntimeError, match="records no gradient"):
        linrec_amd.rms_norm_quantize(torch.zeros((2, 8), device=DEV), w)


def test_the_same_bits_every_time_and_in_a_graph():
    for dtype in DTYPES:
        x, residual, d_y, d_total, weight = (t.to(DEV) for t in make((700, 333), dtype))

        def run():
            y, total, rstd, _ = _layers.rms_fwd(x, weight, residual, EPS)
            q, _, scales, _ = _layers.rms_fwd(x, weight, residual, EPS, torch.int8)
            return [y, total, rstd, q.float(), scales, *_layers.rms_bwd(d_y, d_total, total, weight, rstd, EPS)]
        same_bits_in_a_graph(run)
