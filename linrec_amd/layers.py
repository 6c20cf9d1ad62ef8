"""Operators of a recurrent layer around the scan: the gated linear recurrence and its single-token step, group norm with an
activation, root-mean-square norm with a residual, and the token embedding.

As in ops.py each operator is a torch.library custom op (fake function, autograd rule) for tracing and compilation, and an
equivalent autograd Function, or a plain call where no gradient is recorded, in eager mode.  Device tensors only.
"""
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _layers

__all__ = ["gated_linrec", "gated_linrec_step", "group_norm_act", "rms_norm", "rms_norm_quantize", "embedding"]

Tensor = torch.Tensor
_PLAIN = (torch.Tensor, torch.nn.Parameter)  # (subclasses, fake ones among them, take the registered operators)


def _traced(*tensors):
    """The call has to go through the registered operator: compilation, tracing, a tensor subclass or a function transform."""
    for t in tensors:
        if t is not None and type(t) not in _PLAIN:
            return True
    return (torch.compiler.is_compiling() or torch._C._are_functorch_transforms_active()
            or torch._C._get_tracing_state() is not None)


def _recorded(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return forward_ad._current_level >= 0


def _refuse_tangents(what, *tensors):
    """Neither the registered operators nor the kernels know a derivative forward; they would drop the tangent."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what}: records no gradient forward (jvp), a tangent of its inputs would be lost")


def _once(backward):
    """once_differentiable, whose wrapper is only paid for where a graph of the backward is asked for."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def call(ctx, *gradients):
        return guarded(ctx, *gradients) if torch.is_grad_enabled() else backward(ctx, *gradients)
    return call


# ---- gated linear recurrence -------------------------------------------------------------------
@torch.library.custom_op("linrec_amd::gated_linrec_fwd", mutates_args=(), device_types="cuda")
def gated_linrec_fwd(x: Tensor, gate_a: Tensor, gate_x: Tensor, rate: Tensor, h0: Optional[Tensor], cu_seqlens: Optional[Tensor],
                     reverse: bool, scale: float) -> Tuple[Tensor, Tensor, Tensor]:
    return _layers.gated_fwd(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale, True)[:3]


@torch.library.custom_op("linrec_amd::gated_linrec_bwd", mutates_args=(), device_types="cuda")
def gated_linrec_bwd(d_h: Tensor, d_state: Tensor, x: Tensor, gate_a: Tensor, gate_x: Tensor, rate: Tensor, h0: Optional[Tensor],
                     cu_seqlens: Optional[Tensor], saved: Tensor, reverse: bool,
                     scale: float) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    *grads, d_h0 = _layers.gated_bwd(d_h, d_state, x, gate_a, gate_x, rate, h0, cu_seqlens, saved, reverse, scale)
    return (*grads, rate.new_empty(0) if d_h0 is None else d_h0)


@gated_linrec_fwd.register_fake
def _(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale):
    batch, time, channels, sequences = _layers.gated_shape(x, cu_seqlens)
    torch._check(gate_a.size() == x.size() and gate_x.size() == x.size(), lambda: "gated_linrec: x, gate_a and gate_x differ in size")
    return (x.new_empty(x.size()), x.new_empty((sequences, channels), dtype=torch.float32),
            x.new_empty(_layers.gated_saved_numel(x.dtype, batch, time, channels), dtype=torch.float32))


@gated_linrec_bwd.register_fake
def _(d_h, d_state, x, gate_a, gate_x, rate, h0, cu_seqlens, saved, reverse, scale):
    return (*(x.new_empty(x.size()) for _ in range(3)), rate.new_empty(rate.size()),
            rate.new_empty(0) if h0 is None else rate.new_empty(h0.size()))


def _gated_setup(ctx, inputs, output):
    x, gate_a, gate_x, rate, h0, cu_seqlens, ctx.reverse, ctx.scale = inputs
    ctx.save_for_backward(x, gate_a, gate_x, rate, h0, cu_seqlens, output[2])


def _gated_backward(ctx, d_h, d_state, _):
    *inputs, saved = ctx.saved_tensors
    *grads, d_h0 = gated_linrec_bwd(d_h, d_state, *inputs, saved, ctx.reverse, ctx.scale)
    return (*grads, None if inputs[4] is None else d_h0, None, None, None)


torch.library.register_autograd("linrec_amd::gated_linrec_fwd", _gated_backward, setup_context=_gated_setup)


class _GatedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale, with_state):
        h, state, saved, ctx.number = _layers.gated_fwd(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale, True, with_state)
        ctx.save_for_backward(x, gate_a, gate_x, rate, h0, cu_seqlens, saved)
        ctx.set_materialize_grads(False)
        ctx.reverse, ctx.scale = reverse, scale
        return (h, state) if with_state else h

    @staticmethod
    @_once
    def backward(ctx, d_h, d_state=None):
        x, gate_a, gate_x, rate, h0, cu_seqlens, saved = ctx.saved_tensors
        return (*_layers.gated_bwd(d_h, d_state, x, gate_a, gate_x, rate, h0, cu_seqlens, saved, ctx.reverse, ctx.scale, ctx.number),
                None, None, None, None)


def gated_linrec(x: Tensor, gate_a: Tensor, gate_x: Tensor, rate: Tensor, *, h0: Optional[Tensor] = None,
                 cu_seqlens: Optional[Tensor] = None, reverse: bool = False, scale: float = 8.0, return_state: bool = False):
    """Gated linear recurrence over the time axis of (batch, time, channels) activations:

        log a[t] = -scale * softplus(rate) * sigmoid(gate_a[t])
        h[t] = a[t] * h[t-1] + sqrt(1 - a[t]^2) * sigmoid(gate_x[t]) * x[t]

    x, gate_a and gate_x are of one size and one storage type (float32, float16, bfloat16) and may be strided (chunks of one
    projection); rate, (channels), and h0, (batch, channels), the value before the first position, are float32.  `reverse`
    runs from the last position to the first.  With cu_seqlens, int32 bounds (sequences + 1) on the device, x is
    (positions, channels): sequences side by side, none of which sees another; h0 then has a row per sequence.
    Returns h, or (h, state) with return_state, the float32 value that leaves each sequence: what h0 of the following
    positions or gated_linrec_step goes on from.  Differentiable in x, gate_a, gate_x, rate and h0.
    """
    scale = float(scale)
    _refuse_tangents("gated_linrec", x, gate_a, gate_x, rate, h0)
    if _traced(x, gate_a, gate_x, rate, h0):
        h, state, _ = gated_linrec_fwd(x, gate_a, gate_x, rate, h0, cu_seqlens, bool(reverse), scale)
    elif _recorded(x, gate_a, gate_x, rate, h0):
        return _GatedFn.apply(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale, return_state)
    else:
        h, state, *_ = _layers.gated_fwd(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale, False, return_state)
    return (h, state) if return_state else h


@torch.library.custom_op("linrec_amd::gated_linrec_step", mutates_args=("state",), device_types="cuda")
def _gated_linrec_step(x: Tensor, gate_a: Tensor, gate_x: Tensor, rate: Tensor, state: Tensor, slots: Optional[Tensor],
                       scale: float) -> Tensor:
    return _layers.gated_step(x, gate_a, gate_x, rate, state, slots, scale)


@_gated_linrec_step.register_fake
def _(x, gate_a, gate_x, rate, state, slots, scale):
    return x.new_empty(x.size())


def gated_linrec_step(x: Tensor, gate_a: Tensor, gate_x: Tensor, rate: Tensor, state: Tensor, *, slots: Optional[Tensor] = None,
                      scale: float = 8.0) -> Tensor:
    """One position of gated_linrec for a batch of rows, for serving: x, gate_a and gate_x are (batch, channels), `state`
    (rows, channels) float32 holds the values before this position and is updated in place.  `slots` (int32, on the device)
    names the row of `state` that each row of x uses; a row whose slot is negative or not in `state` takes no part: its
    result is zero.  No row of `state` may be named twice.  Records no gradient, in neither direction.
    """
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, gate_a, gate_x, rate, state)):
        raise RuntimeError("gated_linrec_step: records no gradient; call it under torch.no_grad(), or gated_linrec for training")
    _refuse_tangents("gated_linrec_step", x, gate_a, gate_x, rate, state)
    if _traced(x, gate_a, gate_x, rate, state):
        return _gated_linrec_step(x, gate_a, gate_x, rate, state, slots, float(scale))
    h = _layers.gated_step(x, gate_a, gate_x, rate, state, slots, float(scale))
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)  # (as the registered operator does: whoever saved `state` has to know)
    return h


# ---- group norm with an activation -------------------------------------------------------------
@torch.library.custom_op("linrec_amd::group_norm_act_fwd", mutates_args=(), device_types="cuda")
def group_norm_act_fwd(x: Tensor, groups: int, weight: Optional[Tensor], bias: Optional[Tensor], eps: float,
                       act: str) -> Tuple[Tensor, Tensor]:
    return _layers.norm_fwd(x, groups, weight, bias, eps, act)[:2]


@torch.library.custom_op("linrec_amd::group_norm_act_bwd", mutates_args=(), device_types="cuda")
def group_norm_act_bwd(d_y: Tensor, x: Tensor, groups: int, weight: Optional[Tensor], bias: Optional[Tensor], stats: Tensor,
                       eps: float, act: str) -> Tuple[Tensor, Tensor, Tensor]:
    d_x, d_weight, d_bias = _layers.norm_bwd(d_y, x, groups, weight, bias, stats, eps, act)
    return (d_x, stats.new_empty(0), stats.new_empty(0)) if weight is None else (d_x, d_weight, d_bias)


@group_norm_act_fwd.register_fake
def _(x, groups, weight, bias, eps, act):
    torch._check(x.dim() >= 2 and x.size(-1) % groups == 0, lambda: "group_norm_act: channels cannot be cut into groups")
    return x.new_empty(x.size()), x.new_empty((2, x.size(0), groups), dtype=torch.float32)


@group_norm_act_bwd.register_fake
def _(d_y, x, groups, weight, bias, stats, eps, act):
    params = [stats.new_empty(0) if weight is None else weight.new_empty(weight.size()) for _ in range(2)]
    return (x.new_empty(x.size()), *params)


def _norm_setup(ctx, inputs, output):
    x, ctx.groups, weight, bias, ctx.eps, ctx.act = inputs
    ctx.save_for_backward(x, weight, bias, output[1])


def _norm_backward(ctx, d_y, _):
    x, weight, bias, stats = ctx.saved_tensors
    d_x, d_weight, d_bias = group_norm_act_bwd(d_y, x, ctx.groups, weight, bias, stats, ctx.eps, ctx.act)
    if weight is None:
        d_weight = d_bias = None
    return d_x, None, d_weight, d_bias, None, None


torch.library.register_autograd("linrec_amd::group_norm_act_fwd", _norm_backward, setup_context=_norm_setup)


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, groups, weight, bias, eps, act):
        y, stats, ctx.number = _layers.norm_fwd(x, groups, weight, bias, eps, act)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.groups, ctx.eps, ctx.act = groups, eps, act
        return y

    @staticmethod
    @_once
    def backward(ctx, d_y):
        x, weight, bias, stats = ctx.saved_tensors
        d_x, d_weight, d_bias = _layers.norm_bwd(d_y, x, ctx.groups, weight, bias, stats, ctx.eps, ctx.act, ctx.number)
        return d_x, None, d_weight, d_bias, None, None


def group_norm_act(x: Tensor, groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, *, eps: float = 1e-5,
                   act: str = "silu") -> Tensor:
    """act(group_norm(x)) for channels-last x, (batch, ..., channels): the channels are cut into `groups` equal runs, mean and
    variance are taken over the run and everything between the first and the last dimension.  A norm for each token is that of
    (tokens, channels).  weight and bias, (channels), both or none, float32 or of x's type; act is "none", "relu", "silu" or
    "gelu" (the exact one).  Statistics are float32.  Differentiable in x, weight and bias.
    """
    groups, eps = int(groups), float(eps)
    _refuse_tangents("group_norm_act", x, weight, bias)
    if _traced(x, weight, bias):
        return group_norm_act_fwd(x, groups, weight, bias, eps, act)[0]
    if _recorded(x, weight, bias):
        return _NormFn.apply(x, groups, weight, bias, eps, act)
    return _layers.norm_fwd(x, groups, weight, bias, eps, act)[0]


# ---- root-mean-square norm ---------------------------------------------------------------------
@torch.library.custom_op("linrec_amd::rms_norm_fwd", mutates_args=(), device_types="cuda")
def rms_norm_fwd(x: Tensor, weight: Optional[Tensor], residual: Optional[Tensor], eps: float) -> Tuple[Tensor, Tensor, Tensor]:
    y, total, rstd, _ = _layers.rms_fwd(x, weight, residual, eps)
    return y, x.new_empty(0) if total is None else total, rstd


@torch.library.custom_op("linrec_amd::rms_norm_bwd", mutates_args=(), device_types="cuda")
def rms_norm_bwd(d_y: Tensor, d_total: Optional[Tensor], x: Tensor, weight: Optional[Tensor], rstd: Tensor,
                 eps: float) -> Tuple[Tensor, Tensor]:
    d_x, d_weight = _layers.rms_bwd(d_y, d_total, x, weight, rstd, eps)
    return d_x, rstd.new_empty(0) if d_weight is None else d_weight


@torch.library.custom_op("linrec_amd::rms_norm_quantize", mutates_args=(), device_types="cuda")
def _rms_norm_quantize(x: Tensor, weight: Optional[Tensor], residual: Optional[Tensor], eps: float,
                       dtype: torch.dtype) -> Tuple[Tensor, Tensor, Tensor]:
    q, total, scales, _ = _layers.rms_fwd(x, weight, residual, eps, dtype)
    return q, scales, x.new_empty(0) if total is None else total


@rms_norm_fwd.register_fake
def _(x, weight, residual, eps):
    return (x.new_empty(x.size()), x.new_empty(0 if residual is None else x.size()), x.new_empty(x.size()[:-1], dtype=torch.float32))


@rms_norm_bwd.register_fake
def _(d_y, d_total, x, weight, rstd, eps):
    return x.new_empty(x.size()), rstd.new_empty(0) if weight is None else weight.new_empty(weight.size())


@_rms_norm_quantize.register_fake
def _(x, weight, residual, eps, dtype):
    return (x.new_empty(x.size(), dtype=dtype), x.new_empty(x.size()[:-1], dtype=torch.float32), x.new_empty(0 if residual is None else x.size()))


def _rms_setup(ctx, inputs, output):
    x, weight, residual, ctx.eps = inputs
    ctx.with_residual = residual is not None
    ctx.save_for_backward(output[1] if ctx.with_residual else x, weight, output[2])


def _rms_backward(ctx, d_y, d_total, _):
    x, weight, rstd = ctx.saved_tensors
    d_x, d_weight = rms_norm_bwd(d_y, d_total if ctx.with_residual else None, x, weight, rstd, ctx.eps)
    return d_x, None if weight is None else d_weight, d_x if ctx.with_residual else None, None


torch.library.register_autograd("linrec_amd::rms_norm_fwd", _rms_backward, setup_context=_rms_setup)


class _RmsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, total, rstd, ctx.number = _layers.rms_fwd(x, weight, residual, eps)
        ctx.save_for_backward(x if total is None else total, weight, rstd)
        ctx.set_materialize_grads(False)
        ctx.eps, ctx.with_residual = eps, residual is not None
        return y if total is None else (y, total)

    @staticmethod
    @_once
    def backward(ctx, d_y, d_total=None):
        x, weight, rstd = ctx.saved_tensors
        d_x, d_weight = _layers.rms_bwd(d_y, d_total, x, weight, rstd, ctx.eps, ctx.number)
        return d_x, d_weight, d_x if ctx.with_residual else None, None


def rms_norm(x: Tensor, weight: Optional[Tensor] = None, *, residual: Optional[Tensor] = None, eps: float = 1e-6):
    """x * weight / sqrt(mean(x^2) + eps) over the last dimension of x, (..., channels) with up to 16384 channels.  With a residual, of x's
    size and type, x + residual is normalised instead, rounded to that type, and returned as well: (y, total), total being what
    the next layer's residual is.  weight, (channels), is float32 or of x's type, ones if None.  Sums are float32.
    Differentiable in x, weight and residual.
    """
    eps = float(eps)
    _refuse_tangents("rms_norm", x, weight, residual)
    if _traced(x, weight, residual):
        y, total, _ = rms_norm_fwd(x, weight, residual, eps)
    elif _recorded(x, weight, residual):
        return _RmsFn.apply(x, weight, residual, eps)
    else:
        y, total, *_ = _layers.rms_fwd(x, weight, residual, eps, None, False)
    return y if residual is None else (y, total)


def rms_norm_quantize(x: Tensor, weight: Optional[Tensor] = None, *, residual: Optional[Tensor] = None, eps: float = 1e-6,
                      dtype: torch.dtype = torch.int8):
    """rms_norm with an output in 8 bits, for a product in 8 bits: (q, scales), or (q, scales, total) with a residual.  q is int8 or
    float8_e4m3fn of x's size, scales (float32, x's size without channels) one a row, its largest |y| over 127 or 448: the norm is
    q * scales[..., None].  A row of zeros has the scale 0; one whose norm is not finite has NaN, and zeros for values.
    Records no gradient, in neither direction.
    """
    eps = float(eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_quantize: records no gradient; call it under torch.no_grad(), or rms_norm for training")
    _refuse_tangents("rms_norm_quantize", x, weight, residual)
    if dtype is None:
        raise RuntimeError("rms_norm_quantize: dtype must be torch.int8 or torch.float8_e4m3fn, got None")
    if _traced(x, weight, residual):
        q, scales, total = _rms_norm_quantize(x, weight, residual, eps, dtype)
    else:
        q, total, scales, _ = _layers.rms_fwd(x, weight, residual, eps, dtype)
    return (q, scales) if residual is None else (q, scales, total)


# ---- embedding ---------------------------------------------------------------------------------
@torch.library.custom_op("linrec_amd::embedding_fwd", mutates_args=(), device_types="cuda")
def embedding_fwd(tokens: Tensor, weight: Tensor, scale: float, padding_idx: Optional[int]) -> Tensor:
    return _layers.embedding_fwd(tokens, weight, scale, padding_idx)[0]


@torch.library.custom_op("linrec_amd::embedding_bwd", mutates_args=(), device_types="cuda")
def embedding_bwd(d_y: Tensor, tokens: Tensor, weight: Tensor, scale: float, padding_idx: Optional[int]) -> Tensor:
    return _layers.embedding_bwd(d_y, tokens, weight, scale, padding_idx)


@embedding_fwd.register_fake
def _(tokens, weight, scale, padding_idx):
    return weight.new_empty((*tokens.size(), weight.size(1)))


@embedding_bwd.register_fake
def _(d_y, tokens, weight, scale, padding_idx):
    return weight.new_empty(weight.size())


def _embedding_setup(ctx, inputs, output):
    tokens, weight, ctx.scale, ctx.padding_idx = inputs
    ctx.save_for_backward(tokens, weight)


def _embedding_backward(ctx, d_y):
    tokens, weight = ctx.saved_tensors
    return None, embedding_bwd(d_y, tokens, weight, ctx.scale, ctx.padding_idx), None, None


torch.library.register_autograd("linrec_amd::embedding_fwd", _embedding_backward, setup_context=_embedding_setup)


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx):
        ctx.save_for_backward(tokens)
        ctx.like, ctx.scale, ctx.padding_idx = weight, scale, padding_idx  # (its sizes; the values are not read again)
        y, ctx.number = _layers.embedding_fwd(tokens, weight, scale, padding_idx)
        return y

    @staticmethod
    @_once
    def backward(ctx, d_y):
        return None, _layers.embedding_bwd(d_y, ctx.saved_tensors[0], ctx.like, ctx.scale, ctx.padding_idx, ctx.number), None, None


def embedding(tokens: Tensor, weight: Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """scale * weight[tokens], (*tokens.shape, channels), for int32 or int64 tokens and a (vocabulary, channels) table.  The
    gradient of the table is dense; each of its rows is summed in float32 and rounded once, the same in every run.  A token
    outside the table gives a row of zeros and no gradient; the row `padding_idx` is looked up but gets no gradient.
    """
    scale = float(scale)
    _refuse_tangents("embedding", weight)
    if _traced(tokens, weight):
        return embedding_fwd(tokens, weight, scale, padding_idx)
    if _recorded(weight):
        return _EmbeddingFn.apply(tokens, weight, scale, padding_idx)
    return _layers.embedding_fwd(tokens, weight, scale, padding_idx)[0]
