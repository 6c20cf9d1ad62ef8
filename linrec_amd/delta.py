"""The gated delta rule, a linear recurrence whose state is a matrix, and its single-token step.

As in layers.py each operator is a torch.library custom op (fake function, autograd rule) for tracing and compilation, and an
equivalent autograd Function, or a plain call where no gradient is recorded, in eager mode.  Device tensors only.
"""
from typing import Optional, Tuple

import torch

from . import _delta
from .layers import _once, _recorded, _refuse_tangents, _traced

__all__ = ["gated_delta", "gated_delta_step"]

Tensor = torch.Tensor


@torch.library.custom_op("linrec_amd::gated_delta_fwd", mutates_args=(), device_types="cuda")
def gated_delta_fwd(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, h0: Optional[Tensor], cu_seqlens: Optional[Tensor],
                    scale: float) -> Tuple[Tensor, Tensor]:
    return _delta.delta_fwd(q, k, v, log_decay, beta, h0, cu_seqlens, scale)[:2]


@torch.library.custom_op("linrec_amd::gated_delta_bwd", mutates_args=(), device_types="cuda")
def gated_delta_bwd(d_o: Tensor, d_state: Tensor, q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, h0: Optional[Tensor],
                    cu_seqlens: Optional[Tensor], scale: float) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    *grads, d_h0 = _delta.delta_bwd(d_o, d_state, q, k, v, log_decay, beta, h0, cu_seqlens, scale)
    return (*grads, beta.new_empty(0) if d_h0 is None else d_h0)


@gated_delta_fwd.register_fake
def _(q, k, v, log_decay, beta, h0, cu_seqlens, scale):
    sequences = _delta.delta_shape(q, cu_seqlens)[2]
    torch._check(k.size() == q.size(), lambda: "gated_delta: q and k differ in size")
    return v.new_empty(v.size()), v.new_empty((sequences, v.size(-2), q.size(-1), v.size(-1)), dtype=torch.float32)


@gated_delta_bwd.register_fake
def _(d_o, d_state, q, k, v, log_decay, beta, h0, cu_seqlens, scale):
    return (*(t.new_empty(t.size()) for t in (q, k, v, log_decay, beta)), beta.new_empty(0) if h0 is None else h0.new_empty(h0.size()))


def _delta_setup(ctx, inputs, output):
    *tensors, ctx.scale = inputs
    ctx.save_for_backward(*tensors)


def _delta_backward(ctx, d_o, d_state):
    inputs = ctx.saved_tensors
    *grads, d_h0 = gated_delta_bwd(d_o, d_state, *inputs, ctx.scale)
    return (*grads, None if inputs[5] is None else d_h0, None, None)


torch.library.register_autograd("linrec_amd::gated_delta_fwd", _delta_backward, setup_context=_delta_setup)


class _DeltaFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, beta, h0, cu_seqlens, scale, with_state):
        o, state, ctx.number = _delta.delta_fwd(q, k, v, log_decay, beta, h0, cu_seqlens, scale, with_state)
        ctx.save_for_backward(q, k, v, log_decay, beta, h0, cu_seqlens)
        ctx.set_materialize_grads(False)
        ctx.scale = scale
        return (o, state) if with_state else o

    @staticmethod
    @_once
    def backward(ctx, d_o, d_state=None):
        return (*_delta.delta_bwd(d_o, d_state, *ctx.saved_tensors, ctx.scale, ctx.number), None, None, None)


def gated_delta(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, *, h0: Optional[Tensor] = None,
                cu_seqlens: Optional[Tensor] = None, scale: Optional[float] = None, return_state: bool = False):
    """Gated delta rule over the time axis: every head has a matrix S, (key_dim, value_dim), as its state, and at each position

        S = exp(log_decay) * S
        S = S + outer(k, beta * (v - S.T @ k))
        o = scale * S.T @ q

    q and k are (batch, time, key_heads, key_dim), v is (batch, time, heads, value_dim), of one storage type (float32, float16,
    bfloat16) and strided as they may be (parts of one projection); log_decay and beta, (batch, time, heads), are float32.
    `heads` is a multiple of key_heads: neighbouring value heads share a key head.  key_dim is at most 256; keys are expected to
    be of about unit length (rms_norm of each head) and log_decay not above zero, or the states grow.  scale is key_dim ** -0.5
    unless given.  h0, (batch, heads, key_dim, value_dim) float32, is S before the first position.  With cu_seqlens, int32 bounds
    (sequences + 1) on the device, the tensors are (positions, heads, ...): sequences side by side, none of which sees another;
    h0 then has a row per sequence.

    Returns o, of v's size, or (o, state) with return_state, the float32 S that leaves each sequence: what h0 of the following
    positions or gated_delta_step goes on from.  Differentiable in q, k, v, log_decay, beta and h0.
    """
    scale = q.size(-1) ** -0.5 if scale is None else float(scale)
    _refuse_tangents("gated_delta", q, k, v, log_decay, beta, h0)
    if _traced(q, k, v, log_decay, beta, h0):
        o, state = gated_delta_fwd(q, k, v, log_decay, beta, h0, cu_seqlens, scale)
    elif _recorded(q, k, v, log_decay, beta, h0):
        return _DeltaFn.apply(q, k, v, log_decay, beta, h0, cu_seqlens, scale, return_state)
    else:
        o, state, _ = _delta.delta_fwd(q, k, v, log_decay, beta, h0, cu_seqlens, scale, return_state)
    return (o, state) if return_state else o


@torch.library.custom_op("linrec_amd::gated_delta_step", mutates_args=("state",), device_types="cuda")
def _gated_delta_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, state: Tensor, slots: Optional[Tensor],
                      scale: float) -> Tensor:
    return _delta.delta_step(q, k, v, log_decay, beta, state, slots, scale)


@_gated_delta_step.register_fake
def _(q, k, v, log_decay, beta, state, slots, scale):
    return v.new_empty(v.size())


def gated_delta_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, state: Tensor, *, slots: Optional[Tensor] = None,
                     scale: Optional[float] = None) -> Tensor:
    """One position of gated_delta for a batch of rows, for serving: q and k are (batch, key_heads, key_dim), v is (batch, heads,
    value_dim), log_decay and beta (batch, heads); `state`, (rows, heads, key_dim, value_dim) float32, holds the states before
    this position and is updated in place.  `slots` (int32, on the device) names the row of `state` that each row uses; a row
    whose slot is negative or not in `state` takes no part: its result is zero.  No row of `state` may be named twice.  Records
    no gradient, in neither direction.
    """
    tensors = (q, k, v, log_decay, beta, state)
    scale = q.size(-1) ** -0.5 if scale is None else float(scale)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("gated_delta_step: records no gradient; call it under torch.no_grad(), or gated_delta for training")
    _refuse_tangents("gated_delta_step", *tensors)
    if _traced(*tensors):
        return _gated_delta_step(q, k, v, log_decay, beta, state, slots, scale)
    o = _delta.delta_step(q, k, v, log_decay, beta, state, slots, scale)
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)  # (as the registered operator does: whoever saved `state` has to know)
    return o
