"""ctypes binding of include/linrec_layers.h: argument checks, allocation of results and scratch with torch, one library call.

Device tensors only: there is no host form of these operators, and no fallback.
"""
import ctypes

import torch

from . import _native
from ._native import DTYPES, _on_device, check, lib

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}  # LINREC_ACT_*

_i32, _i64, _f32, _ptr, _u64 = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p, ctypes.c_uint64
_pair = _i64 * 2


class Gated(ctypes.Structure):
    """linrec_gated_t"""
    _fields_ = [("dtype", _i32), ("reverse", _i32), ("scale", _f32), ("reserved", _i32), ("batch", _i64), ("time", _i64),
                ("channels", _i64), ("sequences", _i64), ("cu_seqlens", _ptr), ("x", _ptr), ("gate_a", _ptr), ("gate_x", _ptr),
                ("x_stride", _pair), ("gate_a_stride", _pair), ("gate_x_stride", _pair), ("rate", _ptr), ("h0", _ptr), ("h", _ptr),
                ("state", _ptr), ("saved", _ptr), ("d_h", _ptr), ("d_h_stride", _pair), ("d_state", _ptr), ("d_x", _ptr),
                ("d_gate_a", _ptr), ("d_gate_x", _ptr), ("d_rate", _ptr), ("d_h0", _ptr), ("partial", _ptr), ("workspace", _ptr),
                ("workspace_bytes", _u64), ("stream", _ptr)]


class GatedStep(ctypes.Structure):
    """linrec_gated_step_t"""
    _fields_ = [("dtype", _i32), ("scale", _f32), ("batch", _i64), ("channels", _i64), ("slots_total", _i64), ("x_stride", _i64),
                ("gate_a_stride", _i64), ("gate_x_stride", _i64), ("state_stride", _i64), ("x", _ptr), ("gate_a", _ptr),
                ("gate_x", _ptr), ("rate", _ptr), ("slots", _ptr), ("state", _ptr), ("h", _ptr), ("stream", _ptr)]


class GroupNorm(ctypes.Structure):
    """linrec_group_norm_t"""
    _fields_ = [("dtype", _i32), ("weight_dtype", _i32), ("act", _i32), ("eps", _f32), ("batch", _i64), ("positions", _i64),
                ("channels", _i64), ("groups", _i64), ("x", _ptr), ("x_stride", _pair), ("weight", _ptr), ("bias", _ptr), ("y", _ptr),
                ("mean", _ptr), ("rstd", _ptr), ("d_y", _ptr), ("d_y_stride", _pair), ("d_x", _ptr), ("d_weight", _ptr),
                ("d_bias", _ptr), ("partial", _ptr), ("stream", _ptr)]


class Embedding(ctypes.Structure):
    """linrec_embedding_t"""
    _fields_ = [("dtype", _i32), ("token_bytes", _i32), ("scale", _f32), ("reserved", _i32), ("tokens", _i64), ("vocab", _i64),
                ("channels", _i64), ("padding", _i64), ("token", _ptr), ("weight", _ptr), ("y", _ptr), ("d_y", _ptr),
                ("d_y_stride", _i64), ("d_weight", _ptr), ("scratch", _ptr), ("scratch_bytes", _u64), ("stream", _ptr)]


EXPORTS = {
    "linrec_gated_saved_floats": (_i64, [_i64] * 3),
    "linrec_gated_partial_floats": (_i64, [_i64] * 3),
    "linrec_gated_workspace_bytes": (ctypes.c_size_t, [ctypes.c_int, _i64, _i64, _i64, ctypes.c_int]),
    "linrec_gated_fwd": (ctypes.c_int, [ctypes.POINTER(Gated)]),
    "linrec_gated_bwd": (ctypes.c_int, [ctypes.POINTER(Gated)]),
    "linrec_gated_step": (ctypes.c_int, [ctypes.POINTER(GatedStep)]),
    "linrec_group_norm_partial_floats": (_i64, [ctypes.c_int] + [_i64] * 4 + [ctypes.c_int]),
    "linrec_group_norm_fwd": (ctypes.c_int, [ctypes.POINTER(GroupNorm)]),
    "linrec_group_norm_bwd": (ctypes.c_int, [ctypes.POINTER(GroupNorm)]),
    "linrec_embedding_scratch_bytes": (ctypes.c_size_t, [_i64] * 3),
    "linrec_embedding_fwd": (ctypes.c_int, [ctypes.POINTER(Embedding)]),
    "linrec_embedding_bwd": (ctypes.c_int, [ctypes.POINTER(Embedding)]),
}


def _declare():
    handle = lib()
    for name, (result, arguments) in EXPORTS.items():
        fn = getattr(handle, name)
        fn.restype, fn.argtypes = result, arguments
    return handle


_lib = _declare()


def _call(t, fn, args, what):
    """fn(args) on t's device and current stream."""
    def go(stream):
        args.stream = stream
        return fn(ctypes.byref(args))
    rc = _on_device(t, go)
    if rc:
        check(rc, what)


def _need(condition, message):
    if not condition:
        raise RuntimeError(message)


def _unit_channels(t):
    """`t` if its last dimension has unit stride, else a dense copy."""
    return t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous()


def _p(t):
    return None if t is None else t.data_ptr()


# ---- gated linear recurrence -------------------------------------------------------------------
def _check_activations(what, x, *others, names):
    _need(x.dtype in DTYPES, f"{what}: x must be float32, float16 or bfloat16, got {x.dtype}")
    _need(x.is_cuda, f"{what}: needs device tensors, x is on {x.device}")
    for t, name in zip(others, names):
        _need(t.size() == x.size(), f"{what}: {name} has size {tuple(t.size())}, x has {tuple(x.size())}")
        _need(t.device == x.device, f"{what}: {name} is on {t.device}, x on {x.device}")
        _need(t.dtype == x.dtype, f"{what}: {name} has dtype {t.dtype}, x has {x.dtype}")


def _check_fp32(what, t, name, shape, device):
    _need(t.dtype == torch.float32, f"{what}: {name} must be float32, got {t.dtype}")
    _need(tuple(t.size()) == tuple(shape), f"{what}: {name} has size {tuple(t.size())}, expected {tuple(shape)}")
    _need(t.device == device, f"{what}: {name} is on {t.device}, x on {device}")


def gated_shape(x, cu_seqlens):
    """(batch, time, channels, sequences) of a call; raises if the dimensions do not fit."""
    if cu_seqlens is None:
        _need(x.dim() == 3, f"gated_linrec: x must be (batch, time, channels), got {x.dim()} dimensions")
        return x.size(0), x.size(1), x.size(2), x.size(0)
    _need(x.dim() == 2, f"gated_linrec: with cu_seqlens x must be (positions, channels), got {x.dim()} dimensions")
    _need(cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 1, "gated_linrec: cu_seqlens must be one-dimensional, sequences + 1 bounds")
    _need(cu_seqlens.dtype == torch.int32, f"gated_linrec: cu_seqlens must be int32, got {cu_seqlens.dtype}")
    _need(cu_seqlens.device == x.device, f"gated_linrec: cu_seqlens is on {cu_seqlens.device}, x on {x.device}")
    _need(cu_seqlens.numel() > 1 or x.size(0) == 0, "gated_linrec: positions but no sequence to hold them")
    return 1, x.size(0), x.size(1), cu_seqlens.numel() - 1


def _gated_args(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale):
    """(argument block with the inputs filled in, the tensors it points into)"""
    _check_activations("gated_linrec", x, gate_a, gate_x, names=("gate_a", "gate_x"))
    shape = gated_shape(x, cu_seqlens)
    _check_fp32("gated_linrec", rate, "rate", shape[2:3], x.device)
    if h0 is not None:
        _check_fp32("gated_linrec", h0, "h0", (shape[3], shape[2]), x.device)
        h0 = h0.contiguous()
    x, gate_a, gate_x, rate = _unit_channels(x), _unit_channels(gate_a), _unit_channels(gate_x), rate.contiguous()
    if cu_seqlens is not None:
        cu_seqlens = cu_seqlens.contiguous()
    a = Gated(dtype=DTYPES[x.dtype], reverse=int(bool(reverse)), scale=scale, batch=shape[0], time=shape[1], channels=shape[2],
              sequences=shape[3], cu_seqlens=_p(cu_seqlens), x=x.data_ptr(), gate_a=gate_a.data_ptr(), gate_x=gate_x.data_ptr(),
              rate=rate.data_ptr(), h0=_p(h0))
    for name, t in (("x_stride", x), ("gate_a_stride", gate_a), ("gate_x_stride", gate_x)):
        setattr(a, name, _time_strides(t))
    return a, (x, gate_a, gate_x, rate, h0, cu_seqlens)


def _time_strides(t):
    return _pair(t.stride(0), t.stride(1)) if t.dim() == 3 else _pair(0, t.stride(0))


def _gated_workspace(a, x, is_bwd):
    """Points `a` at the stream's workspace if the call needs one; returns what has to stay alive until it is enqueued."""
    need = _lib.linrec_gated_workspace_bytes(a.dtype, a.batch, a.time, a.channels, is_bwd)
    if not need:
        return None

    def go(stream):
        return _native.workspace(x.device, stream, need)
    ws = _on_device(x, go)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    return ws


def gated_saved_numel(batch, time, channels):
    return _lib.linrec_gated_saved_floats(batch, time, channels)


def gated_fwd(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale, save):
    """(h, state, saved); saved is None without `save`."""
    a, kept = _gated_args(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale)
    h = torch.empty(x.size(), dtype=x.dtype, device=x.device)
    state = torch.empty((a.sequences, a.channels), dtype=torch.float32, device=x.device)
    saved = None
    if save:
        saved = torch.empty(gated_saved_numel(a.batch, a.time, a.channels), dtype=torch.float32, device=x.device)
    a.h, a.state, a.saved = h.data_ptr(), state.data_ptr(), _p(saved)
    ws = _gated_workspace(a, x, 0)
    _call(x, _lib.linrec_gated_fwd, a, "gated_linrec")
    del kept, ws
    return h, state, saved


def gated_bwd(d_h, d_state, x, gate_a, gate_x, rate, h0, cu_seqlens, saved, reverse, scale):
    """(d_x, d_gate_a, d_gate_x, d_rate, d_h0); d_h0 is None without h0, d_h or d_state may be None (zeros)."""
    a, kept = _gated_args(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale)
    if d_h is None:
        d_h = torch.zeros((), dtype=x.dtype, device=x.device).expand(x.size())
    _check_activations("gated_linrec", x, d_h, names=("d_h",))
    d_h = _unit_channels(d_h)
    if d_state is not None:
        _check_fp32("gated_linrec", d_state, "d_state", (a.sequences, a.channels), x.device)
        d_state = d_state.contiguous()
    d_x, d_gate_a, d_gate_x = (torch.empty(x.size(), dtype=x.dtype, device=x.device) for _ in range(3))
    d_rate = torch.empty_like(rate, memory_format=torch.contiguous_format)
    d_h0 = None if h0 is None else torch.empty(h0.size(), dtype=torch.float32, device=x.device)
    partial = torch.empty(_lib.linrec_gated_partial_floats(a.batch, a.time, a.channels), dtype=torch.float32, device=x.device)
    a.d_h, a.d_h_stride, a.d_state, a.saved = d_h.data_ptr(), _time_strides(d_h), _p(d_state), saved.data_ptr()
    a.d_x, a.d_gate_a, a.d_gate_x, a.d_rate, a.d_h0 = d_x.data_ptr(), d_gate_a.data_ptr(), d_gate_x.data_ptr(), d_rate.data_ptr(), _p(d_h0)
    a.partial = partial.data_ptr()
    ws = _gated_workspace(a, x, 1)
    _call(x, _lib.linrec_gated_bwd, a, "gated_linrec")
    del kept, ws
    return d_x, d_gate_a, d_gate_x, d_rate, d_h0


def gated_step(x, gate_a, gate_x, rate, state, slots, scale):
    what = "gated_linrec_step"
    _check_activations(what, x, gate_a, gate_x, names=("gate_a", "gate_x"))
    _need(x.dim() == 2, f"{what}: x must be (batch, channels), got {x.dim()} dimensions")
    batch, channels = x.size()
    _check_fp32(what, rate, "rate", (channels,), x.device)
    _need(state.dim() == 2, f"{what}: state must be (rows, channels), got {state.dim()} dimensions")
    _check_fp32(what, state, "state", (state.size(0), channels), x.device)
    _need(channels <= 1 or state.stride(1) == 1, f"{what}: state is updated in place and needs channels of unit stride")
    _need(state.size(0) <= 1 or state.stride(0) >= channels, f"{what}: rows of state overlap in memory")
    if slots is None:
        _need(state.size(0) == batch, f"{what}: state has {state.size(0)} rows, x has {batch} (name the rows with slots)")
    else:
        _need(slots.dtype == torch.int32 and tuple(slots.size()) == (batch,),
              f"{what}: slots must be int32 of size ({batch},), got {slots.dtype} of {tuple(slots.size())}")
        _need(slots.device == x.device, f"{what}: slots is on {slots.device}, x on {x.device}")
        slots = slots.contiguous()
    x, gate_a, gate_x, rate = _unit_channels(x), _unit_channels(gate_a), _unit_channels(gate_x), rate.contiguous()
    h = torch.empty((batch, channels), dtype=x.dtype, device=x.device)
    a = GatedStep(DTYPES[x.dtype], scale, batch, channels, state.size(0), x.stride(0), gate_a.stride(0), gate_x.stride(0),
                  state.stride(0), x.data_ptr(), gate_a.data_ptr(), gate_x.data_ptr(), rate.data_ptr(), _p(slots), state.data_ptr(),
                  h.data_ptr())
    _call(x, _lib.linrec_gated_step, a, what)
    return h


# ---- group norm with an activation -------------------------------------------------------------
def _norm_args(x, groups, weight, bias, eps, act):
    what = "group_norm_act"
    _need(x.dtype in DTYPES, f"{what}: x must be float32, float16 or bfloat16, got {x.dtype}")
    _need(x.is_cuda, f"{what}: needs device tensors, x is on {x.device}")
    _need(x.dim() >= 2, f"{what}: x must be (batch, ..., channels), got {x.dim()} dimensions")
    channels = x.size(-1)
    _need(groups >= 1 and channels % groups == 0, f"{what}: {channels} channels cannot be cut into {groups} groups")
    _need(act in ACTIVATIONS, f"{what}: act must be one of {', '.join(ACTIVATIONS)}, got {act!r}")
    _need((weight is None) == (bias is None), f"{what}: weight and bias go together")
    a = GroupNorm(dtype=DTYPES[x.dtype], act=ACTIVATIONS[act], eps=eps, channels=channels, groups=groups, batch=x.size(0))
    if weight is not None:
        for t, name in ((weight, "weight"), (bias, "bias")):
            _need(tuple(t.size()) == (channels,), f"{what}: {name} has size {tuple(t.size())}, expected ({channels},)")
            _need(t.device == x.device, f"{what}: {name} is on {t.device}, x on {x.device}")
            _need(t.dtype == weight.dtype and t.dtype in (torch.float32, x.dtype),
                  f"{what}: weight and bias must both be float32 or both {x.dtype}, {name} has {t.dtype}")
        weight, bias = weight.contiguous(), bias.contiguous()
        a.weight, a.bias, a.weight_dtype = weight.data_ptr(), bias.data_ptr(), DTYPES[weight.dtype]
    positions = 1
    for n in x.shape[1:-1]:
        positions *= n
    a.positions = positions
    return a, weight, bias


def _positions_view(t, a):
    """`t` as (batch, positions, channels) with channels of unit stride, and its two strides."""
    t = _unit_channels(t)
    t = t.reshape(a.batch, a.positions, a.channels)
    return t, _pair(t.stride(0), t.stride(1))


def norm_fwd(x, groups, weight, bias, eps, act):
    """(y, mean, rstd)"""
    a, weight, bias = _norm_args(x, groups, weight, bias, eps, act)
    y = torch.empty(x.size(), dtype=x.dtype, device=x.device)
    mean, rstd = (torch.empty((a.batch, a.groups), dtype=torch.float32, device=x.device) for _ in range(2))
    v, a.x_stride = _positions_view(x, a)
    partial = torch.empty(_lib.linrec_group_norm_partial_floats(a.dtype, a.batch, a.positions, a.channels, a.groups, 0),
                          dtype=torch.float32, device=x.device)
    a.x, a.y, a.mean, a.rstd, a.partial = v.data_ptr(), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), partial.data_ptr()
    _call(x, _lib.linrec_group_norm_fwd, a, "group_norm_act")
    return y, mean, rstd


def norm_bwd(d_y, x, groups, weight, bias, mean, rstd, eps, act):
    """(d_x, d_weight, d_bias), the last two None without a weight"""
    a, weight, bias = _norm_args(x, groups, weight, bias, eps, act)
    _check_activations("group_norm_act", x, d_y, names=("d_y",))
    d_x = torch.empty(x.size(), dtype=x.dtype, device=x.device)
    d_weight, d_bias = (None, None) if weight is None else (torch.empty_like(weight), torch.empty_like(bias))
    v, a.x_stride = _positions_view(x, a)
    g, a.d_y_stride = _positions_view(d_y, a)
    partial = torch.empty(_lib.linrec_group_norm_partial_floats(a.dtype, a.batch, a.positions, a.channels, a.groups, 1),
                          dtype=torch.float32, device=x.device)
    a.x, a.d_y, a.mean, a.rstd, a.partial = v.data_ptr(), g.data_ptr(), mean.data_ptr(), rstd.data_ptr(), partial.data_ptr()
    a.d_x, a.d_weight, a.d_bias = d_x.data_ptr(), _p(d_weight), _p(d_bias)
    _call(x, _lib.linrec_group_norm_bwd, a, "group_norm_act")
    return d_x, d_weight, d_bias


# ---- embedding ---------------------------------------------------------------------------------
def _embedding_args(tokens, weight, scale, padding_idx):
    what = "embedding"
    _need(weight.dtype in DTYPES, f"{what}: weight must be float32, float16 or bfloat16, got {weight.dtype}")
    _need(weight.is_cuda, f"{what}: needs device tensors, weight is on {weight.device}")
    _need(weight.dim() == 2, f"{what}: weight must be (vocabulary, channels), got {weight.dim()} dimensions")
    _need(tokens.dtype in (torch.int32, torch.int64), f"{what}: tokens must be int32 or int64, got {tokens.dtype}")
    _need(tokens.device == weight.device, f"{what}: tokens are on {tokens.device}, weight on {weight.device}")
    vocab, channels = weight.size()
    if padding_idx is not None:
        _need(-vocab <= padding_idx < vocab, f"{what}: padding_idx {padding_idx} is not in a table of {vocab} rows")
        padding_idx %= vocab
    return Embedding(dtype=DTYPES[weight.dtype], token_bytes=tokens.element_size(), scale=scale, tokens=tokens.numel(), vocab=vocab,
                     channels=channels, padding=-1 if padding_idx is None else padding_idx)


def embedding_fwd(tokens, weight, scale, padding_idx):
    a = _embedding_args(tokens, weight, scale, padding_idx)
    y = torch.empty((*tokens.size(), weight.size(1)), dtype=weight.dtype, device=weight.device)
    tokens, weight = tokens.contiguous(), weight.contiguous()
    a.token, a.weight, a.y = tokens.data_ptr(), weight.data_ptr(), y.data_ptr()
    _call(weight, _lib.linrec_embedding_fwd, a, "embedding")
    return y


def embedding_bwd(d_y, tokens, weight, scale, padding_idx):
    """The gradient of `weight` (whose values are not read)."""
    a = _embedding_args(tokens, weight, scale, padding_idx)
    _need(tuple(d_y.size()) == (*tokens.size(), weight.size(1)), f"embedding: d_y has size {tuple(d_y.size())}")
    _need(d_y.dtype == weight.dtype and d_y.device == weight.device, f"embedding: d_y is {d_y.dtype} on {d_y.device}")
    d_weight = torch.empty(weight.size(), dtype=weight.dtype, device=weight.device)
    tokens = tokens.contiguous()
    d_y = _unit_channels(d_y).reshape(a.tokens, a.channels)
    scratch = torch.empty(_lib.linrec_embedding_scratch_bytes(a.tokens, a.vocab, a.channels), dtype=torch.uint8, device=weight.device)
    a.token, a.d_y, a.d_y_stride, a.d_weight = tokens.data_ptr(), d_y.data_ptr(), d_y.stride(0), d_weight.data_ptr()
    a.scratch, a.scratch_bytes = scratch.data_ptr(), scratch.numel()
    _call(weight, _lib.linrec_embedding_bwd, a, "embedding")
    return d_weight
