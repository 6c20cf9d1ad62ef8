"""ctypes binding of include/linrec_layers.h: argument checks, allocation of results and scratch with torch, one library call.

Device tensors only: there is no host form of these operators, and no fallback.

A call whose tensors look like an earlier call's (types, devices, sizes, strides; on this thread) skips the checks and fills
only the pointers of that call's argument block in: on small tensors the checks took longer than the kernels.
"""
import ctypes
import itertools
import threading

import torch

from . import _native
from ._native import DTYPES, _raw_stream, check, lib

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
    "linrec_gated_saved_floats": (_i64, [ctypes.c_int] + [_i64] * 3),
    "linrec_gated_partial_floats": (_i64, [ctypes.c_int] + [_i64] * 3),
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


# ---- remembered calls --------------------------------------------------------------------------
_memory = threading.local()
_REMEMBERED_MAX = 256


_numbers = itertools.count()


class _Entry:
    """What is known about calls of one kind: `args`, the argument block, and `ref`, a reference to it; `need`, bytes of
    workspace; `sizes`, of results and scratch; `number`, its own.  args is None where an input has to be copied into another
    layout first."""
    __slots__ = ("args", "ref", "need", "sizes", "number")

    def __init__(self, args=None, need=0, sizes=()):
        self.args, self.need, self.sizes, self.number = args, need, sizes, next(_numbers)
        self.ref = None if args is None else ctypes.byref(args)


def _remembered():
    table = getattr(_memory, "table", None)
    if table is None:
        table = _memory.table = {}
    return table


def _remember(key, entry):
    table = _remembered()
    if len(table) >= _REMEMBERED_MAX:
        table.clear()
    table[key] = entry
    return entry


def _looks(t):
    return None if t is None else (t.dtype, t.device, t.shape, t.stride())


def _stride(t):
    return None if t is None else t.stride()


def _call(t, fn, entry, what):
    """fn on the entry's arguments, on t's device and current stream."""
    index = t.device.index
    if torch.cuda.current_device() == index:
        rc = _enqueue(t, fn, entry, index)
    else:
        with torch.cuda.device(index):
            rc = _enqueue(t, fn, entry, index)
    if rc:
        check(rc, what)


def _enqueue(t, fn, entry, index):
    args = entry.args
    stream = args.stream = _raw_stream(index)
    if entry.need:
        ws = _native.workspace(t.device, stream, entry.need)
        args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    return fn(entry.ref)


def _floats(n, device):
    return torch.empty(n, dtype=torch.float32, device=device)


def _adjacent_channels(t):
    return t.stride(-1) == 1 or t.size(-1) <= 1 or t.numel() == 0


def _p(t):
    return None if t is None else t.data_ptr()


# ---- checks (of calls that are not remembered) --------------------------------------------------
def _check_device(what, t, name):
    if not t.is_cuda:
        raise RuntimeError(f"{what}: needs device tensors, {name} is on {t.device}")


def _check_activations(what, x, *others, names=()):
    if x.dtype not in DTYPES:
        raise RuntimeError(f"{what}: x must be float32, float16 or bfloat16, got {x.dtype}")
    _check_device(what, x, "x")
    for t, name in zip(others, names):
        if t.size() != x.size():
            raise RuntimeError(f"{what}: {name} has size {tuple(t.size())}, x has {tuple(x.size())}")
        if t.device != x.device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, x on {x.device}")
        if t.dtype != x.dtype:
            raise RuntimeError(f"{what}: {name} has dtype {t.dtype}, x has {x.dtype}")


def _check_fp32(what, t, name, shape, device):
    if t.dtype != torch.float32:
        raise RuntimeError(f"{what}: {name} must be float32, got {t.dtype}")
    if tuple(t.size()) != tuple(shape):
        raise RuntimeError(f"{what}: {name} has size {tuple(t.size())}, expected {tuple(shape)}")
    if t.device != device:
        raise RuntimeError(f"{what}: {name} is on {t.device}, x on {device}")


def gated_shape(x, cu_seqlens):
    """(batch, time, channels, sequences) of a call; raises if the dimensions do not fit."""
    what = "gated_linrec"
    if cu_seqlens is None:
        if x.dim() != 3:
            raise RuntimeError(f"{what}: x must be (batch, time, channels), got {x.dim()} dimensions")
        return x.size(0), x.size(1), x.size(2), x.size(0)
    if x.dim() != 2:
        raise RuntimeError(f"{what}: with cu_seqlens x must be (positions, channels), got {x.dim()} dimensions")
    if cu_seqlens.dim() != 1 or cu_seqlens.size(0) < 1:
        raise RuntimeError(f"{what}: cu_seqlens must be one-dimensional, sequences + 1 bounds")
    if cu_seqlens.dtype != torch.int32:
        raise RuntimeError(f"{what}: cu_seqlens must be int32, got {cu_seqlens.dtype}")
    if cu_seqlens.device != x.device:
        raise RuntimeError(f"{what}: cu_seqlens is on {cu_seqlens.device}, x on {x.device}")
    if cu_seqlens.size(0) == 1 and x.size(0) > 0:
        raise RuntimeError(f"{what}: positions but no sequence to hold them")
    return 1, x.size(0), x.size(1), cu_seqlens.size(0) - 1


# ---- gated linear recurrence -------------------------------------------------------------------
def _time_strides(t):
    return _pair(t.stride(0), t.stride(1)) if t.dim() == 3 else _pair(0, t.stride(0))


def _gated_args(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale, *gradients):
    """An argument block with everything but the pointers; None if a tensor has to be copied first."""
    _check_activations("gated_linrec", x, gate_a, gate_x, names=("gate_a", "gate_x"))
    batch, time, channels, sequences = gated_shape(x, cu_seqlens)
    _check_fp32("gated_linrec", rate, "rate", (channels,), x.device)
    if h0 is not None:
        _check_fp32("gated_linrec", h0, "h0", (sequences, channels), x.device)
    whole = all(t is None or t.is_contiguous() for t in (rate, h0, cu_seqlens))
    if not (whole and all(_adjacent_channels(t) for t in (x, gate_a, gate_x, *gradients))):
        return None
    return Gated(dtype=DTYPES[x.dtype], reverse=int(bool(reverse)), scale=scale, batch=batch, time=time, channels=channels,
                 sequences=sequences, x_stride=_time_strides(x), gate_a_stride=_time_strides(gate_a), gate_x_stride=_time_strides(gate_x))


def _dense(*tensors):
    return [t if t is None else t.contiguous() for t in tensors]


def _with_adjacent_channels(*tensors):
    return [t if _adjacent_channels(t) else t.contiguous() for t in tensors]


def gated_saved_numel(dtype, batch, time, channels):
    """linrec_gated_saved_floats, for sizes that may be symbols of a traced call."""
    every = (1 << 20) // _lib.linrec_gated_saved_floats(DTYPES[dtype], 1, 1 << 20, 1)
    return batch * ((time + every - 1) // every) * channels


# (A forward hands back the number of its kind of call as well, which stands for sizes, types, devices and options.  It says nothing
# of how what the backward reads lies in memory: a forward may have copied an input that the backward gets as it was, and hooks
# of saved tensors may give back another layout.  So a backward is looked up by that number and the strides of all that it reads.)
def gated_fwd(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale, save, with_state=True):
    """(h, state, saved, number); state is None without `with_state`, saved without `save`."""
    key = ("gated", x.dtype, x.device, x.shape, x.stride(), _looks(gate_a), _looks(gate_x), _looks(rate), _looks(h0), _looks(cu_seqlens),
           reverse, scale)
    e = _remembered().get(key)
    if e is None:
        a = _gated_args(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale)
        e = _remember(key, _Entry() if a is None else _Entry(
            a, _lib.linrec_gated_workspace_bytes(a.dtype, a.batch, a.time, a.channels, 0),
            ((a.sequences, a.channels), gated_saved_numel(x.dtype, a.batch, a.time, a.channels))))
    a = e.args
    if a is None:
        return gated_fwd(*_with_adjacent_channels(x, gate_a, gate_x), *_dense(rate, h0, cu_seqlens), reverse, scale, save, with_state)
    device = x.device
    h = torch.empty(x.shape, dtype=x.dtype, device=device)
    state = _floats(e.sizes[0], device) if with_state else None
    saved = _floats(e.sizes[1], device) if save else None
    a.x, a.gate_a, a.gate_x, a.rate = x.data_ptr(), gate_a.data_ptr(), gate_x.data_ptr(), rate.data_ptr()
    a.h0, a.cu_seqlens, a.h, a.state, a.saved = _p(h0), _p(cu_seqlens), h.data_ptr(), _p(state), _p(saved)
    _call(x, _lib.linrec_gated_fwd, e, "gated_linrec")
    return h, state, saved, e.number


def gated_bwd(d_h, d_state, x, gate_a, gate_x, rate, h0, cu_seqlens, saved, reverse, scale, number=None):
    """(d_x, d_gate_a, d_gate_x, d_rate, d_h0); d_h0 is None without h0, d_h or d_state may be None (zeros)."""
    if d_h is None:
        d_h = torch.zeros((), dtype=x.dtype, device=x.device).expand(x.size())
    if number is not None:
        key = (number, d_h.stride(), _stride(d_state), x.stride(), gate_a.stride(), gate_x.stride(), rate.stride(), _stride(h0), _stride(cu_seqlens))
    else:
        key = ("gated_bwd", x.dtype, x.device, x.shape, x.stride(), _looks(d_h), _looks(d_state), _looks(gate_a), _looks(gate_x), _looks(rate),
               _looks(h0), _looks(cu_seqlens), reverse, scale)
    e = _remembered().get(key)
    if e is None:
        a = _gated_args(x, gate_a, gate_x, rate, h0, cu_seqlens, reverse, scale, d_h)
        _check_activations("gated_linrec", x, d_h, names=("d_h",))
        if d_state is not None:
            batch, time, channels, sequences = gated_shape(x, cu_seqlens)
            _check_fp32("gated_linrec", d_state, "d_state", (sequences, channels), x.device)
        if a is None or not (d_state is None or d_state.is_contiguous()):
            e = _Entry()
        else:
            a.d_h_stride = _time_strides(d_h)
            e = _Entry(a, _lib.linrec_gated_workspace_bytes(a.dtype, a.batch, a.time, a.channels, 1),
                       (_lib.linrec_gated_partial_floats(a.dtype, a.batch, a.time, a.channels),))
        _remember(key, e)
    a = e.args
    if a is None:
        d_h, x, gate_a, gate_x = _with_adjacent_channels(d_h, x, gate_a, gate_x)
        d_state, rate, h0, cu_seqlens = _dense(d_state, rate, h0, cu_seqlens)
        return gated_bwd(d_h, d_state, x, gate_a, gate_x, rate, h0, cu_seqlens, saved, reverse, scale)
    device, shape, dtype = x.device, x.shape, x.dtype
    if not saved.is_contiguous():
        saved = saved.contiguous()
    d_x, d_gate_a, d_gate_x = (torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device),
                               torch.empty(shape, dtype=dtype, device=device))
    d_rate, partial = _floats(rate.shape, device), _floats(e.sizes[0], device)
    d_h0 = None if h0 is None else _floats(h0.shape, device)
    a.x, a.gate_a, a.gate_x, a.rate = x.data_ptr(), gate_a.data_ptr(), gate_x.data_ptr(), rate.data_ptr()
    a.h0, a.cu_seqlens, a.saved, a.d_h, a.d_state = _p(h0), _p(cu_seqlens), saved.data_ptr(), d_h.data_ptr(), _p(d_state)
    a.d_x, a.d_gate_a, a.d_gate_x, a.d_rate, a.d_h0 = d_x.data_ptr(), d_gate_a.data_ptr(), d_gate_x.data_ptr(), d_rate.data_ptr(), _p(d_h0)
    a.partial = partial.data_ptr()
    _call(x, _lib.linrec_gated_bwd, e, "gated_linrec")
    return d_x, d_gate_a, d_gate_x, d_rate, d_h0


def _step_args(x, gate_a, gate_x, rate, state, slots, scale):
    what = "gated_linrec_step"
    _check_activations(what, x, gate_a, gate_x, names=("gate_a", "gate_x"))
    if x.dim() != 2:
        raise RuntimeError(f"{what}: x must be (batch, channels), got {x.dim()} dimensions")
    batch, channels = x.size()
    _check_fp32(what, rate, "rate", (channels,), x.device)
    if state.dim() != 2:
        raise RuntimeError(f"{what}: state must be (rows, channels), got {state.dim()} dimensions")
    _check_fp32(what, state, "state", (state.size(0), channels), x.device)
    if not _adjacent_channels(state):
        raise RuntimeError(f"{what}: state is updated in place and needs channels of unit stride")
    if state.size(0) > 1 and state.stride(0) < channels:
        raise RuntimeError(f"{what}: rows of state overlap in memory")
    if slots is None:
        if state.size(0) != batch:
            raise RuntimeError(f"{what}: state has {state.size(0)} rows, x has {batch} (name the rows with slots)")
    elif slots.dtype != torch.int32 or tuple(slots.size()) != (batch,):
        raise RuntimeError(f"{what}: slots must be int32 of size ({batch},), got {slots.dtype} of {tuple(slots.size())}")
    elif slots.device != x.device:
        raise RuntimeError(f"{what}: slots is on {slots.device}, x on {x.device}")
    if not (rate.is_contiguous() and (slots is None or slots.is_contiguous()) and all(_adjacent_channels(t) for t in (x, gate_a, gate_x))):
        return None
    return GatedStep(dtype=DTYPES[x.dtype], scale=scale, batch=batch, channels=channels, slots_total=state.size(0), x_stride=x.stride(0),
                     gate_a_stride=gate_a.stride(0), gate_x_stride=gate_x.stride(0), state_stride=state.stride(0))


def gated_step(x, gate_a, gate_x, rate, state, slots, scale):
    key = ("step", x.dtype, x.device, x.shape, x.stride(), _looks(gate_a), _looks(gate_x), _looks(rate), _looks(state), _looks(slots), scale)
    e = _remembered().get(key)
    if e is None:
        e = _remember(key, _Entry(_step_args(x, gate_a, gate_x, rate, state, slots, scale)))
    a = e.args
    if a is None:
        return gated_step(*_with_adjacent_channels(x, gate_a, gate_x), *_dense(rate), state, *_dense(slots), scale)
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a.x, a.gate_a, a.gate_x, a.rate = x.data_ptr(), gate_a.data_ptr(), gate_x.data_ptr(), rate.data_ptr()
    a.slots, a.state, a.h = _p(slots), state.data_ptr(), h.data_ptr()
    _call(x, _lib.linrec_gated_step, e, "gated_linrec_step")
    return h


# ---- group norm with an activation -------------------------------------------------------------
def _norm_args(x, groups, weight, bias, eps, act):
    """An argument block with everything but the pointers and strides."""
    what = "group_norm_act"
    _check_activations(what, x)
    if x.dim() < 2:
        raise RuntimeError(f"{what}: x must be (batch, ..., channels), got {x.dim()} dimensions")
    channels = x.size(-1)
    if groups < 1 or channels % groups:
        raise RuntimeError(f"{what}: {channels} channels cannot be cut into {groups} groups")
    if act not in ACTIVATIONS:
        raise RuntimeError(f"{what}: act must be one of {', '.join(ACTIVATIONS)}, got {act!r}")
    if (weight is None) != (bias is None):
        raise RuntimeError(f"{what}: weight and bias go together")
    a = GroupNorm(dtype=DTYPES[x.dtype], act=ACTIVATIONS[act], eps=eps, channels=channels, groups=groups, batch=x.size(0), positions=1)
    for n in x.shape[1:-1]:
        a.positions *= n
    if weight is not None:
        for t, name in ((weight, "weight"), (bias, "bias")):
            if tuple(t.size()) != (channels,):
                raise RuntimeError(f"{what}: {name} has size {tuple(t.size())}, expected ({channels},)")
            if t.device != x.device:
                raise RuntimeError(f"{what}: {name} is on {t.device}, x on {x.device}")
            if t.dtype != weight.dtype or t.dtype not in (torch.float32, x.dtype):
                raise RuntimeError(f"{what}: weight and bias must both be float32 or both {x.dtype}, {name} has {t.dtype}")
        a.weight_dtype = DTYPES[weight.dtype]
    return a


def _positions_stride(t, a):
    """(batch, position) strides if `t` can be read as (batch, positions, channels) where it lies, else None."""
    if t.numel() == 0:
        return _pair(0, 0)
    if not _adjacent_channels(t):
        return None
    dims = [(n, st) for n, st in zip(t.shape[1:-1], t.stride()[1:-1]) if n != 1]
    for (_, s0), (n1, s1) in zip(dims[:-1], dims[1:]):
        if s0 != s1 * n1:
            return None
    return _pair(t.stride(0), dims[-1][1] if dims else 0)


def _norm_entry(key, x, groups, weight, bias, eps, act, d_y=None):
    a = _norm_args(x, groups, weight, bias, eps, act)
    strides = [_positions_stride(x, a)]
    if d_y is not None:
        _check_activations("group_norm_act", x, d_y, names=("d_y",))
        strides.append(_positions_stride(d_y, a))
    if None in strides or not (weight is None or (weight.is_contiguous() and bias.is_contiguous())):
        return _remember(key, _Entry())
    a.x_stride = strides[0]
    if d_y is not None:
        a.d_y_stride = strides[1]
    partial = _lib.linrec_group_norm_partial_floats(a.dtype, a.batch, a.positions, a.channels, a.groups, int(d_y is not None))
    return _remember(key, _Entry(a, 0, ((2, a.batch, a.groups), partial)))


def norm_fwd(x, groups, weight, bias, eps, act):
    """(y, stats, number); stats is (2, batch, groups): the means, and the reciprocal deviations"""
    key = ("norm", x.dtype, x.device, x.shape, x.stride(), groups, _looks(weight), _looks(bias), eps, act)
    e = _remembered().get(key) or _norm_entry(key, x, groups, weight, bias, eps, act)
    a = e.args
    if a is None:
        return norm_fwd(*_dense(x), groups, *_dense(weight, bias), eps, act)
    device = x.device
    y = torch.empty(x.shape, dtype=x.dtype, device=device)
    stats = _floats(e.sizes[0], device)
    partial = _floats(e.sizes[1], device) if e.sizes[1] else None
    a.x, a.weight, a.bias, a.y, a.partial = x.data_ptr(), _p(weight), _p(bias), y.data_ptr(), _p(partial)
    a.mean = mean = stats.data_ptr()
    a.rstd = mean + 4 * a.batch * a.groups
    _call(x, _lib.linrec_group_norm_fwd, e, "group_norm_act")
    return y, stats, e.number


def norm_bwd(d_y, x, groups, weight, bias, stats, eps, act, number=None):
    """(d_x, d_weight, d_bias), the last two None without a weight"""
    if number is not None:
        key = (number, d_y.stride(), x.stride(), _stride(weight), _stride(bias))
    else:
        key = ("norm_bwd", x.dtype, x.device, x.shape, x.stride(), groups, _looks(d_y), _looks(weight), _looks(bias), eps, act)
    e = _remembered().get(key) or _norm_entry(key, x, groups, weight, bias, eps, act, d_y)
    a = e.args
    if a is None:
        return norm_bwd(*_dense(d_y, x), groups, *_dense(weight, bias), stats, eps, act)
    device = x.device
    if not stats.is_contiguous():
        stats = stats.contiguous()
    d_x = torch.empty(x.shape, dtype=x.dtype, device=device)
    d_weight = d_bias = None
    if weight is not None:
        d_weight, d_bias = torch.empty(weight.shape, dtype=weight.dtype, device=device), torch.empty(weight.shape, dtype=weight.dtype, device=device)
    partial = _floats(e.sizes[1], device)
    a.x, a.d_y, a.weight, a.bias, a.partial = x.data_ptr(), d_y.data_ptr(), _p(weight), _p(bias), partial.data_ptr()
    a.mean = mean = stats.data_ptr()
    a.rstd = mean + 4 * a.batch * a.groups
    a.d_x, a.d_weight, a.d_bias = d_x.data_ptr(), _p(d_weight), _p(d_bias)
    _call(x, _lib.linrec_group_norm_bwd, e, "group_norm_act")
    return d_x, d_weight, d_bias


# ---- embedding ---------------------------------------------------------------------------------
def _embedding_args(tokens, weight, scale, padding_idx):
    what = "embedding"
    if weight.dtype not in DTYPES:
        raise RuntimeError(f"{what}: weight must be float32, float16 or bfloat16, got {weight.dtype}")
    _check_device(what, weight, "weight")
    if weight.dim() != 2:
        raise RuntimeError(f"{what}: weight must be (vocabulary, channels), got {weight.dim()} dimensions")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{what}: tokens must be int32 or int64, got {tokens.dtype}")
    if tokens.device != weight.device:
        raise RuntimeError(f"{what}: tokens are on {tokens.device}, weight on {weight.device}")
    vocab, channels = weight.size()
    if padding_idx is not None:
        if not -vocab <= padding_idx < vocab:
            raise RuntimeError(f"{what}: padding_idx {padding_idx} is not in a table of {vocab} rows")
        padding_idx %= vocab
    return Embedding(dtype=DTYPES[weight.dtype], token_bytes=tokens.element_size(), scale=scale, tokens=tokens.numel(), vocab=vocab,
                     channels=channels, padding=-1 if padding_idx is None else padding_idx)


def embedding_fwd(tokens, weight, scale, padding_idx):
    """(y, number)"""
    key = ("embedding", _looks(tokens), weight.dtype, weight.device, weight.shape, weight.stride(), scale, padding_idx)
    e = _remembered().get(key)
    if e is None:
        a = _embedding_args(tokens, weight, scale, padding_idx)
        whole = tokens.is_contiguous() and weight.is_contiguous()
        e = _remember(key, _Entry(a, 0, ((*tokens.size(), weight.size(1)),)) if whole else _Entry())
    a = e.args
    if a is None:
        return embedding_fwd(*_dense(tokens, weight), scale, padding_idx)
    y = torch.empty(e.sizes[0], dtype=weight.dtype, device=weight.device)
    a.token, a.weight, a.y = tokens.data_ptr(), weight.data_ptr(), y.data_ptr()
    _call(weight, _lib.linrec_embedding_fwd, e, "embedding")
    return y, e.number


def embedding_bwd(d_y, tokens, weight, scale, padding_idx, number=None):
    """The gradient of `weight` (whose values are not read)."""
    if number is not None:
        key = (number, d_y.stride(), tokens.stride())
    else:
        key = ("embedding_bwd", _looks(d_y), _looks(tokens), weight.dtype, weight.device, weight.shape, scale, padding_idx)
    e = _remembered().get(key)
    if e is None:
        a = _embedding_args(tokens, weight, scale, padding_idx)
        if tuple(d_y.size()) != (*tokens.size(), weight.size(1)) or d_y.dtype != weight.dtype or d_y.device != weight.device:
            raise RuntimeError(f"embedding: d_y is {d_y.dtype} of {tuple(d_y.size())} on {d_y.device}")
        e = _Entry()
        stride = _row_stride(d_y)
        if stride is not None and tokens.is_contiguous():
            a.d_y_stride = stride
            e = _Entry(a, 0, (_lib.linrec_embedding_scratch_bytes(a.tokens, a.vocab, a.channels),))
        _remember(key, e)
    a = e.args
    if a is None:
        return embedding_bwd(*_dense(d_y, tokens), weight, scale, padding_idx)
    device = weight.device
    d_weight = torch.empty(weight.shape, dtype=weight.dtype, device=device)
    scratch = torch.empty(e.sizes[0], dtype=torch.uint8, device=device)
    a.token, a.d_y, a.d_weight = tokens.data_ptr(), d_y.data_ptr(), d_weight.data_ptr()
    a.scratch, a.scratch_bytes = scratch.data_ptr(), e.sizes[0]
    _call(weight, _lib.linrec_embedding_bwd, e, "embedding")
    return d_weight


def _row_stride(t):
    """Stride of the rows if `t` is rows of adjacent channels, a uniform distance apart, else None."""
    if t.numel() == 0:
        return t.size(-1)
    if not _adjacent_channels(t):
        return None
    dims = [(n, st) for n, st in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
    for (_, s0), (n1, s1) in zip(dims[:-1], dims[1:]):
        if s0 != s1 * n1:
            return None
    return dims[-1][1] if dims else t.size(-1)
