"""ctypes binding of include/linrec_delta.h: argument checks, allocation of results and scratch with torch, one library call.

As _layers.py, whose table of remembered calls it shares: device tensors only, and a call that looks like an earlier one fills only
the pointers of that call's argument block in.
"""
import ctypes

import torch

from . import _layers
from ._layers import _Entry, _adjacent_channels, _check_activations, _check_device, _check_fp32, _dense, _floats, _looks, _p, _remember, _remembered, \
    _stride, _with_adjacent_channels
from ._native import DTYPES, lib

_i32, _i64, _f32, _ptr, _u64 = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p, ctypes.c_uint64
_pair, _three = _i64 * 2, _i64 * 3
KEY_DIM_MAX = 256  # LINREC_DELTA_KEY_DIM_MAX
ROW_MAX = 1 << 28  # LINREC_DELTA_ROW_MAX


class Delta(ctypes.Structure):
    """linrec_delta_t"""
    _fields_ = [("dtype", _i32), ("key_heads", _i32), ("heads", _i32), ("key_dim", _i32), ("value_dim", _i32), ("scale", _f32),
                ("batch", _i64), ("time", _i64), ("sequences", _i64), ("cu_seqlens", _ptr), ("q", _ptr), ("k", _ptr), ("v", _ptr),
                ("q_stride", _three), ("k_stride", _three), ("v_stride", _three), ("log_decay", _ptr), ("beta", _ptr),
                ("log_decay_stride", _three), ("beta_stride", _three), ("h0", _ptr), ("o", _ptr), ("state", _ptr), ("d_o", _ptr),
                ("d_o_stride", _three), ("d_state", _ptr), ("d_q", _ptr), ("d_k", _ptr), ("d_v", _ptr), ("d_log_decay", _ptr),
                ("d_beta", _ptr), ("d_h0", _ptr), ("scratch", _ptr), ("scratch_bytes", _u64), ("stream", _ptr)]


class DeltaStep(ctypes.Structure):
    """linrec_delta_step_t"""
    _fields_ = [("dtype", _i32), ("key_heads", _i32), ("heads", _i32), ("key_dim", _i32), ("value_dim", _i32), ("scale", _f32),
                ("batch", _i64), ("slots_total", _i64), ("q", _ptr), ("k", _ptr), ("v", _ptr), ("q_stride", _pair), ("k_stride", _pair),
                ("v_stride", _pair), ("log_decay", _ptr), ("beta", _ptr), ("log_decay_stride", _pair), ("beta_stride", _pair),
                ("slots", _ptr), ("state", _ptr), ("state_stride", _i64), ("o", _ptr), ("stream", _ptr)]


EXPORTS = {
    "linrec_delta_scratch_bytes": (ctypes.c_size_t, [ctypes.POINTER(Delta), ctypes.c_int]),
    "linrec_delta_fwd": (ctypes.c_int, [ctypes.POINTER(Delta)]),
    "linrec_delta_bwd": (ctypes.c_int, [ctypes.POINTER(Delta)]),
    "linrec_delta_step": (ctypes.c_int, [ctypes.POINTER(DeltaStep)]),
}


def _declare():
    handle = lib()
    for name, (result, arguments) in EXPORTS.items():
        fn = getattr(handle, name)
        fn.restype, fn.argtypes = result, arguments
    return handle


_lib = _declare()


# ---- checks (of calls that are not remembered) --------------------------------------------------
def _check_heads(what, q, k, v, log_decay, beta, leading, lead):
    """`leading`: names of the dimensions before the heads, `lead`: their sizes."""
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if t.dim() != len(lead) + 2:
            raise RuntimeError(f"{what}: {name} must be ({leading}, heads, {'value_dim' if name == 'v' else 'key_dim'}), got {t.dim()} dimensions")
    _check_activations(what, q, k, names=("k",))
    for t, name in ((v, "v"), (log_decay, "log_decay"), (beta, "beta")):
        if t.device != q.device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, q on {q.device}")
    if v.dtype != q.dtype:
        raise RuntimeError(f"{what}: v has dtype {v.dtype}, q has {q.dtype}")
    if tuple(v.size()[:-2]) != lead:
        raise RuntimeError(f"{what}: v has size {tuple(v.size())}, q has {tuple(q.size())}")
    key_heads, key_dim, heads, value_dim = q.size(-2), q.size(-1), v.size(-2), v.size(-1)
    if key_heads < 1 or heads < 1 or heads % key_heads:
        raise RuntimeError(f"{what}: {heads} value heads cannot share {key_heads} key heads")
    if not 1 <= key_dim <= KEY_DIM_MAX:
        raise RuntimeError(f"{what}: key_dim must be 1 to {KEY_DIM_MAX}, got {key_dim}")
    if not 1 <= value_dim <= 1 << 20:
        raise RuntimeError(f"{what}: value_dim must be 1 to {1 << 20}, got {value_dim}")
    for t, name in ((log_decay, "log_decay"), (beta, "beta")):
        _check_fp32(what, t, name, (*lead, heads), q.device)
    return key_heads, key_dim, heads, value_dim


def delta_shape(q, cu_seqlens):
    """(batch, time, sequences) of a call; raises if the dimensions do not fit."""
    what = "gated_delta"
    if cu_seqlens is None:
        if q.dim() != 4:
            raise RuntimeError(f"{what}: q must be (batch, time, heads, key_dim), got {q.dim()} dimensions")
        return q.size(0), q.size(1), q.size(0)
    if q.dim() != 3:
        raise RuntimeError(f"{what}: with cu_seqlens q must be (positions, heads, key_dim), got {q.dim()} dimensions")
    if cu_seqlens.dim() != 1 or cu_seqlens.size(0) < 1:
        raise RuntimeError(f"{what}: cu_seqlens must be one-dimensional, sequences + 1 bounds")
    if cu_seqlens.dtype != torch.int32:
        raise RuntimeError(f"{what}: cu_seqlens must be int32, got {cu_seqlens.dtype}")
    if cu_seqlens.device != q.device:
        raise RuntimeError(f"{what}: cu_seqlens is on {cu_seqlens.device}, q on {q.device}")
    if cu_seqlens.size(0) == 1 and q.size(0) > 0:
        raise RuntimeError(f"{what}: positions but no sequence to hold them")
    return 1, q.size(0), cu_seqlens.size(0) - 1


def _strides(t, packed, heads=True):
    """batch, time and head strides of (batch, time, heads, channels), or of gates without the last"""
    s = t.stride()[:-1] if heads else t.stride()
    return _three(0, *s) if packed else _three(*s)


def _delta_args(q, k, v, log_decay, beta, h0, cu_seqlens, scale, *gradients):
    """An argument block with everything but the pointers; None if a tensor has to be copied first."""
    what = "gated_delta"
    _check_device(what, q, "q")
    batch, time, sequences = delta_shape(q, cu_seqlens)
    packed = cu_seqlens is not None
    lead = (time,) if packed else (batch, time)
    key_heads, key_dim, heads, value_dim = _check_heads(what, q, k, v, log_decay, beta, "positions" if packed else "batch, time", lead)
    if heads * value_dim > ROW_MAX:
        raise RuntimeError(f"{what}: {heads} heads of {value_dim} values are more than {ROW_MAX} values a position")
    if h0 is not None:
        _check_fp32(what, h0, "h0", (sequences, heads, key_dim, value_dim), q.device)
    whole = all(t is None or t.is_contiguous() for t in (h0, cu_seqlens))
    if not (whole and all(_adjacent_channels(t) for t in (q, k, v, *gradients))):
        return None
    return Delta(dtype=DTYPES[q.dtype], key_heads=key_heads, heads=heads, key_dim=key_dim, value_dim=value_dim, scale=scale, batch=batch, time=time,
                 sequences=sequences, q_stride=_strides(q, packed), k_stride=_strides(k, packed), v_stride=_strides(v, packed),
                 log_decay_stride=_strides(log_decay, packed, False), beta_stride=_strides(beta, packed, False))


def _scratch(e, device):
    return torch.empty(e.sizes[-1], dtype=torch.uint8, device=device) if e.sizes[-1] else None


def delta_fwd(q, k, v, log_decay, beta, h0, cu_seqlens, scale, with_state=True):
    """(o, state, number); state is None without `with_state`."""
    key = ("delta", _looks(q), _looks(k), _looks(v), _looks(log_decay), _looks(beta), _looks(h0), _looks(cu_seqlens), scale)
    e = _remembered().get(key)
    if e is None:
        a = _delta_args(q, k, v, log_decay, beta, h0, cu_seqlens, scale)
        e = _Entry()
        if a is not None:
            a.cu_seqlens = _p(cu_seqlens)
            e = _Entry(a, 0, ((a.sequences, a.heads, a.key_dim, a.value_dim), _lib.linrec_delta_scratch_bytes(ctypes.byref(a), 0)))
        _remember(key, e)
    a = e.args
    if a is None:
        return delta_fwd(*_with_adjacent_channels(q, k, v), log_decay, beta, *_dense(h0, cu_seqlens), scale, with_state)
    device = q.device
    o = torch.empty(v.shape, dtype=v.dtype, device=device)
    state = _floats(e.sizes[0], device) if with_state else None
    scratch = _scratch(e, device)
    a.q, a.k, a.v, a.log_decay, a.beta = q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), beta.data_ptr()
    a.h0, a.cu_seqlens, a.o, a.state = _p(h0), _p(cu_seqlens), o.data_ptr(), _p(state)
    a.scratch, a.scratch_bytes = _p(scratch), e.sizes[-1]
    _layers._call(q, _lib.linrec_delta_fwd, e, "gated_delta")
    return o, state, e.number


def delta_bwd(d_o, d_state, q, k, v, log_decay, beta, h0, cu_seqlens, scale, number=None):
    """(d_q, d_k, d_v, d_log_decay, d_beta, d_h0); d_h0 is None without h0, d_o or d_state may be None (zeros)."""
    if d_o is None:
        d_o = torch.zeros((), dtype=v.dtype, device=v.device).expand(v.size())
    if number is not None:
        key = (number, d_o.stride(), _stride(d_state), q.stride(), k.stride(), v.stride(), log_decay.stride(), beta.stride(), _stride(h0),
               _stride(cu_seqlens))
    else:
        key = ("delta_bwd", _looks(d_o), _looks(d_state), _looks(q), _looks(k), _looks(v), _looks(log_decay), _looks(beta), _looks(h0),
               _looks(cu_seqlens), scale)
    e = _remembered().get(key)
    if e is None:
        a = _delta_args(q, k, v, log_decay, beta, h0, cu_seqlens, scale, d_o)
        _check_activations("gated_delta", v, d_o, names=("d_o",))
        if d_state is not None:
            _check_fp32("gated_delta", d_state, "d_state", (delta_shape(q, cu_seqlens)[2], v.size(-2), q.size(-1), v.size(-1)), q.device)
        e = _Entry()
        if a is not None and (d_state is None or d_state.is_contiguous()):
            a.d_o_stride, a.cu_seqlens = _strides(d_o, cu_seqlens is not None), _p(cu_seqlens)
            e = _Entry(a, 0, (_lib.linrec_delta_scratch_bytes(ctypes.byref(a), 1),))
        _remember(key, e)
    a = e.args
    if a is None:
        return delta_bwd(*_with_adjacent_channels(d_o), *_dense(d_state), *_with_adjacent_channels(q, k, v), log_decay, beta, *_dense(h0, cu_seqlens),
                         scale)
    device = q.device
    d_q, d_k, d_v = (torch.empty(t.shape, dtype=t.dtype, device=device) for t in (q, k, v))
    d_log_decay, d_beta = _floats(log_decay.shape, device), _floats(beta.shape, device)
    d_h0 = None if h0 is None else _floats(h0.shape, device)
    scratch = _scratch(e, device)
    a.q, a.k, a.v, a.log_decay, a.beta = q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), beta.data_ptr()
    a.h0, a.cu_seqlens, a.d_o, a.d_state = _p(h0), _p(cu_seqlens), d_o.data_ptr(), _p(d_state)
    a.d_q, a.d_k, a.d_v, a.d_log_decay, a.d_beta, a.d_h0 = d_q.data_ptr(), d_k.data_ptr(), d_v.data_ptr(), d_log_decay.data_ptr(), d_beta.data_ptr(), \
        _p(d_h0)
    a.scratch, a.scratch_bytes = _p(scratch), e.sizes[-1]
    _layers._call(q, _lib.linrec_delta_bwd, e, "gated_delta")
    return d_q, d_k, d_v, d_log_decay, d_beta, d_h0


def _step_args(q, k, v, log_decay, beta, state, slots, scale):
    what = "gated_delta_step"
    _check_device(what, q, "q")
    if q.dim() != 3:
        raise RuntimeError(f"{what}: q must be (batch, heads, key_dim), got {q.dim()} dimensions")
    batch = q.size(0)
    key_heads, key_dim, heads, value_dim = _check_heads(what, q, k, v, log_decay, beta, "batch", (batch,))
    if state.dim() != 4:
        raise RuntimeError(f"{what}: state must be (rows, heads, key_dim, value_dim), got {state.dim()} dimensions")
    _check_fp32(what, state, "state", (state.size(0), heads, key_dim, value_dim), q.device)
    if state.size(0) > 0 and not state[0].is_contiguous():
        raise RuntimeError(f"{what}: state is updated in place and needs dense rows of (heads, key_dim, value_dim)")
    if state.size(0) > 1 and state.stride(0) < heads * key_dim * value_dim:
        raise RuntimeError(f"{what}: rows of state overlap in memory")
    if slots is None:
        if state.size(0) != batch:
            raise RuntimeError(f"{what}: state has {state.size(0)} rows, q has {batch} (name the rows with slots)")
    elif slots.dtype != torch.int32 or tuple(slots.size()) != (batch,):
        raise RuntimeError(f"{what}: slots must be int32 of size ({batch},), got {slots.dtype} of {tuple(slots.size())}")
    elif slots.device != q.device:
        raise RuntimeError(f"{what}: slots is on {slots.device}, q on {q.device}")
    if not ((slots is None or slots.is_contiguous()) and all(_adjacent_channels(t) for t in (q, k, v))):
        return None
    return DeltaStep(dtype=DTYPES[q.dtype], key_heads=key_heads, heads=heads, key_dim=key_dim, value_dim=value_dim, scale=scale, batch=batch,
                     slots_total=state.size(0), q_stride=_pair(*q.stride()[:2]), k_stride=_pair(*k.stride()[:2]), v_stride=_pair(*v.stride()[:2]),
                     log_decay_stride=_pair(*log_decay.stride()), beta_stride=_pair(*beta.stride()), state_stride=state.stride(0))


def delta_step(q, k, v, log_decay, beta, state, slots, scale):
    key = ("delta_step", _looks(q), _looks(k), _looks(v), _looks(log_decay), _looks(beta), _looks(state), _looks(slots), scale)
    e = _remembered().get(key)
    if e is None:
        e = _remember(key, _Entry(_step_args(q, k, v, log_decay, beta, state, slots, scale)))
    a = e.args
    if a is None:
        return delta_step(*_with_adjacent_channels(q, k, v), log_decay, beta, state, *_dense(slots), scale)
    o = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    a.q, a.k, a.v, a.log_decay, a.beta = q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), beta.data_ptr()
    a.slots, a.state, a.o = _p(slots), state.data_ptr(), o.data_ptr()
    _layers._call(q, _lib.linrec_delta_step, e, "gated_delta_step")
    return o
