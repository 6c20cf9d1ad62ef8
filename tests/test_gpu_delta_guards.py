"""The gated delta rule writes nothing beside its results and its scratch, whatever cu_seqlens holds: all of them lie in one buffer here, with
guards between them.  (That the numbers of chunks and segments stay in their room is tested without a GPU in test_delta_scratch_room.py.)"""
import ctypes

import pytest
import torch

from linrec_amd import _delta

from .test_gpu_delta import DEV, make

pytestmark = pytest.mark.gpu
GUARD, MARK = 512, 0xA5


class Room:
    """Parts of one buffer, 256-byte aligned, MARK everywhere else."""

    def __init__(self, bytes_of):
        self.places, at = {}, GUARD
        for name, n in bytes_of.items():
            self.places[name] = (at, n)
            at += -(-n // 256) * 256 + GUARD
        self.buffer = torch.full((at,), MARK, dtype=torch.uint8, device=DEV)

    def pointer(self, name):
        return self.buffer.data_ptr() + self.places[name][0]

    def values(self, name, dtype):
        at, n = self.places[name]
        return self.buffer[at:at + n].view(dtype)

    def check(self):
        outside = torch.ones_like(self.buffer, dtype=torch.bool)
        for at, n in self.places.values():
            outside[at:at + n] = False
        assert bool((self.buffer[outside] == MARK).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("time,heads,dims", [(200, (1, 2), (20, 33)), (4096, (1, 1), (64, 40)), (2048, (1, 2), (130, 17))])
def test_nothing_beside_the_results_is_written(time, heads, dims, dtype):
    many = [0, 1, time, time, 5, -7, 2 ** 31 - 1, -2 ** 31, time - 1, time]
    for bounds in ([0, time], [0, time // 3, time], [0, time + 500], [-5, time], [0, time - 96, 20, time], [time, 0, time], [10, time // 2],
                   [time] * 3, many, many[::-1]):
        n = len(bounds) - 1
        q, k, v, log_decay, beta, h0, d_o, d_state = (t.to(DEV) for t in make((time,), heads, dims, dtype, seed=2, sequences=n))
        cu = torch.tensor(bounds, dtype=torch.int32, device=DEV)
        a = _delta._delta_args(q, k, v, log_decay, beta, h0, cu, 0.5, d_o)
        a.d_o_stride = _delta._strides(d_o, True)
        a.cu_seqlens = cu.data_ptr()
        need = [_delta._lib.linrec_delta_scratch_bytes(ctypes.byref(a), bwd) for bwd in (0, 1)]
        size = q.element_size()
        room = Room({"o": v.numel() * size, "state": h0.numel() * 4, "scratch": need[0], "d_q": q.numel() * size, "d_k": k.numel() * size,
                     "d_v": v.numel() * size, "d_log_decay": beta.numel() * 4, "d_beta": beta.numel() * 4, "d_h0": h0.numel() * 4, "scratch_bwd": need[1]})
        a.q, a.k, a.v, a.log_decay, a.beta, a.h0 = (t.data_ptr() for t in (q, k, v, log_decay, beta, h0))
        a.d_o, a.d_state = d_o.data_ptr(), d_state.data_ptr()
        for name in ("o", "state", "d_q", "d_k", "d_v", "d_log_decay", "d_beta", "d_h0"):
            setattr(a, name, room.pointer(name))
        a.stream = torch.cuda.current_stream().cuda_stream
        for call, bwd, name in ((_delta._lib.linrec_delta_fwd, 0, "scratch"), (_delta._lib.linrec_delta_bwd, 1, "scratch_bwd")):
            a.scratch, a.scratch_bytes = room.pointer(name), need[bwd]
            assert call(ctypes.byref(a)) == 0
            torch.cuda.synchronize()
            room.check()
        if bounds == [0, time]:  # right ones give all of the result
            o, state, _ = _delta.delta_fwd(q, k, v, log_decay, beta, h0, cu, 0.5)
            assert torch.equal(room.values("o", dtype).view_as(o), o) and torch.equal(room.values("state", torch.float32).view_as(state), state)
            grads = _delta.delta_bwd(d_o, d_state, q, k, v, log_decay, beta, h0, cu, 0.5)
            for name, grad in zip(("d_q", "d_k", "d_v", "d_log_decay", "d_beta", "d_h0"), grads):
                assert torch.equal(room.values(name, grad.dtype).view_as(grad), grad), name
