"""The gated delta rule's single-token step on the device: against the definition in float64, and against the chunk form it goes on from."""
import pytest
import torch

import linrec_amd

from . import delta_reference as ref
from . import test_gpu_delta as delta
from .test_gpu_delta import DEV, DTYPES

pytestmark = pytest.mark.gpu


def make(batch, heads, dims, dtype, seed=0):
    return [t[:, 0] if n < 5 else t for n, t in enumerate(delta.make((batch, 1), heads, dims, dtype, seed)[:6])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,heads,dims", [(1, (1, 1), (1, 1)), (3, (2, 4), (20, 12)), (2, (1, 2), (64, 64)), (5, (2, 2), (128, 128)),
                                              (1, (1, 3), (100, 72)), (2, (1, 1), (256, 130)), (7, (1, 1), (33, 3))])
def test_against_the_definition(batch, heads, dims, dtype):
    q, k, v, log_decay, beta, state = make(batch, heads, dims, dtype, seed=batch + sum(dims))
    o_t, state_t = ref.gated_delta(*(t[:, None] for t in (q, k, v, log_decay, beta)), state)
    # one position is a sum of key_dim products in fp32 whatever the inputs
    cache = state.to(DEV)
    o = linrec_amd.gated_delta_step(*(t.to(DEV) for t in (q, k, v, log_decay, beta)), cache)
    ref.assert_near(o, o_t[:, 0], ref.bound(dtype, torch.float32, 1), "o")
    ref.assert_near(cache, state_t, ref.bound(torch.float32, torch.float32, 1), "state")


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_a_cache(dtype):
    """Slots in any order, some of them none; other rows of the cache stay as they are."""
    q, k, v, log_decay, beta, state = make(6, (2, 4), (40, 36), dtype, seed=3)
    slots = torch.tensor([7, -1, 0, 9, 3, 8], dtype=torch.int32)
    takes = [0, 2, 4, 5]
    wide = torch.randn((9, 2, 4, 40, 36))
    cache = wide.to(DEV)[:, 1]
    before = cache.clone()
    o = linrec_amd.gated_delta_step(*(t.to(DEV) for t in (q, k, v, log_decay, beta)), cache, slots=slots.to(DEV))
    rows = slots[takes].long()
    o_t, state_t = ref.gated_delta(*(t[takes][:, None] for t in (q, k, v, log_decay, beta)), wide[:, 1][rows])
    ref.assert_near(o[takes], o_t[:, 0], ref.bound(dtype, torch.float32, 1), "o")
    ref.assert_near(cache[rows.to(DEV)], state_t, ref.bound(torch.float32, torch.float32, 1), "state")
    assert torch.equal(o[[1, 3]], torch.zeros_like(o[[1, 3]]))
    rest = [n for n in range(9) if n not in rows.tolist()]
    assert torch.equal(cache[rest], before[rest])


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_go_on_from_a_prompt(dtype):
    """A packed prompt and single steps behind it give what one call over all of it gives."""
    lengths, more = [70, 5, 128], 4
    total = [n + more for n in lengths]
    whole = [0] + torch.tensor(total).cumsum(0).tolist()
    data = delta.make((whole[-1],), (2, 4), (64, 40), dtype, seed=11, sequences=3)
    inputs, h0 = [t.to(DEV) for t in data[:5]], data[5].to(DEV)
    o_t, state_t = ref.gated_delta(*data[:5], data[5], whole)
    prompt = torch.cat([torch.arange(a, a + n) for a, n in zip(whole, lengths)]).to(DEV)
    cu = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    cache = torch.zeros((5, 4, 64, 40), device=DEV)
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device=DEV)
    o, state = linrec_amd.gated_delta(*(t[prompt] for t in inputs), h0=h0, cu_seqlens=cu, return_state=True)
    cache[slots.long()] = state
    near = ref.bound(dtype, dtype, max(total))
    ref.assert_near(o, o_t[prompt.cpu()], near, "prompt")
    for n in range(more):
        at = torch.tensor([a + length + n for a, length in zip(whole, lengths)], device=DEV)
        o = linrec_amd.gated_delta_step(*(t[at] for t in inputs), cache, slots=slots)
        ref.assert_near(o, o_t[at.cpu()], near, f"step {n}")
    ref.assert_near(cache[slots.long()], state_t, ref.bound(torch.float32, dtype, max(total)), "state")


def test_refusals_and_empty_batches():
    q, k, v, log_decay, beta, state = (t.to(DEV) for t in make(2, (1, 2), (8, 4), torch.float32))
    step = linrec_amd.gated_delta_step
    with pytest.raises(RuntimeError, match="records no gradient"):
        step(q.clone().requires_grad_(), k, v, log_decay, beta, state)
    with pytest.raises(RuntimeError, match="state must be float32"):
        step(q, k, v, log_decay, beta, state.half())
    with pytest.raises(RuntimeError, match="dense rows"):
        step(q, k, v, log_decay, beta, state.transpose(-1, -2).contiguous().transpose(-1, -2))
    with pytest.raises(RuntimeError, match="overlap"):
        step(q, k, v, log_decay, beta, state[:1].expand(2, -1, -1, -1))
    with pytest.raises(RuntimeError, match="slots must be int32"):
        step(q, k, v, log_decay, beta, state, slots=torch.zeros(2, dtype=torch.long, device=DEV))
    with pytest.raises(RuntimeError, match="rows, q has"):
        step(q, k, v, log_decay, beta, state[:1])
    empty = [t[:0] for t in (q, k, v, log_decay, beta)]
    assert step(*empty, state, slots=torch.empty(0, dtype=torch.int32, device=DEV)).shape == (0, 2, 4)


def test_captured_steps():
    q, k, v, log_decay, beta, state = (t.to(DEV) for t in make(3, (1, 2), (64, 64), torch.bfloat16, seed=5))
    eager, replayed = state.clone(), state.clone()
    want = [linrec_amd.gated_delta_step(q, k, v, log_decay, beta, eager) for _ in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o = linrec_amd.gated_delta_step(q, k, v, log_decay, beta, replayed)
    replayed.copy_(state)
    for n in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[n])
    assert torch.equal(replayed, eager)
