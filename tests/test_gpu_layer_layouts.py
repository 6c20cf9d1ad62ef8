"""The layer operators on inputs that lie differently in memory than those of an earlier call of the same sizes: results and
gradients are the same bits as those of dense copies, whichever came first."""
import threading

import pytest
import torch

import linrec_amd

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def same(got, want):
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


def check(call, layouts, wanted, hooks=None):
    """`call` gives outputs; `layouts` maps names to tensors on the device.  Outputs and gradients of the `wanted` names for the
    tensors as they lie, between those of dense copies."""
    def run(dense, hooks=None):
        leaves = {}
        for name, t in layouts.items():
            leaves[name] = None if t is None else (t.contiguous() if dense else t.detach())
            if name in wanted and t is not None:
                leaves[name].requires_grad_()
        gen = torch.Generator(device=DEV).manual_seed(5)

        def whole():
            outputs = call(**leaves)
            d_outputs = [torch.randn(o.shape, generator=gen, device=DEV).to(o.dtype) for o in outputs]
            return [*(o.detach() for o in outputs), *torch.autograd.grad(outputs, [leaves[n] for n in wanted if leaves[n] is not None], d_outputs)]
        if hooks is None:
            return whole()
        with hooks:
            return whole()

    orders = []
    for order in ([True, False, True], [False, True, False]):
        orders += [run(dense) for dense in order]
    for got in orders[1:]:
        same(got, orders[0])
    dense_again = torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format))
    same(run(False, dense_again), orders[0])
    same(run(False, torch.autograd.graph.save_on_cpu()), orders[0])


GATED = ("x", "gate_a", "gate_x", "rate", "h0")


def gated(x, gate_a, gate_x, rate, h0, cu_seqlens):
    return linrec_amd.gated_linrec(x, gate_a, gate_x, rate, h0=h0, cu_seqlens=cu_seqlens, return_state=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("packed", [False, True])
def test_gated_linrec(packed, dtype):
    def normal(*shape):
        return torch.randn(shape, device=DEV).to(dtype)
    torch.manual_seed(1)
    lead = (150,) if packed else (2, 75)
    sequences = 3 if packed else 2
    bounds = torch.tensor([0, 40, 40, 150], dtype=torch.int32, device=DEV) if packed else None
    base = dict(x=normal(*lead, 34), gate_a=normal(*lead, 34), gate_x=normal(*lead, 34), rate=torch.randn(34, device=DEV),
                h0=torch.randn(sequences, 34, device=DEV), cu_seqlens=bounds)
    changes = [dict(x=normal(*lead[:-1], 34, lead[-1]).transpose(-1, -2)), dict(gate_a=normal(*lead, 1).expand(*lead, 34)),
               dict(gate_x=normal(*lead[:-1], 1, 34).expand(*lead, 34)), dict(zip(("x", "gate_a", "gate_x"), normal(*lead, 102).chunk(3, -1))),
               dict(h0=torch.randn(sequences, 2, 34, device=DEV)[:, 1]), dict(rate=torch.randn(68, device=DEV)[::2])]
    if packed:
        changes.append(dict(cu_seqlens=torch.tensor([0, 9, 33, 9, 34, 9, 150, 9], dtype=torch.int32, device=DEV)[::2]))
    for change in changes:
        check(gated, {**base, **change}, GATED)


@pytest.mark.parametrize("shape,groups", [((150, 64), 4), ((2, 75, 64), 4), ((2, 9000, 16), 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_group_norm_act(shape, groups, dtype):
    torch.manual_seed(2)
    channels = shape[-1]
    base = dict(x=torch.randn(shape, device=DEV).to(dtype), weight=torch.randn(channels, device=DEV), bias=torch.randn(channels, device=DEV))
    turned = torch.randn(*shape[:-2], channels, shape[-2], device=DEV).to(dtype).transpose(-1, -2)
    for change in (dict(x=turned), dict(x=torch.randn(*shape[:-1], channels + 5, device=DEV).to(dtype)[..., 3:channels + 3]),
                   dict(weight=torch.randn(2 * channels, device=DEV)[::2])):
        check(lambda x, weight, bias: [linrec_amd.group_norm_act(x, groups, weight, bias)], {**base, **change}, ("x", "weight", "bias"))


@pytest.mark.parametrize("n", [8, 3000])
def test_embedding(n):
    torch.manual_seed(3)
    weight = torch.randn(50, 20, device=DEV)
    for tokens in (torch.randint(0, 50, (n, 4), device=DEV).t(), torch.randint(0, 50, (4, n + 1), device=DEV)[:, :-1],
                   torch.randint(0, 50, (4, 1), device=DEV).expand(4, n)):
        check(lambda tokens, weight: [linrec_amd.embedding(tokens, weight, scale=2.0)], dict(tokens=tokens, weight=weight), ("weight",))


def test_on_other_threads():
    """Calls are remembered by thread: forwards on three threads at once, each with its own layouts, backwards on the engine's."""
    torch.manual_seed(4)
    tensors = [torch.randn(3, 40, 66, device=DEV).chunk(3, -1) for _ in range(3)]
    rate = torch.randn(22, device=DEV)

    def run(views, dense):
        leaves = [(t.contiguous() if dense else t.detach()).requires_grad_() for t in views]
        h = linrec_amd.gated_linrec(*leaves, rate)
        return [h.detach(), *torch.autograd.grad(h, leaves, torch.ones_like(h))]
    want = [run(views, True) for views in tensors]
    got = [None] * 3

    def work(i):
        for _ in range(4):
            got[i] = run(tensors[i], False)
        torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(3):
        same(got[i], want[i])
