"""The layer operators in compiled programs: the same bits as in eager mode, forward and backward, and one program for all sizes."""
import pytest
import torch

import linrec_amd

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def gated(x, gate_a, gate_x, rate, h0):
    h, state = linrec_amd.gated_linrec(x, gate_a, gate_x, rate, h0=h0, return_state=True)
    return h * 2, state


def packed(x, gate_a, gate_x, rate, cu_seqlens):
    return (linrec_amd.gated_linrec(x, gate_a, gate_x, rate, cu_seqlens=cu_seqlens, reverse=True),)


def norm(x, weight, bias):
    return (linrec_amd.group_norm_act(x, 2, weight, bias),)


def table(tokens, weight):
    return (linrec_amd.embedding(tokens, weight, scale=2.0, padding_idx=1),)


def inputs(name, n):
    g = torch.Generator(device=DEV).manual_seed(n)

    def normal(*shape):
        return torch.randn(shape, device=DEV, generator=g)
    if name == "gated":
        return gated, [normal(2, 40 * n, 6) for _ in range(3)] + [normal(6), normal(2, 6)]
    if name == "packed":
        bounds = torch.tensor([0, n, n, 39 * n, 40 * n], dtype=torch.int32, device=DEV)
        return packed, [normal(40 * n, 6) for _ in range(3)] + [normal(6), bounds]
    if name == "norm":
        return norm, [normal(2, n, 8), normal(8), normal(8)]
    return table, [torch.randint(0, 9, (n, 2), device=DEV, generator=g), normal(9, 6)]


@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("name", ["gated", "packed", "norm", "table"])
def test_a_training_step(name, dynamic):
    torch._dynamo.reset()
    compiled = None
    for n in (3, 5, 9):
        fn, args = inputs(name, n)
        compiled = compiled or torch.compile(fn, backend="aot_eager", dynamic=dynamic, fullgraph=True)
        results = []
        for call in (fn, torch._dynamo.config.patch(error_on_recompile=dynamic)(compiled)):
            leaves = [t.clone().requires_grad_() if t.is_floating_point() else t for t in args]
            outputs = call(*leaves)
            wanted = [t for t in leaves if t.requires_grad]
            results.append([*outputs, *torch.autograd.grad(sum(o.sum() for o in outputs), wanted)])
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_a_single_token_step():
    torch._dynamo.reset()
    compiled = torch.compile(lambda *args: linrec_amd.gated_linrec_step(*args) + 1, backend="aot_eager", dynamic=True, fullgraph=True)
    for n in (3, 7):
        x, gate_a, gate_x, state = (torch.randn(n, 6, device=DEV) for _ in range(4))
        rate, other = torch.randn(6, device=DEV), state.clone()
        with torch.no_grad():
            assert torch.equal(compiled(x, gate_a, gate_x, rate, state), linrec_amd.gated_linrec_step(x, gate_a, gate_x, rate, other) + 1)
        assert torch.equal(state, other)


def test_transforms():
    """vmap goes over the calls one by one; derivatives that nobody has written are refused."""
    x, rate = torch.randn(3, 2, 40, 6, device=DEV), torch.randn(6, device=DEV)
    got = torch.func.vmap(lambda t: linrec_amd.gated_linrec(t, t, t, rate))(x)
    assert torch.equal(got, torch.stack([linrec_amd.gated_linrec(t, t, t, rate) for t in x]))
    got = torch.func.vmap(lambda t: linrec_amd.group_norm_act(t, 2))(x)
    assert torch.equal(got, torch.stack([linrec_amd.group_norm_act(t, 2) for t in x]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: linrec_amd.gated_linrec(t, t, t, rate).sum())(x[0])
    with pytest.raises(RuntimeError, match="jvp"):
        torch.func.jvp(lambda t: linrec_amd.group_norm_act(t, 2), (x,), (x,))
