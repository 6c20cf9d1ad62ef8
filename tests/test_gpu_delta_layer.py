"""A layer of rms_norm, gated_delta and gated_delta_step as a model would use them together, and the calls beside the plain ones: compiled
programs, several streams, a captured training step, one tensor as two arguments.

The layer is compared in fp32 with the same formulas in float64.  Its values pass the delta rule once and five roundings of products
of up to 96 terms and of norms (96^1/2 2^-24 and 4 * 2^-24 each, 2^-19 together), less than the delta rule's own 8 * 2^-20 * sqrt(2 + chunks);
the gradient passes both once more.  A norm divides by what it measures, so errors relative to a tensor's size stay what they are, and
the parts that join at a residual, at q, k and v, or at a weight add up: four times the delta rule's bound."""
import pytest
import torch

import linrec_amd

from . import delta_reference as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CHANNELS, KEY_HEADS, HEADS, KEY_DIM, VALUE_DIM = 96, 2, 4, 24, 40
SPLIT = [KEY_HEADS * KEY_DIM, KEY_HEADS * KEY_DIM, HEADS * VALUE_DIM, HEADS, HEADS]


def weights(seed):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, by=1.0):
        return torch.randn(shape, generator=g) * by
    return {"norm": 1 + normal(CHANNELS, by=0.1), "into": normal(CHANNELS, sum(SPLIT), by=CHANNELS ** -0.5), "q_norm": 1 + normal(KEY_DIM, by=0.1),
            "o_norm": 1 + normal(VALUE_DIM, by=0.1), "out": normal(HEADS * VALUE_DIM, CHANNELS, by=(HEADS * VALUE_DIM) ** -0.5)}


def plain_norm(x, weight=None):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    return y if weight is None else y * weight


def layer(w, x, residual, mix):
    """(out, total); `mix` has q, k, v and the gates of the heads and gives o."""
    if x.dtype == torch.float64:
        total = x + residual
        y, head_norm = plain_norm(total, w["norm"]), plain_norm
    else:
        y, total = linrec_amd.rms_norm(x, w["norm"], residual=residual)
        head_norm = linrec_amd.rms_norm
    q, k, v, decay, beta = (y @ w["into"]).split(SPLIT, -1)
    q, k = (t.unflatten(-1, (KEY_HEADS, KEY_DIM)) for t in (q, k))
    q, k = head_norm(q, w["q_norm"]) * KEY_DIM ** -0.5, head_norm(k) * KEY_DIM ** -0.5
    o = mix(q, k, v.unflatten(-1, (HEADS, VALUE_DIM)), -0.1 * torch.nn.functional.softplus(decay), torch.sigmoid(beta))
    return head_norm(o, w["o_norm"]).flatten(-2) @ w["out"], total


@pytest.mark.parametrize("bounds", [None, [0, 1, 1, 130, 203]])
def test_training(bounds):
    lead = (2, 150) if bounds is None else (203,)
    g = torch.Generator().manual_seed(7)
    x, residual, d_out, d_total = (torch.randn((*lead, CHANNELS), generator=g) for _ in range(4))
    w = weights(1)
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=DEV)

    def run(to, mix):
        leaves = [to(t).requires_grad_() for t in (x, residual, *w.values())]
        out = layer(dict(zip(w, leaves[2:])), *leaves[:2], mix)
        return [*out, *torch.autograd.grad(out, leaves, [to(d_out), to(d_total)])]
    want = run(lambda t: t.double(), lambda *a: ref.gated_delta(*a, bounds=bounds)[0])
    got = run(lambda t: t.to(DEV), lambda *a: linrec_amd.gated_delta(*a, cu_seqlens=cu))
    share = 4 * ref.bound(torch.float32, torch.float32, 150)
    for name, a, b in zip(("out", "total", "d_x", "d_residual", *("d_" + n for n in w)), got, want):
        ref.assert_near(a, b, share, name)


def test_a_prompt_and_single_tokens():
    """Prompts of a batch side by side, then their next tokens one at a time from rows of a cache: what one pass over all gives."""
    w = {n: t.to(DEV) for n, t in weights(2).items()}
    g = torch.Generator().manual_seed(8)
    prompts, more = [5, 64, 0, 131], 3
    slots = torch.tensor([4, 0, 2, 1], dtype=torch.int32, device=DEV)
    x, residual = (torch.randn((sum(prompts) + more * len(prompts), CHANNELS), generator=g).to(DEV) for _ in range(2))
    ends = torch.tensor([n + more for n in prompts]).cumsum(0)
    starts = ends - torch.tensor([n + more for n in prompts])

    def bounds(lengths):
        return torch.tensor([0, *torch.tensor(lengths).cumsum(0)], dtype=torch.int32, device=DEV)
    with torch.no_grad():
        whole, _ = layer(w, x, residual, lambda *a: linrec_amd.gated_delta(*a, cu_seqlens=bounds([n + more for n in prompts])))
        cache = torch.full((6, HEADS, KEY_DIM, VALUE_DIM), 7.0, device=DEV)
        rows = torch.cat([torch.arange(a, a + n) for a, n in zip(starts.tolist(), prompts)]).to(DEV)

        def prefill(*a):
            o, state = linrec_amd.gated_delta(*a, cu_seqlens=bounds(prompts), return_state=True)
            cache[slots.long()] = state
            return o
        got = [(rows, layer(w, x[rows], residual[rows], prefill)[0])]
        for t in range(more):
            rows = (starts + torch.tensor(prompts) + t).to(DEV)
            got.append((rows, layer(w, x[rows], residual[rows], lambda *a: linrec_amd.gated_delta_step(*a, cache, slots=slots))[0]))
    share = 8 * ref.bound(torch.float32, torch.float32, 134)  # (both sides are off by the layer's)
    for rows, out in got:
        ref.assert_near(out, whole[rows].cpu(), share, "out")
    assert torch.equal(cache[[3, 5]], torch.full_like(cache[[3, 5]], 7.0))


def inputs(n, packed):
    g = torch.Generator(device=DEV).manual_seed(n)
    lead = (40 * n,) if packed else (2, 40 * n)

    def normal(*shape):
        return torch.randn((*lead, *shape), device=DEV, generator=g)
    q, k = (linrec_amd.rms_norm(normal(2, 16)) / 4 for _ in range(2))
    rest = torch.tensor([0, n, n, 40 * n], dtype=torch.int32, device=DEV) if packed else torch.randn((2, 4, 16, 24), device=DEV, generator=g)
    return [q, k, normal(4, 24), -normal(4).abs(), normal(4).sigmoid(), rest]


def delta(q, k, v, log_decay, beta, h0):
    o, state = linrec_amd.gated_delta(q, k, v, log_decay, beta, h0=h0, return_state=True)
    return o * 2, state


def delta_packed(q, k, v, log_decay, beta, cu_seqlens):
    return (linrec_amd.gated_delta(q, k, v, log_decay, beta, cu_seqlens=cu_seqlens),)


def norms(q, k, v, log_decay, beta, h0):
    y, total = linrec_amd.rms_norm(q, k[0, 0, 0] + 1, residual=k)
    return linrec_amd.rms_norm(v), y * 2, total


@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("fn", [delta, delta_packed, norms], ids=lambda f: f.__name__)
def test_a_compiled_training_step(fn, dynamic):
    torch._dynamo.reset()
    compiled = torch.compile(fn, backend="aot_eager", dynamic=dynamic, fullgraph=True)
    for n in (3, 5, 9):
        results = []
        for call in (fn, torch._dynamo.config.patch(error_on_recompile=dynamic and n > 3)(compiled)):
            leaves = [t.clone().requires_grad_() if t.is_floating_point() else t for t in inputs(n, fn is delta_packed)]
            outputs = call(*leaves)
            wanted = [t for t in leaves if t.requires_grad]
            grads = torch.autograd.grad(sum(o.sum() for o in outputs), wanted, allow_unused=True)
            results.append([*outputs, *(t for t in grads if t is not None)])
        assert len(results[0]) == len(results[1]) and all(torch.equal(a, b) for a, b in zip(*results))


def test_compiled_calls_that_serve():
    torch._dynamo.reset()

    def step(q, k, v, log_decay, beta, state, slots):
        y, scales, total = linrec_amd.rms_norm_quantize(v.flatten(1), residual=v.flatten(1))
        return linrec_amd.gated_delta_step(q, k, v, log_decay, beta, state, slots=slots) + 1, y, scales, total
    compiled = torch.compile(step, backend="aot_eager", dynamic=True, fullgraph=True)
    for n in (3, 7):
        q, k, v, log_decay, beta, _ = (t[0, :n] if t.dim() > 1 else t for t in inputs(3, False))
        state = torch.randn((n + 2, 4, 16, 24), device=DEV)
        other, slots = state.clone(), torch.arange(n, 0, -1, dtype=torch.int32, device=DEV)
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip(compiled(q, k, v, log_decay, beta, state, slots), step(q, k, v, log_decay, beta, other, slots)))
        assert torch.equal(state, other)


def test_transforms():
    args = inputs(3, False)[:5]
    got = torch.func.vmap(linrec_amd.gated_delta)(*(torch.stack([t, t * 0.5]) for t in args))
    assert torch.equal(got, torch.stack([linrec_amd.gated_delta(*args), linrec_amd.gated_delta(*(t * 0.5 for t in args))]))
    x = args[2]
    assert torch.equal(torch.func.vmap(linrec_amd.rms_norm)(x), linrec_amd.rms_norm(x))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: linrec_amd.gated_delta(*args[:2], t, *args[3:]).sum())(x)
    with pytest.raises(RuntimeError, match="jvp"):
        torch.func.jvp(linrec_amd.rms_norm, (x,), (x,))
    with pytest.raises(RuntimeError, match="jvp"):
        torch.func.jvp(lambda t: linrec_amd.gated_delta(*args[:2], t, *args[3:]), (x,), (x,))


def test_two_streams_at_once():
    sets = [inputs(20, False), inputs(21, False)]

    def run(args):
        leaves = [t.detach().clone().requires_grad_() for t in args]
        o, state = linrec_amd.gated_delta(*leaves[:5], h0=leaves[5], return_state=True)
        y = linrec_amd.rms_norm(o)
        return [y.detach(), *torch.autograd.grad((y, state), leaves, (torch.ones_like(y), torch.ones_like(state)))]
    want = [run(args) for args in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for n, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[n].append(run(sets[n]))
    torch.cuda.synchronize()
    for n in range(2):
        assert all(torch.equal(a, b) for result in got[n] for a, b in zip(result, want[n]))


def test_a_captured_training_step():
    """Forward and backward in one graph, replayed with new values and eager work between."""
    static = [t.detach().clone() for t in inputs(4, False)]

    def run(args):
        leaves = [t.detach().requires_grad_() for t in args]
        o, state = linrec_amd.gated_delta(*leaves[:5], h0=leaves[5], return_state=True)
        y, total = linrec_amd.rms_norm(o, residual=leaves[2])
        loss_grads = (torch.ones_like(y), total.detach() * 0.5, torch.ones_like(state))
        return [y.detach(), state.detach(), *torch.autograd.grad((y, total, state), leaves, loss_grads)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(static)
    for seed in range(3):
        new = [t * (0.5 + 0.1 * seed) for t in inputs(4, False)]
        for t, value in zip(static, new):
            t.copy_(value)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, run(new)))
        torch.cuda.synchronize()


def test_one_tensor_as_two_arguments():
    """Queries that are the keys, a residual that is x, one gate for both: gradients add up."""
    _, k, v, log_decay, _, _ = inputs(3, False)

    one = [t.clone().requires_grad_() for t in (k, v, log_decay)]
    both = linrec_amd.gated_delta(one[0], one[0], one[1], one[2], one[2])
    y = linrec_amd.rms_norm(both, residual=both)[0]
    d_k, d_v, d_gate = torch.autograd.grad(y, one, torch.ones_like(y))
    o = linrec_amd.gated_delta(k, k, v, log_decay, log_decay)
    many = [t.clone().requires_grad_() for t in (k, v, log_decay, k, log_decay)]
    o_many = linrec_amd.gated_delta(many[3], many[0], many[1], many[2], many[4])
    other = o_many.detach().clone().requires_grad_()
    y2 = linrec_amd.rms_norm(o_many, residual=other)[0]
    d_o = torch.autograd.grad(y2, (o_many, other), torch.ones_like(y2), retain_graph=True)
    grads = torch.autograd.grad(o_many, many, d_o[0] + d_o[1])
    assert torch.equal(o, o_many) and torch.equal(y, y2)
    for got, parts in ((d_k, (grads[0], grads[3])), (d_v, (grads[1],)), (d_gate, (grads[2], grads[4]))):
        ref.assert_near(got, sum(p.double() for p in parts).cpu(), 2.0 ** -22, "gradient")


def test_offsets_beyond_32_bits():
    """Rows a megabyte apart, over 2^31 elements in all, and a cache of more: the same bits as from dense tensors."""
    apart, time = 1 << 20, 2100
    room = torch.empty(time * apart, dtype=torch.bfloat16, device=DEV)

    def far(at, *shape):  # (time, ...) in the rows of `room`
        t = room.as_strided((time, *shape), (apart, *torch.empty(shape, device="meta").stride()), at)
        return t.copy_(torch.randn((time, *shape), device=DEV))
    q, k, v = far(0, 1, 16) / 4, far(64, 1, 16) / 4, far(128, 2, 24)
    q, k = (far(at, 1, 16).copy_(t) for at, t in ((0, q), (64, k)))
    d_o = far(256, 2, 24)
    log_decay, beta = -torch.rand((time, 2), device=DEV), torch.rand((time, 2), device=DEV)
    results = []
    for form in (lambda t: t, lambda t: t.contiguous()):
        leaves = [form(t).detach()[None].requires_grad_() for t in (q, k, v)]
        o = linrec_amd.gated_delta(*leaves, log_decay[None], beta[None])
        y, total = linrec_amd.rms_norm(leaves[2], residual=form(d_o)[None])
        results.append([o, y, total, *torch.autograd.grad((o, y), leaves, (form(d_o)[None], form(d_o)[None]))])
    assert q.stride(0) == apart and all(torch.equal(a, b) for a, b in zip(*results))
    del room, q, k, v, d_o, results, leaves, o, y, total
    rows, dims = 8200, (16, 128, 128)  # 2^31 + 2^21 values
    cache = torch.empty((rows, *dims), device=DEV)
    slots = torch.tensor([rows - 1, 0], dtype=torch.int32, device=DEV)
    start = torch.randn((2, *dims), device=DEV)
    cache[slots.long()] = start
    q, k, v = (torch.randn((2, 16, 128), device=DEV) / 11 for _ in range(3))
    gates = torch.rand((2, 16), device=DEV)
    with torch.no_grad():
        a = linrec_amd.gated_delta_step(q, k, v, -gates, gates, cache, slots=slots)
        b = linrec_amd.gated_delta_step(q, k, v, -gates, gates, start)
    assert torch.equal(a, b) and torch.equal(cache[slots.long()], start)


@pytest.mark.parametrize("which", range(6))
def test_gradients_against_differences(which):
    """Along a random direction of one input, in fp32 with a step h of 2^-5.  f = <o, w> + <state, w'> is off by 8 * 2^-20 * sqrt(3) of its terms
    (2e-5), over h by 6e-4; the third derivative adds h^2 / 6 = 2e-4, and nine times that for a log decay, whose steps add up over the ten
    or so positions that a state remembers.  In all 2e-3 of what such a difference is large, |gradient|; 1e-2 allows for terms larger than that."""
    g = torch.Generator(device=DEV).manual_seed(which)
    q, k, v, log_decay, beta, h0 = (t.detach() for t in inputs(3, False))
    leaves = [t.requires_grad_() for t in (q, k, v, -0.1 - 0.1 * log_decay.abs(), beta, h0)]
    weights = [torch.randn(t.shape, device=DEV, generator=g) for t in (v, h0)]

    def f(args):
        o, state = linrec_amd.gated_delta(*args[:5], h0=args[5], return_state=True)
        return [o, state]
    grad = torch.autograd.grad(f(leaves), leaves[which], weights)[0].double()
    step = torch.randn(grad.shape, device=DEV, generator=g) * 2.0 ** -5
    with torch.no_grad():
        up, down = ([t + s * step if n == which else t for n, t in enumerate(leaves)] for s in (1.0, -1.0))
        change = sum(((a.double() - b.double()) * w.double()).sum() for a, b, w in zip(f(up), f(down), weights)) / 2
    assert abs(float(change - (grad * step).sum())) <= 1e-2 * 2.0 ** -5 * float(grad.norm())
