"""Plain 64-bit forms of the layer operators on the CPU, and the error bounds their tests use.

The bounds come from the operations, not from what a run gave: u is the rounding unit of a type, fp32 arithmetic in K
dependent roundings is K u off, and a recurrence with coefficients up to a_max multiplies what a coefficient is off by
1 / (1 - a_max)."""
import torch

U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gated(x, gate_a, gate_x, rate, h0=None, bounds=None, reverse=False, scale=8.0):
    """(h, state, a) in float64 by the loop over positions; x (batch, time, channels), or (positions, channels) with `bounds`."""
    x, gate_a, gate_x, rate = (t.double() for t in (x, gate_a, gate_x, rate))
    log_a = -scale * torch.nn.functional.softplus(rate, threshold=1e9) * torch.sigmoid(gate_a)
    a = torch.exp(log_a)
    b = torch.sqrt(-torch.expm1(2 * log_a)) * torch.sigmoid(gate_x) * x
    if bounds is None:
        spans = [((n,), range(x.shape[1])) for n in range(x.shape[0])]
    else:
        spans = [((), range(lo, hi)) for lo, hi in zip(bounds[:-1], bounds[1:])]
    values, state = {}, []
    for n, (lead, positions) in enumerate(spans):
        h = torch.zeros_like(rate) if h0 is None else h0[n].double()
        for t in (reversed(positions) if reverse else positions):
            h = a[lead + (t,)] * h + b[lead + (t,)]
            values[lead + (t,)] = h
        state.append(h)
    if bounds is None:
        rows = [torch.stack([values[n, t] for t in range(x.shape[1])]) if x.shape[1] else x[n] for n in range(x.shape[0])]
        out = torch.stack(rows) if rows else x
    else:
        out = torch.stack([values[t,] for t in range(x.shape[0])]) if x.shape[0] else x
    return out, torch.stack(state) if state else x.new_zeros(0, rate.numel()), a


def gated_tolerance(a, dtype):
    """Share of the largest value that h may be off.  A coefficient carries about 8 roundings (two of the sigmoid, product,
    exponential), its input as many; both are carried on for 1 / (1 - a) positions, in a sequence of that many at most."""
    if a.numel() == 0:
        return 1.0
    reach = min(1.0 / max(1e-12, 1.0 - float(a.detach().max())), float(a.shape[-2]))
    return UNIT[dtype] + 8 * U32 * (2.0 + reach)


def act(z, name):
    if name == "relu":
        return torch.relu(z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return torch.nn.functional.gelu(z)
    return z


def group_norm_act(x, groups, weight, bias, eps, name):
    """float64, (batch, ..., channels)"""
    shape = x.shape
    v = x.double().reshape(shape[0], -1, groups, shape[-1] // groups)
    var, mean = torch.var_mean(v, (1, 3), correction=0, keepdim=True)
    z = ((v - mean) / torch.sqrt(var + eps)).reshape(shape)
    if weight is not None:
        z = z * weight.double() + bias.double()
    return act(z, name)


def embedding(tokens, weight, scale):
    inside = (tokens >= 0) & (tokens < weight.shape[0])
    rows = weight.double()[torch.where(inside, tokens, torch.zeros_like(tokens)).long()] * scale
    return torch.where(inside[..., None], rows, torch.zeros_like(rows))


def embedding_grad(d_y, tokens, vocab, scale, padding_idx=None):
    """(gradient, sum of the absolute values of the terms, terms of each row), float64"""
    flat, rows = tokens.reshape(-1).long(), d_y.double().reshape(-1, d_y.shape[-1]) * scale
    keep = (flat >= 0) & (flat < vocab)
    if padding_idx is not None:
        keep &= flat != padding_idx
    flat, rows = flat[keep], rows[keep]
    zero = torch.zeros(vocab, d_y.shape[-1], dtype=torch.float64)
    count = torch.zeros(vocab, dtype=torch.float64).index_add_(0, flat, torch.ones(flat.numel(), dtype=torch.float64))
    return zero.index_add(0, flat, rows), zero.index_add(0, flat, rows.abs()), count[:, None]


def assert_within(got, want, bound, what):
    """|got - want| <= bound everywhere (a number, or a tensor of want's size); the same places are NaN or infinite."""
    got = got.detach().double().cpu()
    want = want.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite), f"{what}: not finite in other places"
    off = torch.where(finite, (got - want).abs(), torch.zeros_like(want))
    worst = float((off / (torch.as_tensor(bound, dtype=torch.float64) + 1e-300)).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound, {float(off.max()):.3g} off"


def largest(t):
    finite = t.detach().double().abs()
    finite = finite[torch.isfinite(finite)]
    return float(finite.max()) if finite.numel() else 0.0


def sigmoid_over_softplus(rate):
    rate = rate.double()
    return torch.sigmoid(rate) / torch.nn.functional.softplus(rate, threshold=1e9)


def same_bits_in_a_graph(run):
    """`run` (launches of this library, no autograd) gives the same bits every time: eagerly, on another stream, and in each of
    several replays of a graph with eager work between them."""
    want = [t.clone() for t in run()]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = run()
    for _ in range(3):
        for t in captured:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))
        run()
        torch.cuda.synchronize()
