"""The gated delta rule in float64 by its definition, position after position, and the error bounds its tests use.

A value that is computed goes through about eight roundings of operands a chunk of 64 positions (K S, M, its right side, N, twice each
where the gradient is concerned), which add up like independent numbers, and so do the chunks that a state remembers.  With 16-bit inputs
an operand is two numbers of 8 bits, off by 2^-18 at most; in fp32 what counts is the sum of up to 256 products, 2^-24 each that add up
to 2^-20.  Inverses and decays may make a few times as much of it.  So a result is 8 u sqrt(2 + chunks) off in norm, with u as said, and
half a step of its own type more.

That is of the terms a result is the sum of, which are of about the size of the inputs (states, values and gradients of unit variance,
keys of unit length), one.  The terms of a single value may cancel: d_h0 = e^g d_state + scale q d_o - e^g beta k d_v of one position
and one channel is 1.6 - 1.6 = 0.0265 for one seed, and two terms that are 2^-18 off leave 2 * 1.6 * 2^-18 = 1.2e-5 or 4.6e-4 of the
difference.  Those of n values do not all cancel; so the norm that a tensor's error is measured with is at least that of one value
that has the size of its terms, n^-1/2 for each.  The gradient of a log decay is the inner product of a state and its gradient, key_dim value_dim
terms whose signs are random: their sum is of size sqrt(key_dim value_dim) and may cancel as well (0.02 of 64 for a seed with two
positions of 64 x 64; 4096 terms, each 2^-18 off, are 64 * 2^-18 = 2.4e-4 off together)."""
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _loop(q, k, v, log_decay, beta, s, scale):
    out = []
    for t in range(q.shape[0]):
        s = torch.exp(log_decay[t])[:, None, None] * s
        new = beta[t][:, None] * (v[t] - (k[t][:, :, None] * s).sum(-2))
        s = s + k[t][:, :, None] * new[:, None, :]
        out.append(scale * (q[t][:, :, None] * s).sum(-2))
    return out, s


def gated_delta(q, k, v, log_decay, beta, h0=None, bounds=None, scale=None):
    """(o, state) in float64; tensors (batch, time, heads, ...), or (positions, heads, ...) with `bounds`."""
    shape = v.shape
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    q, k, v, log_decay, beta = (t.double() for t in (q, k, v, log_decay, beta))
    shared = v.shape[-2] // q.shape[-2]
    q, k = (t.repeat_interleave(shared, -2) for t in (q, k))
    if bounds is None:
        sequences = [tuple(t[n] for t in (q, k, v, log_decay, beta)) for n in range(shape[0])]
    else:
        sequences = [tuple(t[lo:hi] for t in (q, k, v, log_decay, beta)) for lo, hi in zip(bounds[:-1], bounds[1:])]
    out, states = [], []
    for n, parts in enumerate(sequences):
        s = torch.zeros(shape[-2], q.shape[-1], shape[-1], dtype=torch.float64) if h0 is None else h0[n].double()
        rows, s = _loop(*parts, s, scale)
        out += rows
        states.append(s)
    return torch.stack(out).reshape(shape) if out else v, torch.stack(states)


def bound(dtype, inputs, time):
    """How far a result of type `dtype` may be off in norm, of inputs of type `inputs`."""
    u = 2.0 ** -20 if inputs == torch.float32 else 2.0 ** -18
    return HALF_STEP[dtype] + 8 * u * (2 + time / 64) ** 0.5


def assert_near(got, want, share, what, size=1.0):
    """|got - want| within `share` of want in norm (at least that of one term, `size`), and none of its values off by more than 16 times what
    that is for each."""
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    if not got.numel():
        return
    each = max(float(want.norm()), size) / want.numel() ** 0.5
    off = (got - want).abs()
    rms = float(off.norm()) / off.numel() ** 0.5
    assert rms <= share * each, f"{what}: {rms / each:.3g} off in norm, {share:.3g} is allowed"
    worst = float((off / torch.clamp(want.abs(), min=each)).max())
    assert worst <= 16 * share, f"{what}: a value is {worst:.3g} off, {16 * share:.3g} is allowed"
