"""Workloads of the layer operators around the scan: the gated linear recurrence and its single-token step, group norm with an
activation, and the embedding with its gradient, as a recurrent language model calls them.

With `own` false every operator is computed in its plain form, elementary torch operations in 32 bits rounded once at the end;
with `own` true it is the call of this package.  `exact` is the definition in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SCALE = 8.0  # of the recurrence's decay rates, the operator's default

# The largest listed case of each operator, in elements of its activations: drawn cases stay below.
_MAX = {"gated": 8 * 4096 * 2048, "step": 512 * 4096, "norm": 8 * 4096 * 1024, "embedding": 8 * 4096 * 1024}
_MAX_TABLE = 128000 * 1024


def _gated(batch, time, channels, dtype, grad, packed=False, views=False, state=False, reverse=False, **name):
    """packed: `batch` sequences of ragged lengths, `time` positions in all; views: the three inputs are chunks of one
    projection; state: an initial state goes in and the final state comes out."""
    return dict(op="gated", batch=batch, time=time, channels=channels, dtype=dtype, grad=grad, packed=packed, views=views,
                state=state, reverse=reverse, **name)


def _step(batch, slots, channels, dtype, **name):
    """slots: rows of the cache of states, 0 where state and batch rows are the same."""
    return dict(op="step", batch=batch, slots=slots, channels=channels, dtype=dtype, **name)


def _norm(batch, positions, channels, groups, dtype, act, grad, **name):
    return dict(op="norm", batch=batch, positions=positions, channels=channels, groups=groups, dtype=dtype, act=act, grad=grad,
                **name)


def _embedding(tokens, vocab, channels, dtype, grad, padding=False, **name):
    return dict(op="embedding", tokens=tokens, vocab=vocab, channels=channels, dtype=dtype, grad=grad, padding=padding, **name)


def listed():
    return [
        # a recurrent layer's training step in mixed precision, the largest activations
        _gated(8, 4096, 2048, "bf16", True, name="gated_training"),
        # the same in single precision, its three inputs the chunks of one projection
        _gated(16, 2048, 512, "f32", True, views=True, name="gated_training_views"),
        # one very long sequence (audio, genomes) of odd length and width, run backwards in time
        _gated(1, 100001, 250, "bf16", True, reverse=True, name="gated_long_odd"),
        # prompts of different lengths, packed, at the start of serving: states come from a cache and go back
        _gated(37, 20011, 2048, "bf16", False, packed=True, state=True, name="gated_prefill_packed"),
        # one token for one user: what counts is the latency of a call
        _step(1, 0, 1024, "f32", name="step_single"),
        # one token for each running request, their states at any rows of the cache
        _step(512, 1024, 4096, "bf16", name="step_batch"),
        # per-token norm of a recurrence's output over its heads, with the gate's activation, in training
        _norm(8 * 4096, 1, 1024, 16, "bf16", "silu", True, name="norm_tokens"),
        # the usual group norm over all positions of a sequence or an image
        _norm(16, 2048, 512, 32, "f32", "gelu", True, name="norm_positions"),
        # a small odd one at inference
        _norm(3, 333, 222, 6, "bf16", "silu", False, name="norm_small_odd"),
        # the embedding of a training step: tokens distributed like words
        _embedding(8 * 4096, 32000, 1024, "bf16", True, name="embedding_training"),
        # a large vocabulary in single precision, few tokens against it, padding among them
        _embedding(4095, 128000, 333, "f32", True, padding=True, name="embedding_large_vocabulary"),
        # the tokens of one decoding step
        _embedding(64, 32000, 4096, "bf16", False, name="embedding_decode"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm; a third of them are powers of two or
    multiples of 64, the rest are left as they fall, odd ones among them."""
    n = int(round(lo * (hi / lo) ** rng.random()))
    kind = rng.randrange(6)
    if kind == 0:
        n = 1 << max(0, n.bit_length() - 1)
    elif kind == 1 and n >= 64:
        n -= n % 64
    return min(max(n, lo), hi)


def draw(rng):
    op = rng.choice(["gated", "gated", "gated", "step", "norm", "norm", "embedding", "embedding"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    grad = rng.random() < 0.7
    if op == "step":
        channels = _spread(rng, 64, 4096)
        batch = _spread(rng, 1, 512)
        return _step(batch, rng.choice([0, 2 * batch, batch + 7]), channels, dtype)
    elements = _spread(rng, 1 << 16, _MAX[op] // (2 if dtype == "f32" else 1))
    if op == "gated":
        channels = min(_spread(rng, 64, 4096), elements // 16)
        time = _spread(rng, 16, min(100001, elements // channels))
        batch = max(1, min(64, elements // (channels * time)))
        packed = rng.random() < 0.35
        if packed:  # `time` positions of all sequences together
            time, batch = batch * time, _spread(rng, 1, 64)
        return _gated(batch, time, channels, dtype, grad, packed, not packed and rng.random() < 0.4, rng.random() < 0.5,
                      rng.random() < 0.3)
    if op == "norm":
        groups = rng.choice([1, 4, 6, 8, 16, 32])
        channels = groups * max(1, min(_spread(rng, 64, 4096), elements // 16) // groups)
        positions = 1 if rng.random() < 0.4 else _spread(rng, 2, max(2, min(16384, elements // channels)))
        return _norm(max(1, elements // (channels * positions)), positions, channels, groups, dtype,
                     rng.choice(["none", "relu", "silu", "gelu"]), grad)
    channels = _spread(rng, 64, 4096)
    vocab = _spread(rng, 256, min(128000, _MAX_TABLE // channels // (2 if dtype == "f32" else 1)))
    return _embedding(max(1, elements // channels), vocab, channels, dtype, grad, rng.random() < 0.5)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _sequence_starts(case, seed):
    """Bounds of ragged sequences that fill case["time"] positions; now and then one is empty."""
    gen = torch.Generator().manual_seed(seed + 1)
    cuts = torch.sort(torch.randint(0, case["time"] + 1, (case["batch"] - 1,), generator=gen)).values
    return torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.tensor([case["time"]])]).to(torch.int32).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def decay_rates(channels):
        # a trained layer's: exp(-scale softplus(rate)) between 0.9 and 0.999
        slowest = 0.9 + 0.099 * torch.rand(channels, generator=gen, device="cuda")
        return torch.log(torch.expm1(-torch.log(slowest) / _SCALE))

    state = dict(case)
    if case["op"] == "gated":
        channels = case["channels"]
        lead = (case["time"],) if case["packed"] else (case["batch"], case["time"])
        if case["views"]:
            projection = torch.cat([normal(*lead, channels).to(dtype) for _ in range(3)], -1)
            x, gate_a, gate_x = projection.chunk(3, -1)
        else:
            x, gate_a, gate_x = (normal(*lead, channels).to(dtype) for _ in range(3))
        state.update(x=x.detach(), gate_a=gate_a.detach(), gate_x=gate_x.detach(), rate=decay_rates(channels),
                     h0=normal(case["batch"], channels) if case["state"] else None,
                     cu_seqlens=_sequence_starts(case, seed) if case["packed"] else None)
        if case["grad"]:
            state["d_h"] = normal(*lead, channels).to(dtype)
            if case["state"]:
                state["d_state"] = normal(case["batch"], channels)
            for name in ("x", "gate_a", "gate_x", "rate", "h0"):
                if state[name] is not None:
                    state[name].requires_grad_()
    elif case["op"] == "step":
        batch, channels, slots = case["batch"], case["channels"], case["slots"]
        state.update(x=normal(batch, channels).to(dtype), gate_a=normal(batch, channels).to(dtype),
                     gate_x=normal(batch, channels).to(dtype), rate=decay_rates(channels),
                     state=normal(slots or batch, channels),
                     slots=torch.randperm(slots, generator=gen, device="cuda")[:batch].to(torch.int32) if slots else None)
    elif case["op"] == "norm":
        lead = (case["batch"],) if case["positions"] == 1 else (case["batch"], case["positions"])
        channels = case["channels"]
        state.update(x=(normal(*lead, channels) + 0.5).to(dtype), weight=1.0 + 0.2 * normal(channels), bias=0.2 * normal(channels))
        if case["grad"]:
            state["d_y"] = normal(*lead, channels).to(dtype)
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_()
    else:
        vocab, channels, n = case["vocab"], case["channels"], case["tokens"]
        # frequencies that fall like 1 / rank, as words' do; ranks are scattered over the table
        rank = torch.exp(torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * math.log(vocab)).long().clamp_(1, vocab) - 1
        tokens = torch.randperm(vocab, generator=gen, device="cuda")[rank]
        padding_idx = None
        if case["padding"]:  # the ends of the batch's shorter sequences
            padding_idx = 0
            tokens[torch.rand(n, generator=gen, device="cuda") < 0.1] = padding_idx
        state.update(tokens=tokens, weight=normal(vocab, channels).mul_(channels ** -0.5).to(dtype), scale=math.sqrt(channels),
                     padding_idx=padding_idx)
        if case["grad"]:
            state["d_y"] = normal(n, channels).to(dtype)
            state["weight"].requires_grad_()
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)[state["op"]](state)


def _own_gated(s):
    import linrec_amd
    h = linrec_amd.gated_linrec(s["x"], s["gate_a"], s["gate_x"], s["rate"], h0=s["h0"], cu_seqlens=s["cu_seqlens"],
                                reverse=s["reverse"], return_state=s["state"])
    h, last = h if s["state"] else (h, None)
    outputs = [h] if last is None else [h, last]
    if not s["grad"]:
        return outputs
    wanted = [s[name] for name in ("x", "gate_a", "gate_x", "rate", "h0") if s[name] is not None]
    d_outputs = [s["d_h"]] if last is None else [s["d_h"], s["d_state"]]
    return [*(o.detach() for o in outputs), *torch.autograd.grad(outputs, wanted, d_outputs)]


def _own_step(s):
    import linrec_amd
    h = linrec_amd.gated_linrec_step(s["x"], s["gate_a"], s["gate_x"], s["rate"], s["state"], slots=s["slots"])
    return [h, s["state"]]


def _own_norm(s):
    import linrec_amd
    y = linrec_amd.group_norm_act(s["x"], s["groups"], s["weight"], s["bias"], act=s["act"])
    if not s["grad"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["d_y"])]


def _own_embedding(s):
    import linrec_amd
    y = linrec_amd.embedding(s["tokens"], s["weight"], scale=s["scale"], padding_idx=s["padding_idx"])
    if not s["grad"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, (s["weight"],), s["d_y"])]


_run_own = {"gated": _own_gated, "step": _own_step, "norm": _own_norm, "embedding": _own_embedding}


def _softplus(t):
    return torch.clamp(t, min=0.0) + torch.log1p(torch.exp(-torch.abs(t)))


def _gates(x, gate_a, gate_x, rate):
    sig_a, sig_x = torch.sigmoid(gate_a), torch.sigmoid(gate_x)
    log_a = -_SCALE * _softplus(rate) * sig_a
    return sig_a, sig_x, log_a, torch.exp(log_a), torch.sqrt(-torch.expm1(2.0 * log_a))


def _scan(coeffs, inputs):
    """inputs[t] += coeffs[t] * (value at t - 1) along dimension 1, by doubling."""
    a, b = coeffs.clone(), inputs.clone()
    d = 1
    while d < b.shape[1]:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return b


def _ends(s, time):
    """(batch rows, positions) at which the sequences start and end in scan order, and which sequences have any."""
    device = s["x"].device
    if s["cu_seqlens"] is None:
        batch = torch.arange(s["batch"], device=device)
        return batch, torch.zeros_like(batch), torch.full_like(batch, time - 1), batch
    bounds = s["cu_seqlens"].long()
    if s["reverse"]:
        bounds = time - bounds.flip(0)
    some = torch.nonzero(bounds[1:] > bounds[:-1]).flatten()
    row = torch.zeros_like(some)
    sequence = s["batch"] - 1 - some if s["reverse"] else some
    return row, bounds[:-1][some], bounds[1:][some] - 1, sequence


def _plain_gated(s):
    def forward_in_time(t):
        t = t.detach().float()
        t = t if t.dim() == 3 else t[None]
        return t.flip(1) if s["reverse"] else t

    def back(t, dtype):
        t = t.flip(1) if s["reverse"] else t
        return (t[0] if s["packed"] else t).to(dtype)

    dtype = s["x"].dtype
    x, rate = forward_in_time(s["x"]), s["rate"].detach()
    sig_a, sig_x, log_a, a, m = _gates(x, forward_in_time(s["gate_a"]), forward_in_time(s["gate_x"]), rate)
    b = m * sig_x * x
    time = x.shape[1]
    row, first, last, sequence = _ends(s, time)
    h0 = s["h0"].detach() if s["state"] else torch.zeros(s["batch"], x.shape[2], device=x.device)
    coeffs, inputs = a.clone(), b.clone()
    inputs[row, first] += a[row, first] * h0[sequence]
    coeffs[row, first] = 0.0
    h = _scan(coeffs, inputs)
    outputs = [back(h, dtype)]
    if s["state"]:
        final = h0.clone()
        final[sequence] = h[row, last]
        outputs.append(final)
    if not s["grad"]:
        return outputs
    d_h = forward_in_time(s["d_h"]).clone()
    if s["state"]:
        d_h[row, last] += s["d_state"][sequence]
    following = torch.cat([coeffs[:, 1:], torch.zeros_like(coeffs[:, :1])], 1)
    g = _scan(following.flip(1), d_h.flip(1)).flip(1)
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    before[row, first] = h0[sequence]
    p = g * (log_a * a * before - sig_x * x * a * a * log_a / m)
    outputs += [back(g * m * sig_x, dtype), back(p * (1.0 - sig_a), dtype), back(g * m * x * sig_x * (1.0 - sig_x), dtype),
                p.sum((0, 1)) * torch.sigmoid(rate) / _softplus(rate)]
    if s["state"]:
        d_h0 = s["d_state"].clone()
        d_h0[sequence] = a[row, first] * g[row, first]
        outputs.append(d_h0)
    return outputs


def _plain_step(s):
    x = s["x"].float()
    _, sig_x, _, a, m = _gates(x, s["gate_a"].float(), s["gate_x"].float(), s["rate"])
    rows = s["slots"].long() if s["slots"] is not None else torch.arange(x.shape[0], device=x.device)
    h = a * s["state"][rows] + m * sig_x * x
    s["state"][rows] = h
    return [h.to(s["x"].dtype), s["state"]]


def _activate(z, act):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.clamp(z, min=0.0), (z > 0).to(z.dtype)
    if act == "silu":
        sig = torch.sigmoid(z)
        return z * sig, sig * (1.0 + z * (1.0 - sig))
    cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_norm(s, eps=1e-5):
    dtype, shape = s["x"].dtype, s["x"].shape
    grouped = (s["batch"], s["positions"], s["groups"], s["channels"] // s["groups"])
    x = s["x"].detach().float().reshape(grouped)
    weight, bias = (s[name].detach().float().reshape(grouped[2:]) for name in ("weight", "bias"))
    centred = x - x.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean((1, 3), keepdim=True) + eps)
    xh = centred * rstd
    y, slope = _activate(xh * weight + bias, s["act"])
    outputs = [y.reshape(shape).to(dtype)]
    if not s["grad"]:
        return outputs
    e = s["d_y"].float().reshape(grouped) * slope
    ew = e * weight
    dx = rstd * (ew - ew.mean((1, 3), keepdim=True) - xh * (ew * xh).mean((1, 3), keepdim=True))
    return outputs + [dx.reshape(shape).to(dtype), (e * xh).sum((0, 1)).reshape(-1).to(s["weight"].dtype),
                      e.sum((0, 1)).reshape(-1).to(s["bias"].dtype)]


def _plain_embedding(s):
    weight = s["weight"].detach()
    y = (weight[s["tokens"]].float() * s["scale"]).to(weight.dtype)
    if not s["grad"]:
        return [y]
    d_weight = torch.zeros(weight.shape, device=weight.device)
    d_weight.index_add_(0, s["tokens"], s["d_y"].float())
    if s["padding_idx"] is not None:
        d_weight[s["padding_idx"]] = 0.0
    return [y, (d_weight * s["scale"]).to(weight.dtype)]


_run_plain = {"gated": _plain_gated, "step": _plain_step, "norm": _plain_norm, "embedding": _plain_embedding}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    channels = case["channels"]
    if case["op"] == "gated":
        positions = case["time"] * (1 if case["packed"] else case["batch"])
        rows = case["batch"] * channels * 4 * case["state"]
        if not case["grad"]:
            return {"bytes": 4 * positions * channels * size + 2 * rows + 4 * channels, "flops": 25 * positions * channels}
        return {"bytes": 8 * positions * channels * size + 4 * rows + 8 * channels, "flops": 70 * positions * channels}
    if case["op"] == "step":
        n = case["batch"] * channels
        return {"bytes": n * (4 * size + 8) + 4 * channels + 4 * case["batch"] * bool(case["slots"]), "flops": 25 * n}
    if case["op"] == "norm":
        n = case["batch"] * case["positions"] * channels
        if not case["grad"]:
            return {"bytes": 2 * n * size + 8 * channels, "flops": 15 * n}
        return {"bytes": 4 * n * size + 16 * channels, "flops": 45 * n}
    n = case["tokens"] * channels
    # rows of the table that are looked up more than once are read once
    distinct = min(case["tokens"], case["vocab"]) * channels
    bytes_forward = 8 * case["tokens"] + size * (distinct + n)
    if not case["grad"]:
        return {"bytes": bytes_forward, "flops": n}
    return {"bytes": bytes_forward + size * (n + case["vocab"] * channels), "flops": 2 * n + case["vocab"] * channels}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def _recur64(a, b, start, first):
    """h[t] = a[t] h[t-1] + b[t], position after position within blocks that run side by side, then block after block.
    a, b: (time, channels); `first`: positions that start a sequence, `start` the values before them."""
    time, channels = a.shape
    b = b.clone()
    b[first] += a[first] * start
    a = a.clone()
    a[first] = 0.0
    block = max(1, int(math.sqrt(time)))
    blocks = -(-time // block)
    pad = blocks * block - time
    a = torch.cat([a, torch.ones(pad, channels, dtype=a.dtype, device=a.device)]).reshape(blocks, block, channels)
    b = torch.cat([b, torch.zeros(pad, channels, dtype=b.dtype, device=b.device)]).reshape(blocks, block, channels)
    for t in range(1, block):
        b[:, t] += a[:, t] * b[:, t - 1]
        a[:, t] *= a[:, t - 1]
    for k in range(1, blocks):
        b[k] += a[k] * b[k - 1, -1]
    return b.reshape(blocks * block, channels)[:time]


def _exact_gated(case, state):
    packed = case["packed"]
    names = ("x", "gate_a", "gate_x")
    x, gate_a, gate_x = (state[name].detach().double().reshape(-1, case["channels"]) for name in names)
    rate = state["rate"].detach().double()
    positions = x.shape[0]
    if packed:
        bounds = state["cu_seqlens"].tolist()
    else:
        bounds = [n * case["time"] for n in range(case["batch"] + 1)]
    # sequence n occupies [bounds[n], bounds[n + 1]); a reversed scan enters it at its far end
    with_positions = [n for n in range(case["batch"]) if bounds[n + 1] > bounds[n]]
    low = torch.tensor([bounds[n] for n in with_positions], device=x.device)
    high = torch.tensor([bounds[n + 1] - 1 for n in with_positions], device=x.device)
    which = torch.tensor(with_positions, device=x.device)
    enter, leave = (high, low) if case["reverse"] else (low, high)
    h0 = state["h0"].detach().double() if case["state"] else x.new_zeros(case["batch"], case["channels"])

    def recur(a, b, start, at, backwards):
        if not backwards:
            return _recur64(a, b, start, at)
        return _recur64(a.flip(0), b.flip(0), start, positions - 1 - at).flip(0)

    decay = _SCALE * torch.logaddexp(rate, torch.zeros_like(rate))
    keep = 1.0 / (1.0 + torch.exp(-gate_a))
    take = 1.0 / (1.0 + torch.exp(-gate_x))
    a = torch.exp(-decay * keep)
    m = torch.sqrt(-torch.expm1(-2.0 * decay * keep))
    h = recur(a, m * take * x, h0[which], enter, case["reverse"])
    shape = state["x"].shape
    outputs = [h.reshape(shape)]
    if case["state"]:
        final = h0.clone()
        final[which] = h[leave]
        outputs.append(final)
    if not case["grad"]:
        return outputs
    # the gradient that arrives at h[t] goes on to the position before with the coefficient of t
    step = -1 if case["reverse"] else 1
    on = torch.roll(a, -step, 0)  # the coefficient of the position after t in scan order; not used at a sequence's end
    d_h = state["d_h"].double().reshape(x.shape)
    beyond = x.new_zeros(len(with_positions), case["channels"])
    if case["state"]:
        beyond = state["d_state"].double()[which]
    on[leave] = 1.0
    g = recur(on, d_h, beyond, leave, not case["reverse"])
    previous = torch.roll(h, step, 0)
    previous[enter] = h0[which]
    # d a from h = a h' + sqrt(1 - a^2) take x, and d decay*keep = -a d a
    d_exponent = g * (-a * previous + take * x * a * a / m)
    outputs += [(g * m * take).reshape(shape), (d_exponent * decay * keep * (1.0 - keep)).reshape(shape),
                (g * m * x * take * (1.0 - take)).reshape(shape),
                (d_exponent * keep).sum(0) * _SCALE / (1.0 + torch.exp(-rate))]
    if case["state"]:
        d_h0 = state["d_state"].double().clone()
        d_h0[which] = a[enter] * g[enter]
        outputs.append(d_h0)
    return outputs


def _exact_step(case, state):
    x, gate_a, gate_x, rate = (state[name].double() for name in ("x", "gate_a", "gate_x", "rate"))
    exponent = _SCALE * torch.logaddexp(rate, torch.zeros_like(rate)) / (1.0 + torch.exp(-gate_a))
    cache = state["state"].double()
    rows = state["slots"].tolist() if state["slots"] is not None else list(range(case["batch"]))
    h = torch.exp(-exponent) * cache[rows] + torch.sqrt(-torch.expm1(-2.0 * exponent)) * x / (1.0 + torch.exp(-gate_x))
    cache[rows] = h
    return [h, cache]


def _exact_norm(case, state):
    groups, eps = case["groups"], 1e-5
    x = state["x"].detach().double().reshape(case["batch"], case["positions"], groups, -1).movedim(2, 1)  # (n, group, position, channel)
    weight, bias = (state[name].detach().double().reshape(1, groups, 1, -1) for name in ("weight", "bias"))
    x, weight, bias = (t.clone().requires_grad_(case["grad"]) for t in (x, weight, bias))
    with torch.enable_grad():
        variance, mean = torch.var_mean(x, (2, 3), correction=0, keepdim=True)
        z = (x - mean) / torch.sqrt(variance + eps) * weight + bias
        if case["act"] == "relu":
            y = torch.where(z > 0, z, torch.zeros_like(z))
        elif case["act"] == "silu":
            y = z / (1.0 + torch.exp(-z))
        elif case["act"] == "gelu":
            y = 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
        else:
            y = z

    def back(t):
        return t.detach().movedim(1, 2).reshape(state["x"].shape)

    if not case["grad"]:
        return [back(y)]
    d_y = state["d_y"].double().reshape(case["batch"], case["positions"], groups, -1).movedim(2, 1)
    d_x, d_weight, d_bias = torch.autograd.grad(y, (x, weight, bias), d_y)
    return [back(y), back(d_x), d_weight.reshape(-1), d_bias.reshape(-1)]


def _exact_embedding(case, state):
    weight = state["weight"].detach().double()
    y = weight[state["tokens"]] * state["scale"]
    if not case["grad"]:
        return [y]
    rows = state["d_y"].double() * state["scale"]
    if state["padding_idx"] is not None:
        rows[state["tokens"] == state["padding_idx"]] = 0.0
    return [y, torch.zeros_like(weight).index_add_(0, state["tokens"], rows)]


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"gated": _exact_gated, "step": _exact_step, "norm": _exact_norm, "embedding": _exact_embedding}[case["op"]](case, state)
