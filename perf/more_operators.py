"""Workloads of the gated delta rule (a recurrence whose state is a matrix), its single-token step, and the root-mean-square norm
before and inside such a layer, with the residual's addition and with an output in 8 bits, as a recurrent language model calls them.

With `own` false every operator is computed in its plain form, elementary torch operations in 32 bits rounded once at the end
(sums of log decays in 64); with `own` true it is the call of this package.  `exact` is the definition in 64 bits.
"""
import math

import torch

own = False

_device = "cuda"
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_CHUNK = 64  # positions that the plain form takes at once
_QUANTIZED = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}

# The largest listed case of each operator: drawn cases stay below.
_MAX_DELTA = 8 * 4096 * 16 * 128 * 128  # positions x heads x key_dim x value_dim
_MAX_TIME = 32769
_MAX_STEP = 256 * 16 * 128 * 128
_MAX_NORM = 8 * 4096 * 2048


def _delta(batch, time, key_heads, heads, key_dim, value_dim, dtype, grad, packed=False, views=False, state=False, **name):
    """packed: `batch` sequences of ragged lengths, `time` positions in all; views: q, k and v are parts of one projection;
    state: an initial state goes in and the final state comes out."""
    return dict(op="delta", batch=batch, time=time, key_heads=key_heads, heads=heads, key_dim=key_dim, value_dim=value_dim,
                dtype=dtype, grad=grad, packed=packed, views=views, state=state, **name)


def _step(batch, slots, key_heads, heads, key_dim, value_dim, dtype, **name):
    """slots: rows of the cache of states, 0 where state and batch rows are the same."""
    return dict(op="step", batch=batch, slots=slots, key_heads=key_heads, heads=heads, key_dim=key_dim, value_dim=value_dim,
                dtype=dtype, **name)


def _norm(rows, channels, dtype, residual, grad, **name):
    return dict(op="norm", rows=rows, channels=channels, dtype=dtype, residual=residual, grad=grad, **name)


def _quantize(rows, channels, dtype, residual, to, **name):
    return dict(op="quantize", rows=rows, channels=channels, dtype=dtype, residual=residual, to=to, **name)


def listed():
    return [
        # a layer's training step in mixed precision: two value heads share a key head
        _delta(8, 4096, 8, 16, 128, 128, "bf16", True, name="delta_training"),
        # a small model's in single precision, q, k and v parts of one projection
        _delta(4, 1000, 6, 6, 64, 64, "f32", True, views=True, name="delta_training_views"),
        # one very long sequence of odd length with few heads of odd sizes: little runs side by side
        _delta(1, 32769, 2, 4, 100, 72, "bf16", True, name="delta_long_odd"),
        # prompts of different lengths, packed, at the start of serving: states come from a cache and go back
        _delta(37, 20011, 16, 16, 128, 128, "bf16", False, packed=True, state=True, name="delta_prefill_packed"),
        # one token for one user: what counts is the latency of a call
        _step(1, 0, 8, 16, 128, 128, "bf16", name="step_single"),
        # one token for each running request, their states at any rows of the cache
        _step(256, 512, 16, 16, 128, 128, "bf16", name="step_batch"),
        # the norm before a layer, which also adds the residual, in training
        _norm(8 * 4096, 2048, "bf16", True, True, name="norm_residual_training"),
        # the norm of every head's keys, short rows, in single precision
        _norm(16 * 2048 * 8, 64, "f32", False, True, name="norm_heads_training"),
        # a small odd one at inference
        _norm(333, 222, "bf16", True, False, name="norm_small_odd"),
        # the norm of a prompt's positions before a product in 8 bits
        _quantize(20011, 4096, "bf16", True, "e4m3", name="quantize_prefill"),
        # that of one decoding step
        _quantize(64, 4096, "bf16", True, "int8", name="quantize_decode"),
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


def _head_sizes(rng):
    key_heads, shared = rng.choice([1, 2, 4, 6, 8, 16]), rng.choice([1, 1, 2, 4])
    return dict(key_heads=key_heads, heads=key_heads * shared, key_dim=rng.choice([64, 128, 128, 256, _spread(rng, 16, 256)]),
                value_dim=rng.choice([64, 128, 128, 256, _spread(rng, 16, 256)]))


def draw(rng):
    op = rng.choice(["delta", "delta", "delta", "step", "norm", "norm", "quantize"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op in ("norm", "quantize"):
        elements = _spread(rng, 1 << 14, _MAX_NORM // (2 if dtype == "f32" else 1))
        channels = _spread(rng, 32, 8192)
        rows, residual = max(1, elements // channels), rng.random() < 0.6
        if op == "norm":
            return _norm(rows, channels, dtype, residual, rng.random() < 0.7)
        return _quantize(rows, channels, dtype, residual, rng.choice(["int8", "e4m3"]))
    sizes = _head_sizes(rng)
    state = sizes["heads"] * sizes["key_dim"] * sizes["value_dim"]
    if op == "step":
        batch = _spread(rng, 1, min(256, _MAX_STEP // state))
        return _step(batch, rng.choice([0, 2 * batch, batch + 7]), dtype=dtype, **sizes)
    positions = _spread(rng, 16, min(8 * 4096, _MAX_DELTA // state // (4 if dtype == "f32" else 1)))
    time = min(_spread(rng, 16, _MAX_TIME), positions)
    batch, packed = max(1, min(64, positions // time)), rng.random() < 0.35
    if packed:  # `time` positions of all sequences together
        time, batch = batch * time, _spread(rng, 1, min(24, batch * time))
    return _delta(batch, time, dtype=dtype, grad=rng.random() < 0.7, packed=packed, views=not packed and rng.random() < 0.4,
                  state=rng.random() < 0.5, **sizes)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _sequence_bounds(case, seed):
    """Bounds of ragged sequences that fill case["time"] positions, on the host; now and then one is empty."""
    gen = torch.Generator().manual_seed(seed + 1)
    cuts = torch.sort(torch.randint(0, case["time"] + 1, (case["batch"] - 1,), generator=gen)).values
    return [0, *cuts.tolist(), case["time"]]


def prepare(case, seed):
    gen = torch.Generator(device=_device).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    state = dict(case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=_device)

    def unit(*shape):
        rows = normal(*shape)
        return rows / torch.sqrt((rows * rows).sum(-1, keepdim=True))

    if case["op"] in ("norm", "quantize"):
        rows, channels = case["rows"], case["channels"]
        state.update(x=normal(rows, channels).to(dtype), weight=1.0 + 0.2 * normal(channels),
                     residual=(2.0 * normal(rows, channels)).to(dtype) if case["residual"] else None)
        if case.get("grad"):
            state["d_y"] = normal(rows, channels).to(dtype)
            state["d_total"] = normal(rows, channels).to(dtype) if case["residual"] else None
            for name in ("x", "weight", "residual"):
                if state[name] is not None:
                    state[name].requires_grad_()
        return state
    step = case["op"] == "step"
    key_heads, heads, key_dim, value_dim = (case[n] for n in ("key_heads", "heads", "key_dim", "value_dim"))
    lead = (case["batch"],) if step else (case["time"],) if case["packed"] else (case["batch"], case["time"])
    q, k, v = unit(*lead, key_heads, key_dim).to(dtype), unit(*lead, key_heads, key_dim).to(dtype), normal(*lead, heads, value_dim).to(dtype)
    if case.get("views"):
        widths = (key_heads * key_dim, key_heads * key_dim, heads * value_dim)
        projection = torch.cat([t.flatten(-2) for t in (q, k, v)], -1)
        q, k, v = (t.unflatten(-1, (n, -1)) for t, n in zip(projection.split(widths, -1), (key_heads, key_heads, heads)))
    # a trained layer's: heads that forget within two positions and heads that remember for hundreds, each more or less by the token
    pace = torch.exp(math.log(0.002) + (math.log(0.5) - math.log(0.002)) * torch.rand(heads, generator=gen, device=_device))
    state.update(q=q.detach(), k=k.detach(), v=v.detach(), log_decay=-pace * _softplus(normal(*lead, heads)),
                 beta=torch.sigmoid(normal(*lead, heads)))
    if step:
        slots = case["slots"]
        state.update(state=0.3 * normal(slots or case["batch"], heads, key_dim, value_dim),
                     slots=torch.randperm(slots, generator=gen, device=_device)[:case["batch"]].to(torch.int32) if slots else None)
        return state
    bounds = _sequence_bounds(case, seed) if case["packed"] else None
    state.update(h0=0.3 * normal(case["batch"], heads, key_dim, value_dim) if case["state"] else None, bounds=bounds,
                 cu_seqlens=torch.tensor(bounds, dtype=torch.int32, device=_device) if bounds else None)
    if case["grad"]:
        state["d_o"] = normal(*lead, heads, value_dim).to(dtype)
        if case["state"]:
            state["d_state"] = normal(case["batch"], heads, key_dim, value_dim)
        for name in ("q", "k", "v", "log_decay", "beta", "h0"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)[state["op"]](state)


def _own_delta(s):
    import linrec_amd
    o = linrec_amd.gated_delta(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], h0=s["h0"], cu_seqlens=s["cu_seqlens"],
                               return_state=s["state"])
    o, last = o if s["state"] else (o, None)
    outputs = [o] if last is None else [o, last]
    if not s["grad"]:
        return outputs
    wanted = [s[name] for name in ("q", "k", "v", "log_decay", "beta", "h0") if s[name] is not None]
    d_outputs = [s["d_o"]] if last is None else [s["d_o"], s["d_state"]]
    return [*(t.detach() for t in outputs), *torch.autograd.grad(outputs, wanted, d_outputs)]


def _own_step(s):
    import linrec_amd
    o = linrec_amd.gated_delta_step(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["state"], slots=s["slots"])
    return [o, s["state"]]


def _own_norm(s):
    import linrec_amd
    y = linrec_amd.rms_norm(s["x"], s["weight"], residual=s["residual"])
    outputs = list(y) if s["residual"] is not None else [y]
    if not s["grad"]:
        return outputs
    wanted = [s[name] for name in ("x", "residual", "weight") if s[name] is not None]
    d_outputs = [s["d_y"]] if s["residual"] is None else [s["d_y"], s["d_total"]]
    return [*(t.detach() for t in outputs), *torch.autograd.grad(outputs, wanted, d_outputs)]


def _own_quantize(s):
    import linrec_amd
    q, scales, *total = linrec_amd.rms_norm_quantize(s["x"], s["weight"], residual=s["residual"], dtype=_QUANTIZED[s["to"]][0])
    return [_worth(q, scales, s["x"].dtype), scales, *total]


_run_own = {"delta": _own_delta, "step": _own_step, "norm": _own_norm, "quantize": _own_quantize}


def _worth(q, scales, dtype):
    """The values that whole numbers in 8 bits stand for; floating ones are values already."""
    if q.is_floating_point():
        return q
    return torch.mul(q, scales[:, None], out=torch.empty(q.shape, dtype=dtype, device=q.device))


def _softplus(t):
    return torch.clamp(t, min=0.0) + torch.log1p(torch.exp(-torch.abs(t)))


def _in_chunks(s, t):
    """(sequences, heads, chunks, _CHUNK, ...) from (batch, time, heads, ...) or packed (positions, heads, ...); zeros fill up."""
    if s["bounds"] is None:
        t = torch.nn.functional.pad(t, (0, 0) * (t.dim() - 2) + (0, -t.shape[1] % _CHUNK))
    else:
        index, valid = _padded_index(s)
        t = torch.where(valid.view(*valid.shape, *(1,) * (t.dim() - 1)), t[index], torch.zeros((), dtype=t.dtype, device=t.device))
    return t.unflatten(1, (-1, _CHUNK)).movedim(3, 1)


def _padded_index(s):
    bounds = s["bounds"]
    longest = max(1, max(b - a for a, b in zip(bounds[:-1], bounds[1:])))
    at = torch.arange(longest + -longest % _CHUNK, device=s["q"].device)
    low, high = s["cu_seqlens"][:-1, None].long(), s["cu_seqlens"][1:, None].long()
    return torch.clamp(low + at, max=bounds[-1] - 1), low + at < high


def _from_chunks(s, t):
    """What _in_chunks made, back in the order of the inputs."""
    t = t.movedim(1, 3).flatten(1, 2)
    return t[:, :s["time"]] if s["bounds"] is None else t[_padded_index(s)[1]]


def _inverse(a):
    """(1 + a)^-1 for strictly lower triangular a, blocks of 1, 2, 4 ... by blocks."""
    n = a.shape[-1]
    m = torch.eye(n, device=a.device).expand(a.shape)
    size = 1
    while size < n:
        i = torch.arange(n, device=a.device)
        below = (i[:, None] // (2 * size) == i // (2 * size)) & (i[:, None] // size > i // size)
        m = m - m @ (torch.where(below, a, torch.zeros_like(a)) @ m)
        size *= 2
    return m


def _plain_delta(s):
    dtype, scale = s["v"].dtype, s["key_dim"] ** -0.5
    shared = s["heads"] // s["key_heads"]
    q, k, v, beta = (_in_chunks(s, s[name].detach()).float() for name in ("q", "k", "v", "beta"))
    q, k = q.repeat_interleave(shared, 1) * scale, k.repeat_interleave(shared, 1)
    total = torch.cumsum(_in_chunks(s, s["log_decay"].detach().double()), -1)  # log decay from before the chunk
    gamma, rest = torch.exp(total).float()[..., None], torch.exp(total[..., -1:] - total).float()[..., None]
    decay = torch.exp((total[..., :, None] - total[..., None, :]).clamp(max=0.0)).float().tril()
    within = decay.tril(-1) * (k @ k.mT)
    m = _inverse(beta[..., None] * within)
    across = decay * (q @ k.mT)
    state = s["h0"].detach() if s["state"] else q.new_zeros(s["batch"], s["heads"], s["key_dim"], s["value_dim"])
    states, news, outs = [], [], []
    for c in range(q.shape[2]):
        states.append(state)
        new = m[:, :, c] @ (beta[:, :, c, :, None] * (v[:, :, c] - gamma[:, :, c] * (k[:, :, c] @ state)))
        outs.append(gamma[:, :, c] * (q[:, :, c] @ state) + across[:, :, c] @ new)
        state = gamma[:, :, c, -1:] * state + k[:, :, c].mT @ (rest[:, :, c] * new)
        news.append(new)
    outputs = [_from_chunks(s, torch.stack(outs, 2)).to(dtype)] + ([state] if s["state"] else [])
    if not s["grad"]:
        return outputs
    d_o = _in_chunks(s, s["d_o"]).float()
    d_state = s["d_state"] if s["state"] else torch.zeros_like(state)
    d_news, d_states = [], []
    for c in reversed(range(q.shape[2])):  # d_new: of beta (v - gamma k state)
        d_states.append(d_state)
        d_new = m[:, :, c].mT @ (across[:, :, c].mT @ d_o[:, :, c] + rest[:, :, c] * (k[:, :, c] @ d_state))
        d_state = gamma[:, :, c, -1:] * d_state + q[:, :, c].mT @ (gamma[:, :, c] * d_o[:, :, c]) \
            - k[:, :, c].mT @ (gamma[:, :, c] * beta[:, :, c, :, None] * d_new)
        d_news.append(d_new)
    states, new, d_new, d_states = torch.stack(states, 2), torch.stack(news, 2), torch.stack(d_news[::-1], 2), torch.stack(d_states[::-1], 2)
    b = beta[..., None]
    d_within = -(d_new @ new.mT) * decay.tril(-1)      # of beta_i k_i . k_j
    d_across = (d_o @ new.mT) * decay                  # of q_i . k_j
    into = gamma * (d_new @ states.mT)                 # rows S d_new
    along = d_within @ k
    over = rest * (new @ d_states.mT)
    d_q = gamma * (d_o @ states.mT) + d_across @ k
    under = d_within.mT @ (b * k) + d_across.mT @ q
    d_k = over - b * into + b * along + under
    d_beta = (d_new * v).sum(-1) + (k * (along - into)).sum(-1)
    over = (k * over).sum(-1)
    d_total = (q * d_q).sum(-1) + beta * (k * (along - into)).sum(-1) - over - (k * under).sum(-1)
    d_total[..., -1] += over.sum(-1) + gamma[..., -1, 0] * (states * d_states).sum((-2, -1))
    d_log = d_total.double().flip(-1).cumsum(-1).flip(-1).float()

    def shared_heads(t):
        return t.unflatten(1, (s["key_heads"], shared)).sum(2)

    outputs += [_from_chunks(s, shared_heads(d_q) * scale).to(dtype), _from_chunks(s, shared_heads(d_k)).to(dtype),
                _from_chunks(s, b * d_new).to(dtype), _from_chunks(s, d_log), _from_chunks(s, d_beta)]
    return outputs + ([d_state] if s["state"] else [])


def _plain_step(s):
    shared = s["heads"] // s["key_heads"]
    q, k = (s[name].float().repeat_interleave(shared, 1)[..., None, :] for name in ("q", "k"))
    rows = s["slots"].long() if s["slots"] is not None else torch.arange(s["batch"], device=q.device)
    state = torch.exp(s["log_decay"])[..., None, None] * s["state"][rows]
    new = s["beta"][..., None, None] * (s["v"].float()[..., None, :] - k @ state)
    state = state + k.mT * new
    s["state"][rows] = state
    return [(s["key_dim"] ** -0.5 * (q @ state))[..., 0, :].to(s["v"].dtype), s["state"]]


def _plain_rms(s, eps=1e-6):
    """What is normalised, the reciprocal root, and the norm without its weight."""
    x = s["x"].detach()
    total = x if s["residual"] is None else (x.float() + s["residual"].detach().float()).to(x.dtype)
    wide = total.float()
    rstd = torch.rsqrt((wide * wide).mean(-1, keepdim=True) + eps)
    return total, rstd, wide * rstd


def _plain_norm(s):
    dtype, weight = s["x"].dtype, s["weight"].detach()
    total, rstd, normed = _plain_rms(s)
    outputs = [(normed * weight).to(dtype)] + ([] if s["residual"] is None else [total])
    if not s["grad"]:
        return outputs
    d_y = s["d_y"].float()
    d_x = d_y * weight
    d_x = rstd * (d_x - normed * (d_x * normed).mean(-1, keepdim=True))
    if s["residual"] is not None:
        d_x = d_x + s["d_total"].float()
    d_x = d_x.to(dtype)
    return outputs + [d_x] + ([] if s["residual"] is None else [d_x]) + [(d_y * normed).sum(0)]


def _plain_quantize(s):
    kind, most = _QUANTIZED[s["to"]]
    total, _, normed = _plain_rms(s)
    y = normed * s["weight"]
    scales = y.abs().amax(-1) / most
    q = y / torch.where(scales > 0, scales, torch.ones_like(scales))[:, None]
    q = (torch.round(q) if s["to"] == "int8" else q.clamp(-most, most)).to(kind)
    return [_worth(q, scales, s["x"].dtype), scales] + ([] if s["residual"] is None else [total])


_run_plain = {"delta": _plain_delta, "step": _plain_step, "norm": _plain_norm, "quantize": _plain_quantize}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("norm", "quantize"):
        n, tensors = case["rows"] * case["channels"], 2 + 2 * case["residual"]
        if case["op"] == "quantize":
            return {"bytes": n * (size * (tensors - 1) + 1) + 4 * (case["rows"] + case["channels"]), "flops": 6 * n}
        if case["grad"]:  # the gradient reads what was normalised again, and is the residual's too
            tensors += 3 + case["residual"]
        return {"bytes": n * size * tensors + 4 * case["channels"] * (1 + case["grad"]), "flops": (14 if case["grad"] else 5) * n}
    heads, state = case["heads"], case["heads"] * case["key_dim"] * case["value_dim"]
    row = size * (2 * case["key_heads"] * case["key_dim"] + 2 * heads * case["value_dim"]) + 8 * heads  # q, k, v, o, both gates
    if case["op"] == "step":
        return {"bytes": case["batch"] * (row + 8 * state + 4 * bool(case["slots"])), "flops": 7 * case["batch"] * state}
    positions = case["time"] * (1 if case["packed"] else case["batch"])
    ends = 8 * case["batch"] * state * case["state"]
    if not case["grad"]:
        return {"bytes": positions * row + ends, "flops": 7 * positions * state}
    # the gradient reads q, k, v, d_o and the gates and writes as many gradients but for d_o
    more = size * (4 * case["key_heads"] * case["key_dim"] + 3 * heads * case["value_dim"]) + 16 * heads
    return {"bytes": positions * (row + more) + 2 * ends, "flops": 21 * positions * state}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def _by_position(case, state):
    """The sequences side by side, (positions, sequences, ...) in 64 bits, zeros behind the shorter ones; and which are filled."""
    if not case["packed"]:
        def lay(t):
            return t.detach().double().movedim(1, 0)
        filled = torch.ones(case["time"], case["batch"], dtype=torch.bool, device=state["q"].device)
        return lay, filled, lambda t: t.movedim(0, 1)
    bounds = state["bounds"]
    longest = max(b - a for a, b in zip(bounds[:-1], bounds[1:]))
    filled = torch.zeros(longest, case["batch"], dtype=torch.bool, device=state["q"].device)
    for n, (a, b) in enumerate(zip(bounds[:-1], bounds[1:])):
        filled[:b - a, n] = True

    def lay(t):
        out = torch.zeros(longest, case["batch"], *t.shape[1:], dtype=torch.float64, device=t.device)
        for n, (a, b) in enumerate(zip(bounds[:-1], bounds[1:])):
            out[:b - a, n] = t.detach()[a:b]
        return out

    def back(t):
        return torch.cat([t[:b - a, n] for n, (a, b) in enumerate(zip(bounds[:-1], bounds[1:]))])
    return lay, filled, back


def _exact_delta(case, state):
    """Position after position: S <- e^g S, then S <- S + k (beta (v - S^T k))^T, o = S^T q / sqrt(key_dim)."""
    lay, filled, back = _by_position(case, state)
    scale, shared = case["key_dim"] ** -0.5, case["heads"] // case["key_heads"]
    head = torch.arange(case["heads"], device=filled.device) // shared
    q, k, v, g, beta = (lay(state[name]) for name in ("q", "k", "v", "log_decay", "beta"))
    keep = torch.exp(g)
    steps = q.shape[0]
    zero = torch.zeros(case["batch"], case["heads"], case["key_dim"], case["value_dim"], dtype=torch.float64, device=filled.device)
    s = state["h0"].detach().double() if case["state"] else zero

    def forward(t, s):
        key = k[t][:, head]
        s = keep[t][..., None, None] * s
        miss = v[t] - torch.matmul(key[..., None, :], s)[..., 0, :]
        return torch.addcmul(s, key[..., :, None], (beta[t][..., None] * miss)[..., None, :]), miss

    out, kept, every = torch.empty_like(v), [], max(16, int(math.sqrt(steps)))
    for t in range(steps):
        if t % every == 0 and case["grad"]:
            kept.append(s)
        s, _ = forward(t, s)
        out[t] = torch.matmul(q[t][:, head][..., None, :], s)[..., 0, :] * scale
    outputs = [back(out)] + ([s] if case["state"] else [])
    if not case["grad"]:
        return outputs
    d_o = lay(state["d_o"]) * scale
    d_s = state["d_state"].double() if case["state"] else zero
    d_q, d_k, d_v, d_g, d_beta = (torch.zeros_like(t) for t in (q, k, v, g, beta))
    for block in reversed(range(len(kept))):
        first, end = block * every, min(steps, (block + 1) * every)
        before, misses = [kept[block]], []
        for t in range(first, end):
            after, miss = forward(t, before[-1])
            before.append(after)
            misses.append(miss)
        for t in reversed(range(first, end)):
            after, s0, miss, key = before[t - first + 1], before[t - first], misses[t - first], k[t][:, head]
            d_q[t].index_add_(1, head, torch.matmul(after, d_o[t][..., None])[..., 0])
            d_s = torch.addcmul(d_s, q[t][:, head][..., :, None], d_o[t][..., None, :])
            d_new = torch.matmul(key[..., None, :], d_s)[..., 0, :]  # of beta miss
            d_beta[t] = (d_new * miss).sum(-1)
            d_miss = beta[t][..., None] * d_new
            d_v[t] = d_miss
            s1 = keep[t][..., None, None] * s0
            d_k[t].index_add_(1, head, torch.matmul(d_s, (beta[t][..., None] * miss)[..., None])[..., 0] - torch.matmul(s1, d_miss[..., None])[..., 0])
            d_s = torch.addcmul(d_s, key[..., :, None], d_miss[..., None, :], value=-1.0)
            d_g[t] = (d_s * s1).sum((-2, -1))
            d_s = keep[t][..., None, None] * d_s
    outputs += [back(t) for t in (d_q, d_k, d_v, d_g, d_beta)]
    return outputs + ([d_s] if case["state"] else [])


def _exact_step(case, state):
    q, k, v, g, beta = (state[name].double() for name in ("q", "k", "v", "log_decay", "beta"))
    cache, head = state["state"].double(), torch.arange(case["heads"], device=q.device) // (case["heads"] // case["key_heads"])
    rows = state["slots"].tolist() if state["slots"] is not None else list(range(case["batch"]))
    s = cache[rows] * torch.exp(g)[..., None, None]
    miss = v - (k[:, head][..., :, None] * s).sum(-2)
    s = s + k[:, head][..., :, None] * (beta[..., None] * miss)[..., None, :]
    cache[rows] = s
    return [(q[:, head][..., :, None] * s).sum(-2) / math.sqrt(case["key_dim"]), cache]


def _total64(state):
    """x + residual as it is stored, rounded once to the type, in 64 bits."""
    x = state["x"].detach().double()
    if state["residual"] is None:
        return x
    return (x + state["residual"].detach().double()).to(state["x"].dtype).double()


def _exact_norm(case, state, eps=1e-6):
    total, weight = _total64(state).requires_grad_(case["grad"]), state["weight"].detach().double().requires_grad_(case["grad"])
    with torch.enable_grad():
        y = total / torch.sqrt(torch.mean(total ** 2, -1, keepdim=True) + eps) * weight
    outputs = [y.detach()] + ([] if state["residual"] is None else [total.detach()])
    if not case["grad"]:
        return outputs
    d_total, d_weight = torch.autograd.grad(y, (total, weight), state["d_y"].double())
    if state["residual"] is not None:
        d_total = d_total + state["d_total"].double()
        return outputs + [d_total, d_total, d_weight]
    return outputs + [d_total, d_weight]


def _exact_quantize(case, state, eps=1e-6):
    total, most = _total64(state), _QUANTIZED[case["to"]][1]
    y = total / torch.sqrt(torch.mean(total ** 2, -1, keepdim=True) + eps) * state["weight"].double()
    scales = y.abs().amax(-1) / most
    q = y / scales.clamp(min=1e-300)[:, None]
    if case["to"] == "int8":
        q = torch.round(q) * scales[:, None]
    else:  # three bits behind the first, steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3.0)
        q = torch.round(q / step) * step
    return [q, scales] + ([] if state["residual"] is None else [total])


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"delta": _exact_delta, "step": _exact_step, "norm": _exact_norm, "quantize": _exact_quantize}[case["op"]](case, state)
