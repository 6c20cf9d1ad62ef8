"""Gated linear recurrence and its single-token step on the device, against the loop over positions in float64."""
import pytest
import torch

import linrec_amd
from linrec_amd import _layers
from linrec_amd import _native as nat

from . import layers_reference as ref
from .layers_reference import same_bits_in_a_graph

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(shape, dtype, seed=0, sequences=None):
    """x, gate_a, gate_x, rate, h0 and output gradients on the CPU, the activations rounded to `dtype`."""
    g = torch.Generator().manual_seed(seed)
    channels = shape[-1]
    x, gate_a, gate_x, d_h = (torch.randn(shape, generator=g).to(dtype) for _ in range(4))
    slowest = 0.9 + 0.099 * torch.rand(channels, generator=g)
    rate = torch.log(torch.expm1(-torch.log(slowest) / 8.0))
    n = shape[0] if sequences is None else sequences
    h0, d_state = (torch.randn((n, channels), generator=g) for _ in range(2))
    return x, gate_a, gate_x, rate, h0, d_h, d_state


def check(data, dtype, reverse=False, bounds=None, with_state=True, scale=8.0, device_inputs=None):
    """Outputs and gradients of one call against the float64 loop and its derivative."""
    x, gate_a, gate_x, rate, h0, d_h, d_state = data
    h0 = h0 if with_state else None
    leaves = [t.double().requires_grad_() for t in (x, gate_a, gate_x, rate)] + ([h0.double().requires_grad_()] if with_state else [])
    h_t, state_t, a = ref.gated(*leaves[:4], leaves[4] if with_state else None, bounds, reverse, scale)
    loss = (h_t * d_h.double()).sum() + ((state_t * d_state.double()).sum() if with_state else 0.0)
    grads_t = torch.autograd.grad(loss, leaves) if h_t.numel() or with_state else [torch.zeros_like(t) for t in leaves]

    inputs = [t.to(DEV) for t in (x, gate_a, gate_x)] if device_inputs is None else device_inputs
    inputs = [t.detach().requires_grad_() for t in inputs] + [rate.to(DEV).requires_grad_()]
    if with_state:
        inputs.append(h0.to(DEV).requires_grad_())
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=DEV)
    h, state = linrec_amd.gated_linrec(*inputs[:4], h0=inputs[4] if with_state else None, cu_seqlens=cu, reverse=reverse, scale=scale,
                                       return_state=True)
    assert h.dtype == dtype and state.dtype == torch.float32
    outputs, d_outputs = ([h, state], [d_h.to(DEV), d_state.to(DEV)]) if with_state else ([h], [d_h.to(DEV)])
    grads = torch.autograd.grad(outputs, inputs, d_outputs)
    tol = ref.gated_tolerance(a, dtype)
    ref.assert_within(h, h_t, tol * max(1.0, ref.largest(h_t)), "h")
    ref.assert_within(state, state_t, ref.gated_tolerance(a, torch.float32) * max(1.0, ref.largest(h_t), ref.largest(state_t)), "state")
    # a gradient multiplies two such values and a few factors more
    for name, got, want in zip(("d_x", "d_gate_a", "d_gate_x"), grads, grads_t):
        ref.assert_within(got, want, 4 * tol * max(1.0, ref.largest(want)), name)
    # the sum over positions: no more than its terms are off, each against the largest (d_gate_a is P (1 - sigmoid))
    positions = max(1, x.numel() // max(1, rate.numel()))
    terms = ref.largest(grads_t[1]) / 0.05 * positions * ref.sigmoid_over_softplus(rate)
    ref.assert_within(grads[3], grads_t[3], 4 * ref.gated_tolerance(a, torch.float32) * torch.clamp(terms, min=1e-6), "d_rate")
    if with_state:
        ref.assert_within(grads[4], grads_t[4], 4 * ref.gated_tolerance(a, torch.float32) * max(1.0, ref.largest(grads_t[4]), ref.largest(grads_t[0])),
                          "d_h0")
    assert nat.gave_up_count() == 0


SHAPES = [(1, 1, 1), (2, 1, 3), (1, 2, 64), (3, 63, 65), (2, 64, 128), (2, 65, 130), (1, 127, 66), (2, 129, 256), (1, 500, 7),
          (1, 1025, 129), (4, 300, 31), (1, 2048, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_loop(shape, dtype):
    check(make(shape, dtype, seed=sum(shape)), dtype, reverse=sum(shape) % 2 == 1)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("shape", [(2, 1, 64), (1, 130, 33), (3, 200, 128)])
def test_both_directions_without_a_state(shape, reverse):
    check(make(shape, torch.float32, seed=3), torch.float32, reverse=reverse, with_state=False)


BOUNDS = [
    [0, 1], [0, 0, 5], [0, 5, 5], [0, 0, 0, 1, 1], [0, 16, 32, 48], [0, 15, 17, 63, 64, 65, 127, 128, 129, 200],
    [0, 64, 128, 256], [0, 300, 300, 300, 301, 640], [0, 1, 2, 3, 4, 5, 6, 7, 8, 200], [0, 700, 701],
]


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bounds", BOUNDS, ids=lambda b: "-".join(map(str, b)))
def test_packed_sequences(bounds, dtype, reverse):
    channels = 66
    check(make((bounds[-1], channels), dtype, seed=len(bounds), sequences=len(bounds) - 1), dtype, reverse, bounds)


def test_packed_sequences_without_a_state_and_many_of_them():
    g = torch.Generator().manual_seed(5)
    bounds = [0] + sorted(torch.randint(0, 1501, (1200,), generator=g).tolist()) + [1500]
    data = make((1500, 5), torch.float32, seed=1, sequences=len(bounds) - 1)
    check(data, torch.float32, bounds=bounds, with_state=False)
    check(data, torch.float32, bounds=bounds, reverse=True)


def test_no_positions_at_all():
    z = torch.empty((2, 0, 8), device=DEV)
    h0 = torch.randn(2, 8, device=DEV)
    h, state = linrec_amd.gated_linrec(z, z, z, torch.zeros(8, device=DEV), h0=h0, return_state=True)
    assert h.shape == z.shape and torch.equal(state, h0)
    h, state = linrec_amd.gated_linrec(z[0], z[0], z[0], torch.zeros(8, device=DEV), cu_seqlens=torch.zeros(3, dtype=torch.int32, device=DEV),
                                       return_state=True)
    assert torch.equal(state, torch.zeros(2, 8, device=DEV))
    for shape in ((0, 4, 8), (2, 4, 0)):
        z = torch.empty(shape, device=DEV, requires_grad=True)
        rate = torch.zeros(shape[2], device=DEV, requires_grad=True)
        y = linrec_amd.gated_linrec(z, z, z, rate)
        d_z, d_rate = torch.autograd.grad(y, (z, rate), torch.empty_like(y))
        assert y.shape == shape and d_z.shape == shape and torch.equal(d_rate, torch.zeros_like(rate))
    z = torch.empty((2, 0, 8), device=DEV, requires_grad=True)
    h0 = h0.clone().requires_grad_()
    _, state = linrec_amd.gated_linrec(z, z, z, torch.zeros(8, device=DEV), h0=h0, return_state=True)
    assert torch.equal(torch.autograd.grad(state, h0, torch.ones_like(state))[0], torch.ones_like(state))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_of_a_projection_and_offsets_inside_a_slot(dtype):
    x, gate_a, gate_x, *rest = make((2, 150, 130), dtype, seed=9)
    whole = torch.cat([x, gate_a, gate_x], -1).to(DEV)
    check((x, gate_a, gate_x, *rest), dtype, device_inputs=list(whole.chunk(3, -1)))
    # views that begin one element into an allocation, rows an odd distance apart; channels that are not adjacent
    wide = torch.zeros((2, 150, 263), dtype=dtype, device=DEV)
    wide[..., 1:131], wide[..., 132:262] = x.to(DEV), gate_a.to(DEV)
    turned = gate_x.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    check((x, gate_a, gate_x, *rest), dtype, device_inputs=[wide[..., 1:131], wide[..., 132:262], turned])


def test_gradients_that_are_expanded_views():
    x, gate_a, gate_x, rate, *_ = (t.to(DEV).requires_grad_() for t in make((2, 70, 40), torch.float32, seed=2))
    sums = torch.autograd.grad(linrec_amd.gated_linrec(x, gate_a, gate_x, rate).sum(), (x, gate_a, gate_x, rate))
    h = linrec_amd.gated_linrec(x, gate_a, gate_x, rate)
    dense = torch.autograd.grad(h, (x, gate_a, gate_x, rate), torch.ones_like(h))
    assert all(torch.equal(s, d) for s, d in zip(sums, dense))
    # one gate for all batches: the gradient of an expanded input is the sum over what it was expanded to
    one = gate_a[:1].detach().requires_grad_()
    d_one, = torch.autograd.grad(linrec_amd.gated_linrec(x, one.expand(2, -1, -1), gate_x, rate).sum(), one)
    both = gate_a[:1].detach().repeat(2, 1, 1).requires_grad_()
    d_both, = torch.autograd.grad(linrec_amd.gated_linrec(x, both, gate_x, rate).sum(), both)
    assert torch.equal(d_one, d_both.sum(0, keepdim=True))


def test_positions_more_than_two_to_the_31_elements_apart():
    apart = (1 << 30) + 64
    store = torch.zeros(2 * apart + 4096, dtype=torch.bfloat16, device=DEV)
    x, gate_a, gate_x, rate, h0, d_h, d_state = make((1, 3, 256), torch.bfloat16, seed=4)
    views = []
    for i, t in enumerate((x, gate_a, gate_x)):
        v = store[i * 300:].as_strided((1, 3, 256), (3 * apart, apart, 1))
        v.copy_(t)
        views.append(v)
    check((x, gate_a, gate_x, rate, h0, d_h, d_state), torch.bfloat16, device_inputs=views)


@pytest.mark.parametrize("reverse", [False, True])
def test_what_is_not_finite_stays_in_its_sequence(reverse):
    bounds = [0, 100, 260, 261, 600]
    x, gate_a, gate_x, rate, h0, d_h, d_state = make((600, 130), torch.float32, seed=6, sequences=4)
    clean = make((600, 130), torch.float32, seed=6, sequences=4)
    for value, at in ((float("nan"), 150), (float("inf"), 120)):
        x[at, 3], x[at + 1, 70] = value, value
    h0[2, 9] = float("inf")
    cu = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    results = []
    for data in ((x, gate_a, gate_x, rate, h0, d_h, d_state), clean):
        leaves = [t.to(DEV).requires_grad_() for t in (data[0], data[1], data[2], data[4])]
        h, state = linrec_amd.gated_linrec(*leaves[:3], data[3].to(DEV), h0=leaves[3], cu_seqlens=cu, reverse=reverse, return_state=True)
        results.append((h, state, *torch.autograd.grad((h, state), leaves, (d_h.to(DEV), d_state.to(DEV)))))
    for got, want in zip(*results):
        per_sequence = got.shape[0] == 4
        for n in (0, 3):
            rows = slice(n, n + 1) if per_sequence else slice(bounds[n], bounds[n + 1])
            assert torch.equal(got[rows], want[rows])
    h_t, _, _ = ref.gated(x, gate_a, gate_x, rate, h0, bounds, reverse)
    assert torch.equal(torch.isfinite(results[0][0]).cpu(), torch.isfinite(h_t))


def test_gates_that_are_shut_or_wide_open():
    """sigmoid(gate_a) down to nothing: a is 1, nothing is taken in, and every gradient is finite."""
    x, gate_a, gate_x, rate, h0, d_h, d_state = make((1, 40, 64), torch.float32, seed=8)
    gate_a[0, ::4], gate_a[0, 1::4], gate_a[0, 2::4] = -200.0, 200.0, -float("inf")
    gate_x[0, ::3], gate_x[0, 1::5] = -float("inf"), float("inf")
    rate[:8], rate[8:16], rate[16:24] = -120.0, -60.0, 30.0
    leaves = [t.to(DEV).requires_grad_() for t in (x, gate_a, gate_x, rate, h0)]
    h, state = linrec_amd.gated_linrec(*leaves[:4], h0=leaves[4], return_state=True)
    h_t, state_t, a = ref.gated(x, gate_a, gate_x, rate, h0)
    ref.assert_within(h, h_t, 8 * ref.U32 * 42 * ref.largest(h_t), "h")
    grads = torch.autograd.grad((h, state), leaves, (d_h.to(DEV), d_state.to(DEV)))
    for g in grads:
        assert torch.isfinite(g).all()
    assert torch.equal(grads[1][0, ::4][:, 24:], torch.zeros_like(grads[1][0, ::4][:, 24:]))


def test_directional_differences():
    data = make((2, 200, 96), torch.float32, seed=11)
    x, gate_a, gate_x, rate, h0, d_h, d_state = (t.to(DEV) for t in data)
    leaves = [x, gate_a, gate_x, rate, h0]

    def loss(values):
        h, state = linrec_amd.gated_linrec(*values[:4], h0=values[4], return_state=True)
        return float((h.double() * d_h).sum() + (state.double() * d_state).sum())

    tracked = [t.clone().requires_grad_() for t in leaves]
    h, state = linrec_amd.gated_linrec(*tracked[:4], h0=tracked[4], return_state=True)
    grads = torch.autograd.grad((h, state), tracked, (d_h, d_state))
    g = torch.Generator(device=DEV).manual_seed(1)
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        v = torch.randn(leaf.shape, generator=g, device=DEV)
        step = 2.0 ** -7
        with torch.no_grad():
            up, down = (loss([t + s * step * v if j == i else t for j, t in enumerate(leaves)]) for s in (1, -1))
        # curvature of third order, step^2 times a directional derivative of the loss's own size
        want = (up - down) / (2 * step)
        got = float((grad.double() * v).sum())
        size = float(grad.double().norm() * v.double().norm())
        assert abs(got - want) <= 1e-3 * size + 1e-3 * abs(want), (i, got, want, size)


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_calls_and_single_steps_go_on_from_a_state(dtype):
    x, gate_a, gate_x, rate, h0, *_ = (t.to(DEV) for t in make((3, 140, 70), dtype, seed=12))
    whole, last = linrec_amd.gated_linrec(x, gate_a, gate_x, rate, h0=h0, return_state=True)
    first, state = linrec_amd.gated_linrec(x[:, :70], gate_a[:, :70], gate_x[:, :70], rate, h0=h0, return_state=True)
    second, state = linrec_amd.gated_linrec(x[:, 70:], gate_a[:, 70:], gate_x[:, 70:], rate, h0=state, return_state=True)
    _, _, a = ref.gated(x.cpu(), gate_a.cpu(), gate_x.cpu(), rate.cpu())
    tol = 2 * ref.gated_tolerance(a, dtype) * max(1.0, ref.largest(whole.cpu()))
    ref.assert_within(torch.cat([first, second], 1), whole.cpu(), tol, "two calls")
    ref.assert_within(state, last.cpu(), tol, "state")
    running = h0.clone()
    steps = [linrec_amd.gated_linrec_step(x[:, t], gate_a[:, t], gate_x[:, t], rate, running) for t in range(140)]
    ref.assert_within(torch.stack(steps, 1), whole.cpu(), tol, "steps")
    ref.assert_within(running, last.cpu(), tol, "state of the steps")


def test_the_same_bits_every_time_and_in_a_graph():
    x, gate_a, gate_x, rate, h0, d_h, d_state = (t.to(DEV) for t in make((2, 900, 260), torch.bfloat16, seed=13))

    # both passes without autograd, whose nodes would tie the capture to the stream that they were made on
    def run():
        h, state, saved, _ = _layers.gated_fwd(x, gate_a, gate_x, rate, h0, None, False, 8.0, True)
        return (h, state, *_layers.gated_bwd(d_h, d_state, x, gate_a, gate_x, rate, h0, None, saved, False, 8.0))
    same_bits_in_a_graph(run)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,channels", [(1, 1), (3, 7), (5, 64), (2, 1025), (33, 514)])
def test_step_on_slots_of_a_cache(batch, channels, dtype):
    x, gate_a, gate_x, rate, _, _, _ = make((batch, channels), dtype, seed=batch + channels)
    rows = 2 * batch + 1
    cache = torch.randn((rows, channels), generator=torch.Generator().manual_seed(1))
    slots = torch.randperm(rows, generator=torch.Generator().manual_seed(2))[:batch].to(torch.int32)
    out_of_it = batch > 2
    if out_of_it:
        slots[1], slots[2] = -1, rows
    wide = torch.full((rows, channels + 3), 7.0, device=DEV)
    wide[:, :channels] = cache.to(DEV)
    got = linrec_amd.gated_linrec_step(x.to(DEV), gate_a.to(DEV), gate_x.to(DEV), rate.to(DEV), wide[:, :channels], slots=slots.to(DEV))
    want, want_cache = torch.zeros((batch, channels), dtype=torch.float64), cache.double().clone()
    for n in range(batch):
        if 0 <= slots[n] < rows:
            h, _, _ = ref.gated(x[n][None, None], gate_a[n][None, None], gate_x[n][None, None], rate, cache[slots[n]][None])
            want[n] = want_cache[slots[n]] = h[0, 0]
    size = max(1.0, ref.largest(want))
    ref.assert_within(got, want, (ref.UNIT[dtype] + 24 * ref.U32) * size, "h")
    ref.assert_within(wide[:, :channels], want_cache, 24 * ref.U32 * size, "state")
    assert torch.equal(wide[:, channels:].cpu(), torch.full((rows, 3), 7.0))


def test_step_takes_strided_rows_and_an_empty_batch():
    x, gate_a, gate_x, rate, h0, *_ = (t.to(DEV) for t in make((4, 50), torch.bfloat16, seed=3))
    rate = rate[:50]
    whole = torch.cat([x, gate_a, gate_x], 1)
    one, two = h0.clone()[:, :50], h0.clone()[:, :50]
    a = linrec_amd.gated_linrec_step(*whole.chunk(3, 1), rate, one)
    b = linrec_amd.gated_linrec_step(x, gate_a, gate_x, rate, two)
    assert torch.equal(a, b) and torch.equal(one, two)
    none = linrec_amd.gated_linrec_step(x[:0], gate_a[:0], gate_x[:0], rate, one[:0])
    assert none.shape == (0, 50)


def test_traced_calls_are_the_same_operator():
    x, gate_a, gate_x, rate, h0, d_h, _ = (t.to(DEV) for t in make((2, 33, 12), torch.float32, seed=14))
    leaves = [t.requires_grad_() for t in (x, gate_a, gate_x, rate, h0)]
    args = (*leaves, None, False, 8.0)
    torch.library.opcheck(linrec_amd.layers.gated_linrec_fwd, args, test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    h, state, _ = linrec_amd.layers.gated_linrec_fwd(*args)
    grads = torch.autograd.grad(h, leaves, d_h)
    h2 = linrec_amd.gated_linrec(*leaves[:4], h0=leaves[4])
    assert torch.equal(h, h2)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(h2, leaves, d_h)))


def test_refusals():
    x, gate_a, gate_x, rate, h0, *_ = (t.to(DEV) for t in make((2, 5, 8), torch.float32))
    call = linrec_amd.gated_linrec
    bounds = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    for args, kw, text in [
            ((x[0], gate_a[0], gate_x[0], rate), {}, "batch, time, channels"),
            ((x, gate_a[:, :4], gate_x, rate), {}, "gate_a has size"),
            ((x, gate_a, gate_x.half(), rate), {}, "gate_x has dtype"),
            ((x, gate_a, gate_x.cpu(), rate), {}, "gate_x is on"),
            ((x.double(), gate_a, gate_x, rate), {}, "float32, float16 or bfloat16"),
            ((x, gate_a, gate_x, rate.half()), {}, "rate must be float32"),
            ((x, gate_a, gate_x, rate[:4]), {}, "rate has size"),
            ((x, gate_a, gate_x, rate), {"h0": h0[:1]}, "h0 has size"),
            ((x, gate_a, gate_x, rate), {"cu_seqlens": bounds}, "positions, channels"),
            ((x[0], gate_a[0], gate_x[0], rate), {"cu_seqlens": bounds.long()}, "int32"),
            ((x[0], gate_a[0], gate_x[0], rate), {"cu_seqlens": bounds.cpu()}, "cu_seqlens is on"),
            ((x[0], gate_a[0], gate_x[0], rate), {"cu_seqlens": bounds[:1]}, "no sequence")]:
        with pytest.raises(RuntimeError, match=text):
            call(*args, **kw)
    step = linrec_amd.gated_linrec_step
    x, gate_a, gate_x = x[:, 0], gate_a[:, 0], gate_x[:, 0]
    slots = torch.zeros(2, dtype=torch.int32, device=DEV)
    for args, kw, text in [
            ((x, gate_a, gate_x, rate, h0[:1]), {}, "name the rows"),
            ((x, gate_a, gate_x, rate, h0.half()), {}, "state must be float32"),
            ((x, gate_a, gate_x, rate, h0), {"slots": slots.long()}, "slots must be int32"),
            ((x, gate_a, gate_x, rate, h0), {"slots": slots[:1]}, "slots must be int32"),
            ((x, gate_a, gate_x, rate, h0[:1].expand(2, -1)), {}, "overlap"),
            ((x, gate_a, gate_x, rate, h0.t().contiguous().t()), {}, "unit stride"),
            ((x.clone().requires_grad_(), gate_a, gate_x, rate, h0), {}, "no gradient")]:
        with pytest.raises(RuntimeError, match=text):
            step(*args, **kw)


@pytest.mark.parametrize("bounds", [None, [0, 1, 700, 700, 1500, 1501, 2300]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_waits_that_run_out(dtype, bounds):
    """With a limit of one poll most segments give up on the ones before them and walk their channels themselves."""
    shape = (1, 2300, 96) if bounds is None else (2300, 96)
    x, gate_a, gate_x, rate, h0, d_h, d_state = (t.to(DEV) for t in make(shape, dtype, seed=15, sequences=None if bounds is None else len(bounds) - 1))
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=DEV)

    def run():
        h, state, saved, _ = _layers.gated_fwd(x, gate_a, gate_x, rate, h0, cu, False, 8.0, True)
        return (h, state, *_layers.gated_bwd(d_h, d_state, x, gate_a, gate_x, rate, h0, cu, saved, False, 8.0))
    want = run()
    before = nat.gave_up_count()
    old = nat.lib().linrec_set_spin_limit(1)
    try:
        got = run()
        torch.cuda.synchronize()
    finally:
        nat.lib().linrec_set_spin_limit(old)
    assert nat.gave_up_count() > before
    # the other tests take a count of zero as the sign that nobody had to fall back: start over
    for ws in list(nat._workspaces.values()):
        ws[:16].view(torch.int32)[1] = 0
    _, _, a = ref.gated(x.cpu(), gate_a.cpu(), gate_x.cpu(), rate.cpu(), bounds=bounds)
    for w, g in zip(want, got):
        tol = ref.gated_tolerance(a, g.dtype)
        ref.assert_within(g, w.cpu(), 8 * tol * max(1.0, ref.largest(w.cpu())), "after waits that ran out")
    after = run()
    assert all(torch.equal(a, b) for a, b in zip(after, want))


def test_many_segments_and_channels():
    """More groups of segments than are looked at at a time, more blocks of channels than one."""
    data = make((2, 3000, 200), torch.bfloat16, seed=16)
    check_on_device(data, torch.bfloat16)
    data = make((1, 6000, 130), torch.float32, seed=17)
    check_on_device(data, torch.float32)


def check_on_device(data, dtype):
    """As `check`, the float64 loop on the device (over positions, all channels at once)."""
    x, gate_a, gate_x, rate, h0, d_h, d_state = (t.to(DEV) for t in data)
    leaves = [t.requires_grad_() for t in (x, gate_a, gate_x, rate, h0)]
    h, state = linrec_amd.gated_linrec(*leaves[:4], h0=leaves[4], return_state=True)
    grads = torch.autograd.grad((h, state), leaves, (d_h, d_state))
    xs, gas, gxs, r = (t.detach().double() for t in leaves[:4])
    sig_a, sig_x = torch.sigmoid(gas), torch.sigmoid(gxs)
    log_a = -8.0 * torch.nn.functional.softplus(r) * sig_a
    a, m = torch.exp(log_a), torch.sqrt(-torch.expm1(2 * log_a))
    time = x.shape[1]
    before, value = torch.empty_like(a), h0.detach().double()
    for t in range(time):
        before[:, t] = value
        value = a[:, t] * value + m[:, t] * sig_x[:, t] * xs[:, t]
    after = a * before + m * sig_x * xs
    g, carry = torch.empty_like(a), d_state.double()
    for t in reversed(range(time)):
        g[:, t] = d_h[:, t].double() + carry
        carry = a[:, t] * g[:, t]
    p = g * (log_a * a * before - sig_x * xs * a * a * log_a / m)
    tol, tol32 = ref.gated_tolerance(a.cpu(), dtype), ref.gated_tolerance(a.cpu(), torch.float32)
    ref.assert_within(h, after.cpu(), tol * ref.largest(after.cpu()), "h")
    ref.assert_within(state, value.cpu(), tol32 * ref.largest(after.cpu()), "state")
    for got, want, name in zip(grads[:3], (g * m * sig_x, p * (1 - sig_a), g * m * xs * sig_x * (1 - sig_x)), ("d_x", "d_gate_a", "d_gate_x")):
        ref.assert_within(got, want.cpu(), 4 * tol * ref.largest(want.cpu()), name)
    ratio = ref.sigmoid_over_softplus(r.cpu())
    ref.assert_within(grads[3], p.sum((0, 1)).cpu() * ratio, 4 * tol32 * p.abs().sum((0, 1)).cpu() * ratio, "d_rate")
    ref.assert_within(grads[4], carry.cpu(), 4 * tol32 * max(1.0, ref.largest(carry.cpu()), ref.largest(g.cpu())), "d_h0")


@pytest.mark.parametrize("bounds", [None, [0, 9000, 9001, 24000]])
def test_long_chains(bounds):
    """More blocks of groups of segments than are looked at at a time; sequences that start inside one."""
    if bounds is None:
        check(make((1, 24000, 3), torch.bfloat16, seed=18), torch.bfloat16)
        check(make((1, 24000, 2), torch.float32, seed=19), torch.float32, reverse=True)
    else:
        check(make((24000, 3), torch.bfloat16, seed=20, sequences=3), torch.bfloat16, bounds=bounds)
