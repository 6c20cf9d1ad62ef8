"""Waits of the gated recurrence that run out, in chains of several blocks of groups and of channels: the values stay right, and
those of later calls are the same bits as before."""
import pytest
import torch

from linrec_amd import _layers
from linrec_amd import _native as nat

from . import layers_reference as ref
from .test_gpu_gated import make

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("spin", [1, 3])
@pytest.mark.parametrize("dtype,shape,bounds", [(torch.float32, (2, 9001, 70), None), (torch.float16, (1, 12000, 130), None),
                                                (torch.bfloat16, (9000, 200), [0, 10, 3300, 3300, 3301, 8999, 9000]),
                                                (torch.float16, (9000, 66), [0, 4096, 9000])])
def test_waits_that_run_out_in_long_chains(dtype, shape, bounds, spin):
    data = make(shape, dtype, seed=21, sequences=None if bounds is None else len(bounds) - 1)
    x, gate_a, gate_x, rate, h0, d_h, d_state = (t.to(DEV) for t in data)
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device=DEV)

    def run():
        h, state, saved, _ = _layers.gated_fwd(x, gate_a, gate_x, rate, h0, cu, False, 8.0, True)
        return (h, state, *_layers.gated_bwd(d_h, d_state, x, gate_a, gate_x, rate, h0, cu, saved, False, 8.0))
    want = run()
    before = nat.gave_up_count()
    old = nat.lib().linrec_set_spin_limit(spin)
    try:
        got = run()
        torch.cuda.synchronize()
    finally:
        nat.lib().linrec_set_spin_limit(old)
    assert nat.gave_up_count() > before or spin > 1
    # the other tests take a count of zero as the sign that nobody had to fall back: start over
    for ws in list(nat._workspaces.values()):
        ws[:16].view(torch.int32)[1] = 0
    # two orders of the same roundings; a is what the tolerance needs
    log_a = -8.0 * torch.nn.functional.softplus(rate.double()) * torch.sigmoid(gate_a.double())
    a = torch.exp(log_a).cpu()
    for w, g in zip(want, got):
        ref.assert_within(g, w.cpu(), 8 * ref.gated_tolerance(a, g.dtype) * max(1.0, ref.largest(w.cpu())), "after waits that ran out")
    assert all(torch.equal(a, b) for a, b in zip(run(), want))
