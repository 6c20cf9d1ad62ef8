"""CPU tests of the gated delta rule: the header and the binding agree, host tensors and bad arguments are refused, fake functions give the
sizes of the results, the step's bookkeeping, and the chunk form agrees with the loop in float64."""
import ctypes
import os
import re

import pytest
import torch

import linrec_amd
from linrec_amd import _delta, _layers
from linrec_amd import _native as nat

from . import delta_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = open(os.path.join(ROOT, "include", "linrec_delta.h")).read()


def test_every_declared_function_is_exported_and_bound():
    declared = set(re.findall(r"^\s*(?:int|int64_t|size_t)\s+(linrec_\w+)\s*\(", HEADER, flags=re.M))
    assert declared == set(_delta.EXPORTS)
    library = ctypes.CDLL(nat.LIB_PATH)
    for name in declared:
        assert hasattr(library, name)
    assert _delta.KEY_DIM_MAX == int(re.search(r"#define LINREC_DELTA_KEY_DIM_MAX (\d+)", HEADER).group(1))


def test_argument_blocks_have_the_fields_of_the_header_in_its_order():
    header = re.sub(r"/\*.*?\*/", "", HEADER, flags=re.S)
    for struct, name in ((_delta.Delta, "linrec_delta"), (_delta.DeltaStep, "linrec_delta_step")):
        body = re.search(r"typedef struct %s \{(.*?)\} %s_t;" % (name, name), header, flags=re.S).group(1)
        fields = []
        for line in body.split(";"):
            if line.strip():
                kind, names = re.match(r"\s*((?:const )?\w+\s*\*?)\s*(.*)", line.strip(), flags=re.S).groups()
                fields += [re.sub(r"\W.*", "", n.strip().lstrip("*")) for n in names.split(",")]
        assert fields == [f for f, _ in struct._fields_], name


def arguments(batch=2, time=3, heads=(1, 2), dims=(8, 4), dtype=torch.float32):
    (key_heads, heads), (key_dim, value_dim) = heads, dims
    lead = (batch, time)
    return [torch.randn(*lead, key_heads, key_dim).to(dtype), torch.randn(*lead, key_heads, key_dim).to(dtype), torch.randn(*lead, heads, value_dim).to(dtype),
            -torch.rand(*lead, heads), torch.rand(*lead, heads)]


def test_host_tensors_are_refused():
    whole = arguments()
    with pytest.raises((RuntimeError, NotImplementedError), match="needs device tensors"):
        linrec_amd.gated_delta(*whole)
    with pytest.raises((RuntimeError, NotImplementedError), match="needs device tensors"):
        linrec_amd.gated_delta_step(*(t[:, 0] for t in whole), torch.zeros(2, 2, 8, 4))


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(_layers, "_call", lambda *_: None)
    monkeypatch.setattr(_layers, "_check_device", lambda *_: None)
    monkeypatch.setattr(_delta, "_check_device", lambda *_: None)
    monkeypatch.setattr(_layers._memory, "table", {}, raising=False)


def test_bad_calls_are_refused(no_launch):
    q, k, v, log_decay, beta = arguments()
    call = linrec_amd.gated_delta
    assert call(q, k, v, log_decay, beta).shape == v.shape
    for bad, what in (((q[0], k, v, log_decay, beta), "must be"), ((q, k[0], v, log_decay, beta), "dimensions"), ((q, k[:, :2], v, log_decay, beta), "k has size"),
                      ((q, k.half(), v, log_decay, beta), "k has dtype"), ((q, k, v.half(), log_decay, beta), "v has dtype"),
                      ((q.double(), k.double(), v.double(), log_decay, beta), "float32, float16 or bfloat16"),
                      ((q, k, v[:, :2], log_decay, beta), "v has size"), ((q, k, v, log_decay.half(), beta), "log_decay must be float32"),
                      ((q, k, v, log_decay, beta[..., :1]), "beta has size"), ((q, k, v, log_decay.double(), beta), "log_decay must be float32")):
        with pytest.raises(RuntimeError, match=what):
            call(*bad)
    with pytest.raises(RuntimeError, match="cannot share"):
        call(*arguments(heads=(2, 3)))
    with pytest.raises(RuntimeError, match="key_dim must be"):
        call(*arguments(dims=(257, 4)))
    with pytest.raises(RuntimeError, match="key_dim must be"):
        call(*arguments(dims=(0, 4)), scale=1.0)
    with pytest.raises(RuntimeError, match="value_dim must be"):
        call(*arguments(dims=(8, 0)))
    with pytest.raises(RuntimeError, match="h0 has size"):
        call(q, k, v, log_decay, beta, h0=torch.zeros(2, 2, 4, 8))
    packed = [t[0] for t in (q, k, v, log_decay, beta)]
    assert call(*packed, cu_seqlens=torch.tensor([0, 3], dtype=torch.int32)).shape == packed[2].shape
    for cu, what in ((torch.tensor([0, 3]), "must be int32"), (torch.zeros((1, 2), dtype=torch.int32), "one-dimensional"), (torch.zeros(1, dtype=torch.int32), "no sequence")):
        with pytest.raises(RuntimeError, match=what):
            call(*packed, cu_seqlens=cu)
    with pytest.raises(RuntimeError, match="with cu_seqlens"):
        call(q, k, v, log_decay, beta, cu_seqlens=torch.tensor([0, 3], dtype=torch.int32))


def test_fake_functions_give_the_sizes_of_the_results():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q, v = torch.empty((2, 300, 2, 8), device="cuda", dtype=torch.bfloat16), torch.empty((2, 300, 4, 6), device="cuda", dtype=torch.bfloat16)
        gate = torch.empty((2, 300, 4), device="cuda")
        o, state = linrec_amd.gated_delta(q, q, v, gate, gate, return_state=True)
        assert o.shape == v.shape and o.dtype == v.dtype and state.shape == (2, 4, 8, 6) and state.dtype == torch.float32
        o, state = linrec_amd.gated_delta(q[0], q[0], v[0], gate[0], gate[0], cu_seqlens=torch.empty(6, device="cuda", dtype=torch.int32), return_state=True)
        assert o.shape == (300, 4, 6) and state.shape == (5, 4, 8, 6)
        assert linrec_amd.gated_delta_step(q[0], q[0], v[0], gate[0], gate[0], torch.empty((300, 4, 8, 6), device="cuda")).shape == (300, 4, 6)


def test_bad_arguments_are_rejected_by_the_library():
    library = _delta._lib
    good = dict(dtype=0, key_heads=1, heads=2, key_dim=4, value_dim=4, batch=1, time=4, sequences=1)
    changes = ((dict(dtype=7), -3), (dict(batch=-1), -1), (dict(sequences=2), -1), (dict(time=1 << 31), -4), (dict(heads=0), -1), (dict(key_heads=3), -1),
               (dict(key_dim=300), -3), (dict(value_dim=0), -1), (dict(value_dim=1 << 21), -4), ({}, -1))
    for change, code in changes:
        for call in (library.linrec_delta_fwd, library.linrec_delta_bwd):
            assert call(ctypes.byref(_delta.Delta(**{**good, **change}))) == code, change
    step = dict(dtype=0, key_heads=1, heads=2, key_dim=4, value_dim=4, batch=1, slots_total=1)
    for change, code in ((dict(dtype=7), -3), (dict(batch=-1), -1), (dict(heads=0), -1), (dict(key_dim=300), -3), (dict(value_dim=0), -1), ({}, -1)):
        assert library.linrec_delta_step(ctypes.byref(_delta.DeltaStep(**{**step, **change}))) == code, change
    for call in (library.linrec_delta_fwd, library.linrec_delta_bwd, library.linrec_delta_step):
        assert call(None) == -1
    # scratch that is missing, too small or not aligned is found before any launch
    one = (ctypes.c_char * 64)()
    filled = {name: ctypes.addressof(one) for name in ("q", "k", "v", "log_decay", "beta", "o", "d_o", "d_q", "d_k", "d_v", "d_log_decay", "d_beta")}
    for call, bwd in ((library.linrec_delta_fwd, 0), (library.linrec_delta_bwd, 1)):
        args = _delta.Delta(**good, **filled)
        need = library.linrec_delta_scratch_bytes(ctypes.byref(args), bwd)
        assert need > 0 and call(ctypes.byref(args)) == -2
        args.scratch, args.scratch_bytes = 4096, need - 1
        assert call(ctypes.byref(args)) == -2
        args.scratch, args.scratch_bytes = 4104, need
        assert call(ctypes.byref(args)) == -2


def test_positions_of_too_many_values_are_refused(no_launch):
    library = _delta._lib
    wide = _delta.Delta(dtype=2, key_heads=1, heads=512, key_dim=4, value_dim=(1 << 19) + 1, batch=1, time=4, sequences=1)
    assert library.linrec_delta_fwd(ctypes.byref(wide)) == library.linrec_delta_bwd(ctypes.byref(wide)) == -4
    assert library.linrec_delta_scratch_bytes(ctypes.byref(wide), 0) == 0
    v = torch.empty(1).expand(1, 1, 512, (1 << 19) + 1)
    with pytest.raises(RuntimeError, match="values a position"):
        linrec_amd.gated_delta(torch.empty(1, 1, 1, 4), torch.empty(1, 1, 1, 4), v, torch.empty(1, 1, 512), torch.empty(1, 1, 512))


def test_a_step_counts_as_a_change_of_the_states_and_refuses_tangents(no_launch):
    from torch.autograd import forward_ad
    tensors = [t[:, 0] for t in arguments()] + [torch.zeros(2, 2, 8, 4)]
    before = tensors[5]._version
    linrec_amd.gated_delta_step(*tensors)
    assert tensors[5]._version == before + 1
    for which in range(6):
        with forward_ad.dual_level(), torch.no_grad():
            dual = list(tensors)
            dual[which] = forward_ad.make_dual(tensors[which], torch.ones_like(tensors[which]))
            with pytest.raises(RuntimeError, match="records no gradient"):
                linrec_amd.gated_delta_step(*dual)
    whole = arguments()
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(whole[0], torch.ones_like(whole[0]))] + whole[1:]
        with pytest.raises(RuntimeError, match="records no gradient"):
            linrec_amd.gated_delta(*dual)


def test_the_reference_form():
    """One position by hand, and a gradient against differences."""
    one = [torch.tensor(x) for x in ([[[[2.0]]]], [[[[0.5]]]], [[[[3.0]]]], [[[-0.7]]], [[[0.25]]])]
    o, state = ref.gated_delta(*one, h0=torch.tensor([[[[4.0]]]]), scale=1.0)
    kept = 4.0 * torch.exp(torch.tensor(-0.7)).double()
    want = kept + 0.5 * 0.25 * (3.0 - 0.5 * kept)
    assert torch.allclose(state, want.reshape(1, 1, 1, 1), rtol=1e-6) and torch.allclose(o, 2.0 * want.reshape(1, 1, 1, 1), rtol=1e-6)
    inputs = [t.double().requires_grad_() for t in arguments(1, 5, (1, 2), (3, 2))]
    assert torch.autograd.gradcheck(lambda *t: ref.gated_delta(*t), inputs)
    with pytest.raises(AssertionError):
        ref.assert_near(torch.ones(4), torch.ones(4) * 1.001, 1e-4, "planted")
