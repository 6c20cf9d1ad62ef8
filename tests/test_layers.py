"""CPU tests of the layer operators: the header and the binding agree, host tensors are refused, fake functions give the sizes
of the results, and the float64 forms that the device tests compare with agree with torch's own."""
import ctypes
import os
import re

import pytest
import torch

import linrec_amd
from linrec_amd import _layers
from linrec_amd import _native as nat

from . import layers_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_declared_function_is_exported_and_bound():
    header = open(os.path.join(ROOT, "include", "linrec_layers.h")).read()
    declared = set(re.findall(r"^\s*(?:int|int64_t|size_t)\s+(linrec_\w+)\s*\(", header, flags=re.M))
    assert declared == set(_layers.EXPORTS)
    library = ctypes.CDLL(nat.LIB_PATH)
    for name in declared:
        assert hasattr(library, name)


def test_argument_blocks_have_the_fields_of_the_header_in_its_order():
    header = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "linrec_layers.h")).read(), flags=re.S)
    for struct, name in ((_layers.Gated, "linrec_gated"), (_layers.GatedStep, "linrec_gated_step"),
                         (_layers.GroupNorm, "linrec_group_norm"), (_layers.Embedding, "linrec_embedding")):
        body = re.search(r"typedef struct %s \{(.*?)\} %s_t;" % (name, name), header, flags=re.S).group(1)
        fields = []
        for line in body.split(";"):
            if line.strip():
                kind, names = re.match(r"\s*((?:const )?\w+\s*\*?)\s*(.*)", line.strip(), flags=re.S).groups()
                fields += [re.sub(r"\W.*", "", n.strip().lstrip("*")) for n in names.split(",")]
        assert fields == [f for f, _ in struct._fields_], name


def test_host_tensors_are_refused():
    x = torch.zeros((2, 3, 4))
    with pytest.raises((RuntimeError, NotImplementedError), match="needs device tensors"):
        linrec_amd.gated_linrec(x, x, x, torch.zeros(4))
    with pytest.raises((RuntimeError, NotImplementedError), match="needs device tensors"):
        linrec_amd.gated_linrec_step(x[0], x[0], x[0], torch.zeros(4), torch.zeros(3, 4))
    with pytest.raises((RuntimeError, NotImplementedError), match="needs device tensors"):
        linrec_amd.group_norm_act(x, 2)
    with pytest.raises((RuntimeError, NotImplementedError), match="needs device tensors"):
        linrec_amd.embedding(torch.zeros(3, dtype=torch.long), x[0])


def test_fake_functions_give_the_sizes_of_the_results():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty((2, 300, 6), device="cuda", dtype=torch.bfloat16)
        rate = torch.empty(6, device="cuda")
        h, state = linrec_amd.gated_linrec(x, x, x, rate, return_state=True)
        assert h.shape == x.shape and h.dtype == x.dtype and state.shape == (2, 6) and state.dtype == torch.float32
        h, state = linrec_amd.gated_linrec(x[0], x[0], x[0], rate, cu_seqlens=torch.empty(6, device="cuda", dtype=torch.int32),
                                           return_state=True)
        assert h.shape == (300, 6) and state.shape == (5, 6)
        assert linrec_amd.gated_linrec_step(x[0], x[0], x[0], rate, torch.empty((300, 6), device="cuda")).shape == (300, 6)
        assert linrec_amd.group_norm_act(x, 3).shape == x.shape
        weight = torch.empty((9, 6), device="cuda")
        assert linrec_amd.embedding(torch.empty((2, 3), device="cuda", dtype=torch.long), weight).shape == (2, 3, 6)


def test_bad_arguments_are_rejected_by_the_library():
    library = _layers._lib
    good = dict(dtype=0, batch=1, time=4, channels=4, sequences=1)
    for change, code in ((dict(dtype=7), -3), (dict(batch=-1), -1), (dict(sequences=2), -1), (dict(time=1 << 31), -4), ({}, -1)):
        assert library.linrec_gated_fwd(ctypes.byref(_layers.Gated(**{**good, **change}))) == code
        assert library.linrec_gated_bwd(ctypes.byref(_layers.Gated(**{**good, **change}))) == code
    for change, code in ((dict(dtype=7), -3), (dict(batch=-1), -1), ({}, -1)):
        args = {**dict(dtype=0, batch=1, channels=4, slots_total=1), **change}
        assert library.linrec_gated_step(ctypes.byref(_layers.GatedStep(**args))) == code
    for change, code in ((dict(dtype=7), -3), (dict(weight_dtype=7), -3), (dict(groups=3), -1), (dict(act=9), -1), ({}, -1)):
        args = {**dict(dtype=0, batch=1, positions=1, channels=4, groups=2), **change}
        assert library.linrec_group_norm_fwd(ctypes.byref(_layers.GroupNorm(**args))) == code
        assert library.linrec_group_norm_bwd(ctypes.byref(_layers.GroupNorm(**args))) == code
    for change, code in ((dict(dtype=7), -3), (dict(token_bytes=2), -1), (dict(vocab=-1), -1), (dict(tokens=1 << 31), -4), ({}, -1)):
        args = {**dict(dtype=0, token_bytes=8, tokens=3, vocab=5, channels=4, padding=-1), **change}
        assert library.linrec_embedding_fwd(ctypes.byref(_layers.Embedding(**args))) == code
        assert library.linrec_embedding_bwd(ctypes.byref(_layers.Embedding(**args))) == code
    for call in (library.linrec_gated_fwd, library.linrec_gated_bwd, library.linrec_gated_step, library.linrec_group_norm_fwd,
                 library.linrec_group_norm_bwd, library.linrec_embedding_fwd, library.linrec_embedding_bwd):
        assert call(None) == -1


def test_the_reference_forms():
    g = torch.Generator().manual_seed(0)
    x = torch.randn((2, 5, 6), generator=g, dtype=torch.float64)
    ours = ref.group_norm_act(x, 3, None, None, 1e-5, "silu")
    theirs = torch.nn.functional.silu(torch.nn.functional.group_norm(x.movedim(-1, 1), 3, eps=1e-5)).movedim(1, -1)
    assert torch.allclose(ours, theirs, rtol=1e-12, atol=1e-12)
    tokens, weight = torch.randint(0, 6, (20,), generator=g), torch.randn((6, 4), generator=g, dtype=torch.float64, requires_grad=True)
    y = torch.nn.functional.embedding(tokens, weight, padding_idx=2)
    assert torch.equal(ref.embedding(tokens, weight, 1.0), y)
    d_y = torch.randn((20, 4), generator=g, dtype=torch.float64)
    assert torch.allclose(ref.embedding_grad(d_y, tokens, 6, 1.0, 2)[0], torch.autograd.grad(y, weight, d_y)[0], rtol=1e-12)
    # a sequence of one position, by hand: h = a h0 + sqrt(1 - a^2) sigmoid(gate_x) x
    one = torch.tensor([[[2.0]]]), torch.tensor([[[0.0]]]), torch.tensor([[[0.0]]]), torch.tensor([0.0])
    h, state, a = ref.gated(*one, h0=torch.tensor([[3.0]]), scale=2.0)
    assert abs(float(a) - 0.5) < 1e-12 and abs(float(h) - (1.5 + 0.75 ** 0.5)) < 1e-12 and torch.equal(h[:, 0], state)
    # the values a bound accepts and those it does not: the mistake is planted in the expected value
    with pytest.raises(AssertionError):
        ref.assert_within(h, h + 1e-3, 1e-4, "planted")
    ref.assert_within(h, h + 1e-5, 1e-4, "within")
