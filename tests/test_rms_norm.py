"""CPU tests of the root-mean-square norm: the argument block, refusals, fake functions, and which rows the binding can address."""
import ctypes
import os
import re

import pytest
import torch

import linrec_amd
from linrec_amd import _layers

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_argument_block_has_the_fields_of_the_header_in_its_order():
    header = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "linrec_layers.h")).read(), flags=re.S)
    body = re.search(r"typedef struct linrec_rms_norm \{(.*?)\} linrec_rms_norm_t;", header, flags=re.S).group(1)
    fields = []
    for line in body.split(";"):
        if line.strip():
            kind, names = re.match(r"\s*((?:const )?\w+\s*\*?)\s*(.*)", line.strip(), flags=re.S).groups()
            fields += [re.sub(r"\W.*", "", n.strip().lstrip("*")) for n in names.split(",")]
    assert fields == [f for f, _ in _layers.RmsNorm._fields_]
    assert int(re.search(r"#define LINREC_RMS_NORM_CHANNELS_MAX (\d+)", header).group(1)) == _layers.RMS_NORM_CHANNELS_MAX


def test_host_tensors_are_refused():
    x = torch.zeros((3, 4))
    with pytest.raises((RuntimeError, NotImplementedError), match="needs device tensors"):
        linrec_amd.rms_norm(x)
    with pytest.raises((RuntimeError, NotImplementedError), match="needs device tensors"):
        linrec_amd.rms_norm_quantize(x)


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(_layers, "_call", lambda *_: None)
    monkeypatch.setattr(_layers, "_check_device", lambda *_: None)
    monkeypatch.setattr(_layers._memory, "table", {}, raising=False)


def test_bad_calls_are_refused(no_launch):
    x, w = torch.zeros((3, 8)), torch.ones(8)
    y, total = linrec_amd.rms_norm(x, w, residual=x)
    assert y.shape == total.shape == x.shape
    for call, what in ((lambda: linrec_amd.rms_norm(x.double()), "float32, float16 or bfloat16"), (lambda: linrec_amd.rms_norm(x, w[:4]), "weight has size"),
                       (lambda: linrec_amd.rms_norm(x, w.half()), "weight must be"), (lambda: linrec_amd.rms_norm(x, residual=x[:2]), "residual has size"),
                       (lambda: linrec_amd.rms_norm(x, residual=x.half()), "residual has dtype"), (lambda: linrec_amd.rms_norm(x[:, :0]), "1 to 16384"),
                       (lambda: linrec_amd.rms_norm(torch.zeros((1, 16385))), "1 to 16384"), (lambda: linrec_amd.rms_norm(torch.zeros(())), "channels"),
                       (lambda: linrec_amd.rms_norm_quantize(x, dtype=torch.uint8), "dtype must be"), (lambda: linrec_amd.rms_norm_quantize(x, dtype=None), "dtype must be"),
                       (lambda: linrec_amd.rms_norm_quantize(x, w.clone().requires_grad_()), "records no gradient")):
        with pytest.raises(RuntimeError, match=what):
            call()
    from torch.autograd import forward_ad
    with forward_ad.dual_level(), torch.no_grad():
        dual = forward_ad.make_dual(x, x)
        for call in (linrec_amd.rms_norm, linrec_amd.rms_norm_quantize):
            with pytest.raises(RuntimeError, match="records no gradient"):
                call(dual)


def test_bad_arguments_are_rejected_by_the_library():
    library = _layers._lib
    good = dict(dtype=0, rows=2, inner=1, channels=4)
    for change, code in ((dict(dtype=7), -3), (dict(rows=-1), -1), (dict(inner=0), -1), (dict(channels=0), -1), (dict(channels=20000), -4),
                         (dict(quantized=3), -3), (dict(weight=8, weight_dtype=5), -3), ({}, -1)):
        for call in (library.linrec_rms_norm_fwd, library.linrec_rms_norm_bwd):
            assert call(ctypes.byref(_layers.RmsNorm(**{**good, **change}))) == code, change
    assert library.linrec_rms_norm_fwd(None) == -1 and library.linrec_rms_norm_bwd(None) == -1


def test_fake_functions_give_the_sizes_of_the_results():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty((2, 30, 6), device="cuda", dtype=torch.bfloat16)
        assert linrec_amd.rms_norm(x).shape == x.shape
        y, total = linrec_amd.rms_norm(x, torch.empty(6, device="cuda"), residual=x)
        assert y.shape == total.shape == x.shape and total.dtype == x.dtype
        q, scales, total = linrec_amd.rms_norm_quantize(x, residual=x, dtype=torch.float8_e4m3fn)
        assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn and scales.shape == (2, 30) and total.shape == x.shape


def test_rows_that_can_be_addressed():
    def rows(*tensors):
        layout = _layers._row_layout(list(tensors))
        return layout if layout is None else (layout[0], [tuple(s) for s in layout[1]])
    whole = torch.zeros(2, 5, 3 * 4 * 8)
    assert rows(whole) == (10, [(0, 96)])
    part = whole[..., 32:64].unflatten(-1, (4, 8))
    assert rows(part) == (4, [(96, 8)])
    assert rows(part, torch.zeros(2, 5, 4, 8)) == (4, [(96, 8), (32, 8)])
    assert rows(whole[:, ::2]) == (3, [(480, 192)])
    assert rows(torch.zeros(3, 4, 5, 8).transpose(0, 2)) is None
    assert rows(torch.zeros(8)) == (1, [(0, 0)])
    assert rows(torch.zeros(4, 8)[:, ::2]) is None
    # every address of the two strides, against the tensor's own
    for t in (whole, part, whole[:, ::2], torch.zeros(1, 7, 8)[:, 2:]):
        inner, ((outer_stride, inner_stride),) = rows(t)
        n = t.numel() // t.shape[-1]
        mine = [(r // inner) * outer_stride + (r % inner) * inner_stride for r in range(n)]
        index = torch.arange(t.storage().size()).as_strided(t.shape, t.stride())
        assert mine == index.reshape(n, -1)[:, 0].tolist()
