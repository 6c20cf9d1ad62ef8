"""What the binding of the layer operators hands to the library, on the CPU: the launch is replaced by a recorder, and every
tensor of an argument block has to be described by the strides that it really has."""
import pytest
import torch

import linrec_amd
from linrec_amd import _layers


@pytest.fixture
def blocks(monkeypatch):
    """(function's name, fields of its argument block) of every launch, on host tensors."""
    seen = []

    def record(t, fn, entry, what):
        seen.append((fn.__name__, {name: tuple(value) if isinstance(value := getattr(entry.args, name), _layers._pair) else value
                                   for name, _ in entry.args._fields_}))
    monkeypatch.setattr(_layers, "_call", record)
    monkeypatch.setattr(_layers, "_check_device", lambda *_: None)
    monkeypatch.setattr(_layers._memory, "table", {}, raising=False)
    return seen


def dense_strides(shape):
    return torch.empty(shape).stride()


def kept(tensors):
    """Saved tensors come back as dense ones, which are collected here (so that no address is used twice)."""
    def unpack(t):
        tensors.append(t.contiguous() if not t.is_contiguous() else t.clone())
        return tensors[-1]
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack)


def owners_of(inputs, unpacked):
    """Who has an address in the forward, and in the backward (what a hook gave back may lie where a copy of the forward lay)."""
    return [{t.data_ptr(): t for t in tensors} for tensors in (inputs, inputs + unpacked)]


def check_gated(fields, owners, sizes):
    for name in ("x", "gate_a", "gate_x"):
        got, owner = fields[name + "_stride"], owners.get(fields[name])
        want = dense_strides(sizes["x"]) if owner is None else owner.stride()
        assert got == ((0, want[0]) if len(want) == 2 else want[:2]), name
        assert owner is None or owner.stride(-1) == 1 or owner.size(-1) == 1, name
    for name in ("rate", "h0", "cu_seqlens"):
        owner = owners.get(fields[name])
        assert owner is None or owner.is_contiguous(), name


def gated_inputs(layout, packed):
    """x, gate_a, gate_x, rate, h0, cu_seqlens; `layout` names what is not dense."""
    lead, sequences = ((12,), 3) if packed else ((3, 4), 3)
    tensors = {name: torch.randn(*lead, 6) for name in ("x", "gate_a", "gate_x")}
    tensors.update(rate=torch.randn(6), h0=torch.randn(sequences, 6), cu_seqlens=torch.tensor([0, 3, 3, 12], dtype=torch.int32) if packed else None)
    if layout == "transposed":
        tensors["x"] = torch.randn(*lead[:-1], 6, lead[-1]).transpose(-1, -2)
    elif layout == "expanded gate":
        tensors["gate_a"] = torch.randn(*lead, 1).expand(*lead, 6)
    elif layout == "expanded over time":
        tensors["gate_x"] = torch.randn(*lead[:-1], 1, 6).expand(*lead, 6)
    elif layout == "chunks":
        tensors["x"], tensors["gate_a"], tensors["gate_x"] = torch.randn(*lead, 18).chunk(3, -1)
    elif layout == "state of a layer":
        tensors["h0"] = torch.randn(sequences, 2, 6)[:, 1]
    elif layout == "every second rate":
        tensors["rate"] = torch.randn(12)[::2]
    elif layout == "every second bound" and packed:
        tensors["cu_seqlens"] = torch.tensor([0, 9, 3, 9, 3, 9, 12, 9], dtype=torch.int32)[::2]
    return tensors


def gated_step(tensors, hooks=None):
    leaves = {n: t if t is None or t.dtype == torch.int32 else t.detach().requires_grad_() for n, t in tensors.items()}
    wanted = [t for t in leaves.values() if t is not None and t.requires_grad]
    call = lambda: linrec_amd.gated_linrec(leaves["x"], leaves["gate_a"], leaves["gate_x"], leaves["rate"], h0=leaves["h0"],  # noqa: E731
                                           cu_seqlens=leaves["cu_seqlens"], return_state=True)
    if hooks is None:
        h, state = call()
        torch.autograd.grad((h, state), wanted, (torch.empty(h.shape), torch.empty(state.shape)))
    else:
        with kept(hooks):
            h, state = call()
            torch.autograd.grad((h, state), wanted, (torch.empty(h.shape), torch.empty(state.shape)))
    return [t for t in leaves.values() if t is not None]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("layout", ["transposed", "expanded gate", "expanded over time", "chunks", "state of a layer", "every second rate",
                                    "every second bound"])
@pytest.mark.parametrize("hooked", [False, True])
@pytest.mark.parametrize("dense_first", [False, True])
def test_gated_linrec_reads_every_layout_by_its_own_strides(blocks, packed, layout, hooked, dense_first):
    for kind in (["dense", layout, "dense"] if dense_first else [layout, "dense", layout]):
        tensors, unpacked = gated_inputs(kind, packed), []
        # a hook gives back dense tensors only after a call without hooks has been remembered
        for hooks in ([None, unpacked] if hooked else [None, None]):
            del blocks[:]
            owned = gated_step(tensors, hooks)
            assert [name for name, _ in blocks] == ["linrec_gated_fwd", "linrec_gated_bwd"]
            for (_, fields), owners in zip(blocks, owners_of(owned, unpacked)):
                check_gated(fields, owners, {"x": tensors["x"].shape})


def norm_inputs(layout):
    tensors = {"x": torch.randn(2, 5, 8), "weight": torch.randn(8), "bias": torch.randn(8)}
    if layout == "transposed":
        tensors["x"] = torch.randn(2, 8, 5).transpose(1, 2)
    elif layout == "rows of a wider tensor":
        tensors["x"] = torch.randn(2, 5, 20)[..., 3:11]
    elif layout == "expanded over channels":
        tensors["x"] = torch.randn(2, 5, 1).expand(2, 5, 8)
    elif layout == "every second weight":
        tensors["weight"] = torch.randn(16)[::2]
    return tensors


@pytest.mark.parametrize("layout", ["transposed", "rows of a wider tensor", "expanded over channels", "every second weight"])
@pytest.mark.parametrize("hooked", [False, True])
@pytest.mark.parametrize("dense_first", [False, True])
def test_group_norm_act_reads_every_layout_by_its_own_strides(blocks, layout, hooked, dense_first):
    for kind in (["dense", layout, "dense"] if dense_first else [layout, "dense", layout]):
        tensors, unpacked = norm_inputs(kind), []
        for hooks in ([None, unpacked] if hooked else [None, None]):
            del blocks[:]
            leaves = [t.detach().requires_grad_() for t in tensors.values()]
            with kept(hooks if hooks is not None else []) if hooks is not None else torch.enable_grad():
                y = linrec_amd.group_norm_act(leaves[0], 2, *leaves[1:])
                torch.autograd.grad(y, leaves, torch.empty(y.shape))
            assert [name for name, _ in blocks] == ["linrec_group_norm_fwd", "linrec_group_norm_bwd"]
            for (_, fields), owners in zip(blocks, owners_of(leaves, unpacked)):
                x = owners.get(fields["x"])
                assert fields["x_stride"] == (dense_strides((2, 5, 8)) if x is None else x.stride())[:2]
                assert x is None or x.stride(-1) == 1
                for name in ("weight", "bias"):
                    assert fields[name] not in owners or owners[fields[name]].is_contiguous()


@pytest.mark.parametrize("layout", ["transposed", "without the last", "expanded"])
@pytest.mark.parametrize("hooked", [False, True])
@pytest.mark.parametrize("dense_first", [False, True])
def test_embedding_reads_every_layout_of_tokens(blocks, layout, hooked, dense_first):
    weight = torch.randn(9, 5, requires_grad=True)
    make = {"dense": lambda: torch.randint(0, 9, (4, 7)), "transposed": lambda: torch.randint(0, 9, (7, 4)).t(),
            "without the last": lambda: torch.randint(0, 9, (4, 8))[:, :-1], "expanded": lambda: torch.randint(0, 9, (4, 1)).expand(4, 7)}
    for kind in (["dense", layout, "dense"] if dense_first else [layout, "dense", layout]):
        tokens, unpacked = make[kind](), []
        for hooks in ([None, unpacked] if hooked else [None, None]):
            del blocks[:]
            with kept(hooks if hooks is not None else []) if hooks is not None else torch.enable_grad():
                y = linrec_amd.embedding(tokens, weight)
                torch.autograd.grad(y, weight, torch.empty(y.shape))
            assert [name for name, _ in blocks] == ["linrec_embedding_fwd", "linrec_embedding_bwd"]
            for (_, fields), owners in zip(blocks, owners_of([tokens], unpacked)):
                assert fields["token"] not in owners or owners[fields["token"]].is_contiguous()
