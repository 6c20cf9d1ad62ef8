"""Token embedding and its gradient on the device, against their definition in float64."""
import pytest
import torch

import linrec_amd
from linrec_amd import _layers

from . import layers_reference as ref
from .layers_reference import same_bits_in_a_graph

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def words(n, vocab, seed=0):
    """Tokens whose frequencies fall like 1 / rank."""
    g = torch.Generator().manual_seed(seed)
    rank = torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * torch.tensor(float(vocab)).log()).long().clamp_(1, vocab) - 1
    return torch.randperm(vocab, generator=g)[rank]


def check(tokens, vocab, channels, dtype, scale=1.0, padding_idx=None, seed=0, device_d_y=None):
    g = torch.Generator().manual_seed(seed)
    weight = torch.randn((vocab, channels), generator=g).to(dtype)
    d_y = torch.randn((*tokens.shape, channels), generator=g).to(dtype)
    if device_d_y is not None:
        device_d_y, d_y = device_d_y(d_y)
    w = weight.to(DEV).requires_grad_()
    y = linrec_amd.embedding(tokens.to(DEV), w, scale=scale, padding_idx=padding_idx)
    want = ref.embedding(tokens, weight, scale)
    # one fp32 product, one rounding
    ref.assert_within(y, want, (ref.UNIT[dtype] + ref.U32 * 2) * want.abs(), "y")
    got, = torch.autograd.grad(y, w, d_y.to(DEV) if device_d_y is None else device_d_y)
    grad, size, count = ref.embedding_grad(d_y, tokens, vocab, scale, padding_idx)
    # a sum of k terms in fp32 and a product, then one rounding; fp16 denormals have no relative precision
    ref.assert_within(got, grad, ref.UNIT[dtype] * grad.abs() + (count + 2) * ref.U32 * size + (2.0 ** -25 if dtype == torch.float16 else 0.0),
                      "d_weight")
    again, = torch.autograd.grad(linrec_amd.embedding(tokens.to(DEV), w, scale=scale, padding_idx=padding_idx), w,
                                 d_y.to(DEV) if device_d_y is None else device_d_y)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,channels", [(1, 1, 1), (1, 100, 64), (5, 3, 7), (64, 50, 33), (65, 1000, 128), (1000, 17, 130), (4096, 300, 40),
                                              (4097, 70000, 9), (9000, 257, 66), (20000, 5000, 24), (3000, 65536, 8)])
def test_against_the_definition(n, vocab, channels, dtype):
    check(words(n, vocab, seed=n), vocab, channels, dtype, scale=channels ** 0.5, seed=vocab)


@pytest.mark.parametrize("n", [63, 64, 65, 128, 129, 4095, 4096, 4097, 8192, 20000])
def test_one_token_again_and_again(n):
    check(torch.full((n,), 3), 5, 20, torch.float32, seed=n)
    tokens = torch.full((n,), 3)
    tokens[0], tokens[-1] = 4, 2
    check(tokens, 5, 20, torch.bfloat16, seed=n)


@pytest.mark.parametrize("n", [7, 300, 6000])
def test_padding_and_tokens_outside_the_table(n):
    tokens = words(n, 90, seed=1)
    tokens[::5], tokens[1::7] = 11, -1
    tokens[2], tokens[-1] = 90, 2 ** 40 if n != 300 else -2 ** 40
    for padding_idx in (None, 11, 0, 89):
        check(tokens, 90, 12, torch.float32, padding_idx=padding_idx)


def test_a_padding_index_counted_from_the_end():
    tokens = words(500, 90, seed=2).to(DEV)
    weight = torch.randn((90, 12), device=DEV, requires_grad=True)
    d_y = torch.randn((500, 12), device=DEV)
    grads = [torch.autograd.grad(linrec_amd.embedding(tokens, weight, padding_idx=p), weight, d_y)[0] for p in (-1, 89)]
    assert torch.equal(*grads)


@pytest.mark.parametrize("tokens", ["ascending", "descending", "all"])
def test_orders(tokens):
    t = {"ascending": torch.arange(5000) // 3, "descending": 1999 - torch.arange(6000) // 3, "all": torch.arange(2000)}[tokens]
    check(t, 2000, 10, torch.float32, seed=1)


def test_shapes_types_and_strides():
    check(words(60, 40).reshape(3, 4, 5).to(torch.int32), 40, 16, torch.bfloat16)
    check(words(60, 40).reshape(6, 10).t(), 40, 16, torch.float32)
    check(torch.empty((2, 0), dtype=torch.long), 40, 16, torch.float32)

    def strided(d_y):
        wide = torch.zeros((*d_y.shape[:-1], 2 * d_y.shape[-1] + 1), dtype=d_y.dtype, device=DEV)
        wide[..., 1:1 + d_y.shape[-1]] = d_y.to(DEV)
        return wide[..., 1:1 + d_y.shape[-1]], d_y
    check(words(700, 40), 40, 17, torch.bfloat16, device_d_y=strided)
    check(words(700, 40), 40, 17, torch.float32, device_d_y=lambda d: (torch.ones((), device=DEV).expand(d.shape), torch.ones_like(d)))
    w = torch.randn((8, 40), device=DEV).t().requires_grad_()
    y = linrec_amd.embedding(torch.tensor([0, 39, 5], device=DEV), w)
    assert torch.equal(y, w[[0, 39, 5]])
    assert torch.equal(torch.autograd.grad(y.sum(), w)[0].sum(1), torch.zeros(40, device=DEV).index_fill(0, torch.tensor([0, 39, 5], device=DEV), 8.0))


def test_what_is_not_finite_stays_in_its_row():
    tokens = words(5000, 50, seed=3)
    weight = torch.randn((50, 6), device=DEV, requires_grad=True)
    d_y = torch.randn((5000, 6))
    clean, = torch.autograd.grad(linrec_amd.embedding(tokens.to(DEV), weight), weight, d_y.to(DEV))
    d_y[7, 2], d_y[4000, 5] = float("nan"), float("inf")
    got, = torch.autograd.grad(linrec_amd.embedding(tokens.to(DEV), weight), weight, d_y.to(DEV))
    bad = torch.zeros((50, 6), dtype=torch.bool)
    bad[tokens[7], 2] = bad[tokens[4000], 5] = True
    assert torch.equal(got[~bad], clean[~bad]) and not torch.isfinite(got[bad]).any()


def test_rows_more_than_two_to_the_31_elements_into_the_table():
    channels = 1 << 15
    vocab = (1 << 16) + 3
    weight = torch.zeros((vocab, channels), dtype=torch.bfloat16, device=DEV)
    weight[vocab - 1], weight[vocab - 2] = 2.0, 3.0
    weight.requires_grad_()
    tokens = torch.tensor([vocab - 1, 0, vocab - 2, vocab - 1], device=DEV)
    y = linrec_amd.embedding(tokens, weight)
    assert torch.equal(y[:, 0].cpu().float(), torch.tensor([2.0, 0.0, 3.0, 2.0])) and torch.equal(y, weight[tokens])
    d_weight, = torch.autograd.grad(y, weight, torch.ones_like(y))
    assert torch.equal(d_weight[vocab - 1].cpu().float(), torch.full((channels,), 2.0))
    assert torch.equal(d_weight[vocab - 2].cpu().float(), torch.ones(channels)) and torch.equal(d_weight[0].cpu().float(), torch.ones(channels))
    assert float(d_weight[1:vocab - 2].abs().max()) == 0.0


@pytest.mark.parametrize("n", [500, 12000])
def test_in_a_graph(n):
    tokens = words(n, 900, seed=4).to(DEV)
    weight, d_y = torch.randn((900, 32), device=DEV), torch.randn((n, 32), device=DEV)
    same_bits_in_a_graph(lambda: (_layers.embedding_fwd(tokens, weight, 2.0, None)[0], _layers.embedding_bwd(d_y, tokens, weight, 2.0, None)))


def test_traced_calls_are_the_same_operator():
    weight, tokens = torch.randn((30, 8), device=DEV, requires_grad=True), words(40, 30).to(DEV)
    args = (tokens, weight, 2.0, 3)
    torch.library.opcheck(linrec_amd.layers.embedding_fwd, args, test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    y, y2 = linrec_amd.layers.embedding_fwd(*args), linrec_amd.embedding(tokens, weight, scale=2.0, padding_idx=3)
    assert torch.equal(y, y2)
    d_y = torch.randn_like(y)
    assert torch.equal(*(torch.autograd.grad(t, weight, d_y)[0] for t in (y, y2)))


def test_refusals():
    weight, tokens = torch.randn((30, 8), device=DEV), words(40, 30).to(DEV)
    call = linrec_amd.embedding
    for args, kw, text in [
            ((tokens.float(), weight), {}, "int32 or int64"), ((tokens.cpu(), weight), {}, "tokens are on"),
            ((tokens, weight.double()), {}, "float32, float16 or bfloat16"), ((tokens, weight[0]), {}, "vocabulary, channels"),
            ((tokens, weight), {"padding_idx": 30}, "padding_idx"), ((tokens, weight), {"padding_idx": -31}, "padding_idx")]:
        with pytest.raises(RuntimeError, match=text):
            call(*args, **kw)
