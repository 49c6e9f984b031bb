"""gated_delta_rule's gradients beside values and cotangents far from one: what the forward keeps, and what the
backward keeps of the states' gradients, has float16's range, and a cotangent's hundredth or thousandth in it."""

import pytest
import torch

from delta_helpers import assert_rows, delta_reference, make_delta
from sequence_helpers import TINY
from test_gpu_delta_rule import GRADS, train

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


def assert_results(got, reference, sizes):
    """assert_rows beside half a spacing of the result's type, in which results near zero are rounded."""
    dtype = got[0].dtype
    for name, t in zip(("o", "last", *GRADS), got):
        expected, t = reference[name], t.detach().double().cpu()
        off = t - expected
        if name in ("o", "dq", "dk", "dv"):
            assert expected.abs().max() < torch.finfo(dtype).max
            off = off.sign() * (off.abs() - TINY[dtype] / 2).clamp(min=0)
        assert_rows(name, expected + off, reference, dtype, sizes)


def scaled(data, value, cotangent):
    """Values, first states and cotangents times powers of two."""
    data = list(data)
    for i, by in ((2, value), (5, value), (6, cotangent), (7, cotangent)):
        data[i] = data[i] * by
    return data


# One walk, keys shared, walks of 64 columns, segments.
@pytest.mark.parametrize("shape", [(2, 200, 2, 2, 64, 64), (1, 150, 2, 4, 128, 100), (3, 90, 24, 48, 32, 32), (1, 2100, 1, 1, 64, 40)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("exponents", [(0, -10), (0, -13), (0, -17), (0, 9), (-10, 0), (-13, -10), (6, 0), (-12, 12)])
def test_sizes_of_values_and_cotangents(exponents, dtype, shape):
    data = scaled(make_delta(*shape, dtype), *(2.0**e for e in exponents))
    *inputs, first, dy, dlast = (t.cuda() for t in data)
    ref = delta_reference(*data[:6], dy=data[6], dlast=data[7])
    assert_results(train(inputs, first, dy, dlast), ref, shape[4:])


@pytest.mark.parametrize("exponent", [-12, -22, 8])
def test_gradients_are_linear(exponent):
    """Cotangents times a power of two, exact in float16: gradients in float32 times the same, to the bit where the
    cotangents are normal numbers (from 2^-14 on; how the matrix instructions align sums of smaller ones with others
    is theirs, and those are held to the definition like any)."""
    data = list(make_delta(2, 150, 1, 2, 64, 64, torch.float16))
    g = torch.Generator().manual_seed(3)
    data[6] = (torch.randint(-8, 9, data[6].shape, generator=g) / 4).half()
    by = 2.0**exponent
    *inputs, first, dy, dlast = (t.cuda() for t in data)
    assert torch.equal((dy * by).double(), dy.double() * by)
    one, other = train(inputs, first, dy, dlast), train(inputs, first, dy * by, dlast * by)
    assert_results(other, delta_reference(*data[:6], dy=data[6] * by, dlast=data[7] * by), (64, 64))
    for name, a, b in zip(GRADS, one[2:], other[2:]):
        if a.dtype == torch.float32 and exponent >= -12:
            assert torch.equal(a * by, b), name


def test_a_state_gradient_past_the_range():
    """Tokens that ask for the same row of the state, no key of which comes near it: its gradient adds up to 1.3e5."""
    data = list(make_delta(1, 512, 1, 1, 64, 64, torch.float16, normalize=True))
    q, k, v, decay, beta, first, dy, dlast = data
    q.zero_()
    q[..., 0] = 3
    k[..., 0] = 0
    v *= 0.01
    first *= 0.01
    decay.zero_()
    dy.copy_((2000 + 50 * dy.float()).half())
    ref = delta_reference(*data[:6], normalize=True, dy=dy, dlast=dlast)
    assert ref["dfirst"].abs().max() > 65504
    *inputs, first, dy, dlast = (t.cuda() for t in data)
    assert_results(train(inputs, first, dy, dlast, normalize=True), ref, (64, 64))


def test_lengths_and_infinities_do_not_set_the_unit():
    """Nothing past a length, nor a value that is not finite, decides how the rest is kept."""
    data = scaled(make_delta(3, 150, 1, 2, 64, 64, torch.float16), 2.0**-8, 2.0**-12)
    lengths = torch.tensor([150, 70, 0])
    *inputs, first, dy, dlast = (t.cuda() for t in data)
    clean = train(inputs, first, dy, dlast, lengths.cuda())
    for b, n in enumerate(lengths.tolist()):
        for t in (inputs[2], dy):
            t[b, n:] = 60000.0
    for a, b in zip(train(inputs, first, dy, dlast, lengths.cuda()), clean):
        assert torch.equal(a, b)
    # Another head's infinity is no other head's business.
    inputs[2][0, 149, 1] = dy[0, 149, 1] = float("inf")
    dlast[0, 1, 0, 0] = float("inf")
    for name, a, b in zip(("o", "last", *GRADS), train(inputs, first, dy, dlast, lengths.cuda()), clean):
        axis = 1 if name in ("last", "dfirst") else 2
        if name not in ("dq", "dk"):  # sums over both heads
            assert torch.equal(a.select(axis, 0), b.select(axis, 0)), name
        assert torch.equal(a[1:], b[1:])


def test_a_replayed_graph_finds_its_own_units():
    held = [t.cuda() for t in make_delta(2, 150, 1, 2, 64, 64, torch.float16)]

    def step():
        return train(held[:5], held[5], held[6], held[7])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed, value, cotangent in ((1, 0, -16), (2, -9, 8), (3, 0, 0)):
        new = scaled(make_delta(2, 150, 1, 2, 64, 64, torch.float16, seed=seed), 2.0**value, 2.0**cotangent)
        for t, u in zip(held, new):
            t.copy_(u)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize(("batch", "tokens"), [(0, 5), (2, 0)])
def test_empty(batch, tokens):
    *inputs, first, dy, dlast = (t.cuda() for t in make_delta(batch, tokens, 1, 2, 16, 16, torch.float16))
    got = train(inputs, first, dy, dlast)
    assert torch.equal(got[1], first) and torch.equal(got[7], dlast)
    for grad, t in zip(got[2:7], inputs):
        assert grad.shape == t.shape
