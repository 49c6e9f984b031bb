"""gated_delta_rule with keys and queries near zero, whose unit lengths are factors of up to 1000: beside float16
what such a token brings has to stay within the type's range on its way into a product."""

import pytest
import torch

from delta_helpers import assert_rows, delta_reference, make_delta
from test_gpu_delta_rule import GRADS, TYPES, train
from torch_convnd import gated_delta_rule

pytestmark = pytest.mark.gpu

# One walk, value heads that share keys, walks of 64 columns, segments.
SHAPES = [(2, 200, 2, 2, 64, 64), (1, 150, 2, 4, 128, 128), (3, 90, 24, 48, 32, 32), (1, 2100, 1, 2, 64, 64)]


def with_small_rows(batch, tokens, key_heads, heads, key_size, value_size, dtype, value, cotangent):
    """Inputs whose values are `value` in size, beside keys and queries of which some are zero or next to it; the
    tokens of the others."""
    data = list(make_delta(batch, tokens, key_heads, heads, key_size, value_size, torch.float32, normalize=True))
    sizes = (0.0, 1e-5, 1e-3, 1e-2, 0.1)  # of a row
    usual = torch.ones(tokens, dtype=torch.bool)
    for i, size in enumerate(sizes):
        for t in (7 + 3 * i, 66 + i, tokens - 1 - 2 * i):
            usual[t] = False
            data[1][:, t] *= size / key_size**0.5
            data[0][:, (t + 1) % tokens] *= size / key_size**0.5
            usual[(t + 1) % tokens] = False
    for i, size in ((2, value), (5, value), (6, cotangent), (7, cotangent)):
        data[i] = data[i] * size
    for i in (0, 1, 2, 6):
        data[i] = data[i].to(dtype)
    return data, usual


# The state's updates, and the gradients on their way back, past 65504 where a factor of 1000 is in them; the
# products of the two, and with them every result, stay within.
@pytest.mark.parametrize(("value", "cotangent"), [(80.0, 0.1), (0.1, 80.0)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_small_rows(shape, dtype, value, cotangent):
    data, usual = with_small_rows(*shape, dtype, value, cotangent)
    *inputs, first, dy, dlast = (t.cuda() for t in data)
    ref = delta_reference(*data[:6], normalize=True, dy=data[6], dlast=data[7])
    sizes = shape[4:]
    got = train(inputs, first, dy, dlast, normalize=True)
    with torch.no_grad():
        o, last = gated_delta_rule(*inputs, first, normalize=True)
    assert torch.equal(o, got[0]) and torch.equal(last, got[1])
    # The usual rows by themselves too, since the others' gradients are a thousand times as large.
    few = {name: t[:, usual] for name, t in ref.items() if name not in ("last", "dfirst", "terms")}
    few["terms"] = {name: t[:, usual] for name, t in ref["terms"].items()}
    for name, t in zip(("o", "last", *GRADS), got):
        assert ref[name].abs().max() < 65504
        assert_rows(name, t, ref, dtype, sizes)
        if name in few:
            assert_rows(name, t[:, usual.cuda()], few, dtype, sizes)


def test_a_zero_key_adds_nothing():
    """Its token leaves the state as it is, however large its value; 9 tokens are taken in a chunk, 8 one by one.

    Beside 1000 * 60000 < 2^26, brought below 2^15, another update's two terms end at 2^-36 of it, 2^-25 in the
    update's own units: in the state that times 64 keys, which is below what assert_rows allows."""
    for tokens in (8, 9, 70):
        q, k, v, decay, beta, first, _, _ = make_delta(2, tokens, 2, 2, 32, 32, torch.float16, normalize=True)
        k[:, 4], decay[:, 4], beta[:, 4] = 0, 0, 1
        for value in (0.0, 60000.0):
            v[:, 4] = value
            ref = delta_reference(q, k, v, decay, beta, first, normalize=True)
            with torch.no_grad():
                o, last = gated_delta_rule(*(t.cuda() for t in (q, k, v, decay, beta, first)), normalize=True)
            assert_rows("o", o, ref, torch.float16, (32, 32))
            assert_rows("last", last, ref, torch.float16, (32, 32))
