"""gated_delta_rule on the gfx950 kernels against its 64-bit definition: token counts around chunks and
steps, head sizes and shared heads, lengths, closed gates, states, strides, streams, graphs, refusals."""

import pytest
import torch

from delta_helpers import assert_rows, delta_reference, make_delta
from torch_convnd import gated_delta_rule

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
GRADS = ("dq", "dk", "dv", "ddecay", "dbeta", "dfirst")


def train(inputs, first, dy, dlast, lengths=None, **options):
    leaves = [t.detach().requires_grad_() for t in (*inputs, *([] if first is None else [first]))]
    state = None if first is None else leaves[5]
    o, last = gated_delta_rule(*leaves[:5], state, lengths=lengths, backend="native", **options)
    return (o.detach(), last.detach(), *torch.autograd.grad((o, last), leaves, (dy, dlast)))


def check(data, lengths=None, state=True, normalize=False, scale=None):
    """Training and inference against the definition; returns what training gave."""
    *inputs, first, dy, dlast = (t.cuda() for t in data)
    first = first if state else None
    if lengths is not None:
        lengths = lengths.cuda()
    options = {"normalize": normalize, "scale": scale}
    got = train(inputs, first, dy, dlast, lengths, **options)
    ref = delta_reference(*inputs, first, lengths, scale, normalize, dy, dlast)
    dtype = inputs[0].dtype
    sizes = (inputs[0].shape[3], inputs[2].shape[3])
    assert got[0].dtype == dtype and got[0].is_contiguous() and got[1].dtype == torch.float32
    for name, t in zip(("o", "last", *GRADS), got):
        assert_rows(name, t, ref, dtype, sizes)
    for t, grad in zip(inputs, got[2:]):
        assert grad.dtype == t.dtype
    with torch.no_grad():
        o, last = gated_delta_rule(*inputs, first, lengths=lengths, **options)
    assert_rows("o", o, ref, dtype, sizes)
    assert_rows("last", last, ref, dtype, sizes)
    if inputs[0].shape[1] > 8:  # not step by step: the same kernels
        assert torch.equal(o, got[0]) and torch.equal(last, got[1])
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 2, 8, 9, 31, 32, 33, 63, 64, 65, 128, 200])
def test_tokens(tokens, dtype):
    check(make_delta(2, tokens, 1, 2, 64, 64, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(
    ("key_size", "value_size"),
    [(1, 1), (3, 5), (16, 16), (40, 71), (64, 8), (65, 64), (96, 130), (100, 200), (128, 128), (127, 257)],
)
def test_head_sizes(key_size, value_size, dtype):
    check(make_delta(2, 75, 1, 1, key_size, value_size, dtype))
    check(make_delta(1, 3, 2, 2, key_size, value_size, dtype), normalize=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(("key_heads", "heads"), [(1, 3), (2, 4), (3, 3), (1, 8)])
def test_shared_heads(key_heads, heads, dtype):
    check(make_delta(2, 70, key_heads, heads, 64, 32, dtype))
    check(make_delta(1, 100, key_heads, heads, 128, 128, dtype), normalize=True, state=False)


@pytest.mark.parametrize("gates", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("normalize", [False, True])
def test_gate_types_and_scale(normalize, gates):
    check(make_delta(2, 90, 2, 2, 48, 64, torch.bfloat16, gates=gates), normalize=normalize, scale=0.7)
    check(make_delta(2, 5, 2, 2, 48, 64, torch.bfloat16, gates=gates), normalize=normalize, scale=0.7)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_chunks(dtype):
    check(make_delta(1, 1500, 1, 2, 64, 64, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(
    ("batch", "heads", "key_size", "value_size"), [(1, 1, 64, 64), (3, 2, 40, 20), (2, 4, 128, 100), (1, 3, 100, 130)]
)
def test_segments(batch, heads, key_size, value_size, dtype):
    """Few heads and many tokens: segments of the tokens side by side, some of them past a sequence's end."""
    data = make_delta(batch, 1030, 1, heads, key_size, value_size, dtype)
    data[3][:, 700] = -float("inf")
    lengths = torch.tensor([1030, 300, 0][:batch])
    got = check(data, lengths)
    got = check(data, state=False)
    again = check(data, state=False)
    for a, b in zip(got, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize(("batch", "heads", "key_size", "value_size"), [(1, 1, 128, 130), (3, 2, 40, 20)])
def test_segments_of_many_tokens(batch, heads, key_size, value_size, dtype):
    data = make_delta(batch, 2100, 1, heads, key_size, value_size, dtype)
    data[3][:, 900] = -float("inf")
    check(data, torch.tensor([2100, 700, 0][:batch]))
    check(data, state=False, normalize=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens", [1, 7, 64, 150])
def test_lengths(tokens, kind, dtype):
    data = make_delta(7, tokens, 1, 2, 32, 48, dtype)
    lengths = torch.tensor([tokens, 0, 1, tokens // 2, tokens + 5, -3, max(0, tokens - 1)]).to(kind)
    got = check(data, lengths)
    *inputs, first, dy, dlast = (t.cuda() for t in data)
    assert torch.equal(got[1][1], first[1]) and torch.equal(got[7][1], dlast[1])
    # Nothing held past a length reaches any result.
    poisoned = [t.clone() for t in (*inputs, dy)]
    for b, n in enumerate(lengths.clamp(0, tokens).tolist()):
        for t in poisoned:
            t[b, n:] = float("nan")
        for t in (got[0], *got[2:7]):
            assert not t[b, n:].any()
    again = train(poisoned[:5], first, poisoned[5], dlast, lengths.cuda())
    for a, b in zip(again, got):
        assert torch.equal(a, b)
    with torch.no_grad():
        clean = gated_delta_rule(*inputs, first, lengths=lengths.cuda())
        other = gated_delta_rule(*poisoned[:5], first, lengths=lengths.cuda())
    assert torch.equal(clean[0], other[0]) and torch.equal(clean[1], other[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_closed_gates_start_documents(dtype):
    data = make_delta(2, 290, 1, 2, 64, 32, dtype)
    starts = (0, 15, 16, 64, 200)
    for t in starts:
        data[3][:, t] = -float("inf")
    data[3][:, 130] = -200.0  # its exp is zero too
    got = check(data)
    assert not got[7].any() and not got[5][:, starts].any() and not got[5][:, 130].any()
    # A document does not depend on what was packed before it.
    *inputs, first, _, _ = (t.cuda() for t in data)
    with torch.no_grad():
        alone, last = gated_delta_rule(*(t[:, 200:] for t in inputs))
    size = alone.float().norm(dim=-1)
    assert ((got[0][:, 200:].float() - alone.float()).norm(dim=-1) <= 2.0**-6 * size + 1e-30).all()
    assert torch.allclose(last, got[1], rtol=1e-3, atol=1e-4)


@pytest.mark.parametrize("dtype", TYPES)
def test_strong_decays_beside_weak_ones(dtype):
    """Sums of decays of some thousand and differences of a hundredth, within a chunk."""
    data = make_delta(1, 140, 1, 2, 32, 32, dtype)
    data[3][:, 5:60:3] = -90.0
    data[3][:, 100] = -103.0
    check(data)


def test_no_decay_and_no_beta():
    """beta 0 leaves the state as it is; with a decay of 0 as well, every state is the first."""
    data = make_delta(2, 100, 1, 1, 32, 32, torch.float32)
    data[3].zero_()
    data[4].zero_()
    *inputs, first, dy, dlast = (t.cuda() for t in data)
    got = train(inputs, first, dy, dlast)
    assert torch.equal(got[1], first) and not got[4].any()
    check(data)


def test_partial_cotangents():
    data = make_delta(2, 100, 1, 2, 32, 32, torch.bfloat16)
    *inputs, first, dy, dlast = (t.cuda() for t in data)
    leaves = [t.requires_grad_() for t in (*inputs, first)]
    o, last = gated_delta_rule(*leaves)
    only_o = torch.autograd.grad(o, leaves, dy, retain_graph=True)
    only_last = torch.autograd.grad(last, [leaves[1], leaves[5]], dlast)
    ref = delta_reference(*data[:6], dy=data[6])
    for name, t in zip(GRADS, only_o):
        assert_rows(name, t, ref, torch.bfloat16, (32, 32))
    ref = delta_reference(*data[:6], dy=torch.zeros_like(data[6]), dlast=data[7])
    assert_rows("dk", only_last[0], ref, torch.bfloat16, (32, 32))
    assert_rows("dfirst", only_last[1], ref, torch.bfloat16, (32, 32))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_prompt_in_parts_and_steps(dtype):
    data = make_delta(3, 107, 2, 4, 64, 64, dtype)
    *inputs, first, _, _ = (t.cuda() for t in data)
    ref = delta_reference(*data[:6])
    state, outputs = first, []
    with torch.no_grad():
        for begin, end in ((0, 70), (70, 100), (100, 103), *((t, t + 1) for t in range(103, 107))):
            o, state = gated_delta_rule(*(t[:, begin:end] for t in inputs), state)
            outputs.append(o)
    assert_rows("o", torch.cat(outputs, 1), ref, dtype, (64, 64))
    # Five calls each leave the rounding of a state in float32.
    assert_rows("last", state, ref, dtype, (64, 64))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [3, 80])
def test_strides(tokens, dtype):
    data = make_delta(2, tokens, 2, 4, 32, 32, dtype)
    *inputs, first, dy, dlast = (t.cuda() for t in data)
    expected = train(inputs, first, dy, dlast)

    def same(changed, cotangent=dy):
        for a, b in zip(train(changed, first, cotangent, dlast), expected):
            assert torch.equal(a, b)

    q, k, v, decay, beta = inputs
    # One projection's slices, from an even and from an odd offset.
    for shift in (0, 1):
        wide = torch.randn(2, tokens, 300, device="cuda").to(dtype)
        parts = [wide[..., shift : 64 + shift], wide[..., 64 + shift : 128 + shift], wide[..., 130 + shift : 258 + shift]]
        parts = [p.unflatten(-1, (-1, 32)) for p in parts]
        for part, t in zip(parts, (q, k, v)):
            part.copy_(t)
        same([*parts, decay, beta])
    # Heads before tokens, tokens before batches, the last axis not contiguous.
    swap = lambda t, a, b: t.transpose(a, b).contiguous().transpose(a, b)  # noqa: E731
    same([swap(t, 1, 2) for t in inputs], swap(dy, 1, 2))
    same([swap(t, 0, 1) for t in inputs], swap(dy, 0, 1))
    same([swap(q, 2, 3), swap(k, 1, 3), swap(v, 2, 3), swap(decay, 0, 2), swap(beta, 1, 2)], swap(dy, 1, 3))
    # A broadcast batch.
    shared = [t[:1].expand_as(t) for t in inputs]
    one = train([t[:1] for t in inputs], first[:1], dy[:1], dlast[:1])
    two = train(shared, first, dy, dlast)
    for a, b in zip(two, one):
        assert torch.equal(a[:1], b)


@pytest.mark.parametrize(("batch", "tokens"), [(0, 5), (2, 0)])
def test_empty(batch, tokens):
    data = make_delta(batch, tokens, 1, 2, 16, 16, torch.float32)
    *inputs, first, dy, dlast = (t.cuda() for t in data)
    got = train(inputs, first, dy, dlast)
    assert got[0].shape == dy.shape and torch.equal(got[1], first) and torch.equal(got[7], dlast)
    for grad, t in zip(got[2:7], inputs):
        assert grad.shape == t.shape
    last = gated_delta_rule(*inputs)[1]
    assert not last.any()


def test_gradient_against_differences():
    data = make_delta(1, 40, 1, 2, 12, 10, torch.float32, normalize=True)
    *inputs, first, dy, dlast = (t.cuda() for t in data)
    inputs[3].clamp_(max=-0.05)
    grads = train(inputs, first, dy, dlast, normalize=True)[2:]
    g = torch.Generator(device="cuda").manual_seed(5)
    step = 2.0**-7
    values = [*inputs, first]
    for i, grad in enumerate(grads):
        direction = torch.randn(grad.shape, device="cuda", generator=g)
        total = []
        for sign in (1, -1):
            moved = [t.detach().double().cpu() for t in values]
            moved[i] += sign * step * direction.double().cpu()
            out = delta_reference(*moved, normalize=True)
            total.append((out["o"] * data[6]).sum() + (out["last"] * data[7]).sum())
        slope = (total[0] - total[1]) / (2 * step)
        scale = (grad.double() * direction).abs().sum().item()
        # Differences in 64 bits are off by a third derivative of the size of the terms; gradients in float32.
        assert abs(slope - (grad.double() * direction).sum().item()) <= scale * (64 * step**2 + 2.0**-14)


def test_a_nan_stays_in_its_head_and_sequence():
    data = make_delta(2, 150, 1, 2, 32, 32, torch.bfloat16)
    *inputs, first, _, _ = (t.cuda() for t in data)
    with torch.no_grad():
        clean = gated_delta_rule(*inputs, first)
        inputs[2][0, 70, 1, 5] = float("nan")
        o, last = gated_delta_rule(*inputs, first)
    assert torch.equal(o[1], clean[0][1]) and torch.equal(o[0, :, 0], clean[0][0, :, 0])
    assert torch.equal(o[0, :64, 1], clean[0][0, :64, 1]) and o[0, 70:, 1, 5].isnan().all()
    others = [c for c in range(32) if c != 5]
    assert torch.equal(o[0, :, 1, others], clean[0][0, :, 1, others])
    assert last[0, 1, :, 5].isnan().all() and torch.equal(last[0, 1][:, others], clean[1][0, 1][:, others])


@pytest.mark.parametrize("tokens", [4, 200])
def test_same_bits_on_another_stream(tokens):
    *inputs, first, dy, dlast = (t.cuda() for t in make_delta(2, tokens, 1, 2, 64, 64, torch.bfloat16))
    expected = train(inputs, first, dy, dlast)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = train(inputs, first, dy, dlast)
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(got, expected):
        assert torch.equal(a, b)


@pytest.mark.parametrize("tokens", [1, 150])
def test_graph_replays(tokens):
    held = [t.cuda() for t in make_delta(2, tokens, 2, 4, 64, 64, torch.bfloat16)]

    def step():
        return train(held[:5], held[5], held[6], held[7], normalize=True)

    def infer():
        with torch.no_grad():
            return gated_delta_rule(*held[:6], normalize=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), infer()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for call in (step, infer):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = call()
        graphs.append((graph, captured, call))
    for seed in (1, 2, 3):
        for t, new in zip(held, make_delta(2, tokens, 2, 4, 64, 64, torch.bfloat16, seed=seed)):
            t.copy_(new)
        for graph, captured, call in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(captured, call()):
                assert torch.equal(a, b)


def test_refusals():
    q, k, v, decay, beta, first, _, _ = (t.cuda() for t in make_delta(2, 6, 2, 4, 16, 8, torch.bfloat16))

    def refused(match, *inputs, **options):
        with pytest.raises(RuntimeError, match=match):
            gated_delta_rule(*inputs, **options)

    refused("supports float16, bfloat16 and float32", *(t.double() for t in (q, k, v, decay, beta)), backend="native")
    refused(r"query and key of \[batch", q[0], k[0], v, decay, beta)
    refused(r"query and key of \[batch", q, k[..., :8], v, decay, beta)
    refused("a value of", q, k, v[:, :3], decay, beta)
    refused("a value of", q, k, v[:, :, :3], decay[..., :3], beta[..., :3])
    refused("decay and beta of", q, k, v, decay[..., :2], beta)
    refused("decay and beta of", q, k, v, decay, beta[:1])
    refused("same device and dtype", q, k.half(), v, decay, beta)
    refused("both of their dtype or float32", q, k, v, decay.half(), beta.half())
    refused("both of their dtype or float32", q, k, v, decay, beta.bfloat16())
    refused("both of their dtype or float32", q, k, v, decay.cpu(), beta.cpu())
    refused("initial_state must be float32", q, k, v, decay, beta, first.bfloat16())
    refused("initial_state must be float32", q, k, v, decay, beta, first[:, :2])
    refused("lengths must be int32 or int64", q, k, v, decay, beta, lengths=torch.ones(2, device="cuda"))
    refused("lengths must be int32 or int64", q, k, v, decay, beta, lengths=torch.ones(2, dtype=torch.int32))
    wide = torch.zeros(1, 2, 1, 129, device="cuda")
    refused("key sizes up to 128", wide, wide, wide, wide[..., 0], wide[..., 0])
    o, _ = gated_delta_rule(q.requires_grad_(), k, v, decay, beta)
    refused_twice = pytest.raises(RuntimeError, match="differentiable once")
    with refused_twice:
        torch.autograd.grad(o.float().sum(), q, create_graph=True)
