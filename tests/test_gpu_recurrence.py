"""gated_recurrence on the gfx950 kernels against its 64-bit definition: token counts around runs,
tiles and splits, lengths, closed gates, states, strides, refusals, streams and graphs."""

import pytest
import torch

from sequence_helpers import assert_within, recurrence_reference
from torch_convnd import gated_recurrence

pytestmark = pytest.mark.gpu


def make(b, t, c, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, t, c, generator=g).to(dtype)
    gate = (torch.randn(b, t, c, generator=g) + torch.linspace(-1, 8, c)).clamp(-12, 12).to(dtype)
    first = torch.randn(b, c, generator=g)
    dy = torch.randn(b, t, c, generator=g).to(dtype)
    dlast = torch.randn(b, c, generator=g)
    return [v.cuda() for v in (x, gate, first, dy, dlast)]


def check(x, gate, first, dy, dlast, lengths=None):
    leaves = [v.detach().requires_grad_() for v in (x, gate, first) if v is not None]
    state = leaves[2] if first is not None else None
    h, last = gated_recurrence(leaves[0], leaves[1], state, lengths=lengths, backend="native")
    grads = torch.autograd.grad((h, last), leaves, (dy, dlast))
    ref = recurrence_reference(x, gate, first, lengths, dy, dlast)
    assert h.dtype == x.dtype and h.is_contiguous() and last.dtype == torch.float32
    assert_within(h, *ref["h"], "h")
    assert_within(last, *ref["last"], "last")
    for name, got in zip(("dx", "dgate", "dfirst"), grads):
        assert_within(got, *ref[name], name)
    with torch.no_grad():
        h2, last2 = gated_recurrence(leaves[0], leaves[1], state, lengths=lengths)
    assert torch.equal(h, h2) and torch.equal(last, last2)
    return h, last, grads


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 127, 128, 129, 300])
@pytest.mark.parametrize(("batch", "c"), [(1, 1), (3, 65), (2, 130)])
def test_sizes(batch, tokens, c, dtype):
    check(*make(batch, tokens, c, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize(("batch", "tokens", "c"), [(1, 2500, 70), (2, 1025, 64), (1, 5000, 3), (3, 9000, 131)])
def test_chunks_of_the_token_axis(batch, tokens, c, dtype):
    """Few channels and many tokens: workgroups take chunks of the token axis, several groups of them."""
    check(*make(batch, tokens, c, dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_chunks_with_lengths_and_closed_gates(dtype):
    """Lengths around the chunks' edges, documents that start there, and the same bits every time."""
    x, gate, first, dy, dlast = make(6, 4200, 33, dtype)
    lengths = torch.tensor([4200, 0, 256, 2049, 4097, 63], device="cuda")
    for t in (0, 63, 64, 255, 256, 2048, 4096):
        gate[:, t, ::2] = -float("inf")
    h, last, grads = check(x, gate, first, dy, dlast, lengths)
    for _ in range(3):
        again = check(x, gate, first, dy, dlast, lengths)
        for got, want in zip((again[0], again[1], *again[2]), (h, last, *grads)):
            assert torch.equal(got, want)


def test_chunks_of_infinities():
    """A non-finite state goes on to the tokens after it, of its channel only."""
    x, gate, first, dy, dlast = make(1, 3000, 64, torch.float32)
    clean, _ = gated_recurrence(x, gate, first)
    x[0, 1500, 7] = float("inf")
    x[0, 10, 9] = float("nan")
    h, last = gated_recurrence(x, gate, first)
    others = [c for c in range(64) if c not in (7, 9)]
    assert torch.equal(h[..., others], clean[..., others])
    assert torch.equal(h[:, :1500, 7], clean[:, :1500, 7]) and not torch.isfinite(h[:, 1500:, 7]).any()
    assert torch.equal(h[:, :10, 9], clean[:, :10, 9]) and h[:, 10:, 9].isnan().all()
    assert torch.isfinite(last[:, others]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_channels(dtype):
    """Enough rows for two channels a lane (16-bit, even channels), and an odd count."""
    check(*make(33, 20, 2050, dtype))
    check(*make(33, 9, 2049, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize(("tokens", "c"), [(1, 20), (40, 67), (300, 64), (2300, 9)])
def test_lengths(tokens, c, kind, dtype):
    x, gate, first, dy, dlast = make(7, tokens, c, dtype)
    lengths = torch.tensor([tokens, 0, 1, tokens // 2, tokens + 5, -3, max(0, tokens - 1)], device="cuda").to(kind)
    h, last, grads = check(x, gate, first, dy, dlast, lengths)
    assert torch.equal(last[1], first[1]) and torch.equal(grads[2][1], dlast[1])
    # Nothing held past a length reaches any result.
    poisoned = [v.clone() for v in (x, gate, dy)]
    for b, n in enumerate(lengths.clamp(0, tokens).tolist()):
        for v in poisoned:
            v[b, n:] = float("nan")
    leaves = [v.requires_grad_() for v in (poisoned[0], poisoned[1], first.clone())]
    h2, last2 = gated_recurrence(*leaves, lengths=lengths)
    grads2 = torch.autograd.grad((h2, last2), leaves, (poisoned[2], dlast))
    for got, want in zip((h2, last2, *grads2), (h, last, *grads)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_closed_gates_start_documents(dtype):
    x, gate, first, dy, dlast = make(2, 290, 40, dtype)
    starts = (0, 16, 17, 128, 200)
    for t in starts:
        gate[:, t] = -float("inf")
    h, last, grads = check(x, gate, first, dy, dlast)
    for t in starts:
        assert torch.equal(h[:, t], x[:, t])
    assert torch.equal(grads[2], torch.zeros_like(first))
    # A document's states do not depend on what was packed before it.
    alone, _ = gated_recurrence(x[:, 200:], gate[:, 200:])
    assert_within(h[:, 200:].float(), alone.double(), 2.0**-7 * alone.abs().double() + 1e-30)


def test_open_gates_keep_the_state():
    x, gate, first, dy, dlast = make(2, 150, 64, torch.float32)
    gate.fill_(float("inf"))
    h, last, grads = check(x, gate, first, dy, dlast)
    assert torch.equal(h, first[:, None].expand_as(h)) and torch.equal(last, first)


def test_without_state_and_partial_cotangents():
    x, gate, _, dy, dlast = make(2, 140, 96, torch.bfloat16)
    check(x, gate, None, dy, dlast)
    leaves = [x.requires_grad_(), gate.requires_grad_()]
    zero = torch.zeros_like(dlast)
    h, last = gated_recurrence(*leaves)
    only_h = torch.autograd.grad(h, leaves, dy, retain_graph=True)
    only_last = torch.autograd.grad(last, leaves, dlast)
    for got, (name, d, dl) in zip((only_h, only_last), (("h", dy, zero), ("last", torch.zeros_like(dy), dlast))):
        ref = recurrence_reference(x, gate, None, None, d, dl)
        assert_within(got[0], *ref["dx"], f"dx from {name}")
        assert_within(got[1], *ref["dgate"], f"dgate from {name}")


def test_step_by_step_is_the_prompt():
    """Decoding token by token from the state each call returns."""
    x, gate, first, _, _ = make(3, 37, 80, torch.float32)
    h, last = gated_recurrence(x, gate, first)
    state, outputs = first, []
    for t in range(37):
        out, state = gated_recurrence(x[:, t : t + 1], gate[:, t : t + 1], state)
        outputs.append(out)
    ref = recurrence_reference(x, gate, first)
    assert_within(torch.cat(outputs, 1), *ref["h"], "h")
    assert_within(state, *ref["last"], "last")
    assert_within(last, *ref["last"], "last")


def test_strides():
    x, gate, first, dy, dlast = make(3, 150, 66, torch.bfloat16)
    both = torch.randn(3, 150, 200, device="cuda").to(torch.bfloat16)
    both[..., 1:67], both[..., 100:166] = x, gate  # one projection's two slices, one at an odd offset
    check(both[..., 1:67], both[..., 100:166], first, dy, dlast)
    check(x.transpose(0, 1).contiguous().transpose(0, 1), gate, first, dy, dlast)
    channels_first = x.transpose(1, 2).contiguous().transpose(1, 2)  # channels not contiguous: a copy
    check(channels_first, gate, first, dy, dlast)
    check(x[:1].expand(3, 150, 66), gate, first, dy, dlast)
    check(x, gate, first, dy.transpose(0, 1).contiguous().transpose(0, 1), dlast)


@pytest.mark.parametrize("shape", [(0, 5, 8), (2, 0, 8)])
def test_empty(shape):
    x, gate = (torch.zeros(shape, device="cuda", requires_grad=True) for _ in range(2))
    first = torch.randn(shape[0], shape[2], device="cuda", requires_grad=True)
    h, last = gated_recurrence(x, gate, first)
    assert h.shape == shape and torch.equal(last, first)
    dlast = torch.randn_like(first)
    dx, dg, df = torch.autograd.grad((h, last), (x, gate, first), (torch.empty_like(h), dlast))
    assert dx.shape == dg.shape == shape and torch.equal(df, dlast)


def test_gradient_against_differences():
    x, gate, first, dy, dlast = make(2, 35, 10, torch.float32)
    gate = gate.clamp(-2, 2)
    leaves = [v.requires_grad_() for v in (x, gate, first)]
    grads = torch.autograd.grad(gated_recurrence(*leaves), leaves, (dy, dlast))
    g = torch.Generator(device="cuda").manual_seed(5)
    step = 2.0**-6
    for i, grad in enumerate(grads):
        direction = torch.randn(grad.shape, device="cuda", generator=g)
        value = []
        for sign in (1, -1):
            moved = [v.detach().clone() for v in leaves]
            moved[i] += sign * step * direction
            h, last = gated_recurrence(*moved)
            value.append((h.double() * dy.double()).sum() + (last.double() * dlast.double()).sum())
        slope = (value[0] - value[1]) / (2 * step)
        scale = (grad.double() * direction).abs().sum() + dy.abs().sum() + dlast.abs().sum()
        assert abs(slope - (grad.double() * direction).sum()) <= scale * (4 * step**2 + 64 * 2.0**-24 / step)


def test_same_bits_on_another_stream():
    x, gate, first, dy, dlast = make(2, 2000, 64, torch.bfloat16)
    expected = gated_recurrence(x, gate, first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = gated_recurrence(x, gate, first)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])


def test_graph_replays():
    inputs = make(2, 1100, 48, torch.bfloat16)
    x, gate, first, dy, dlast = inputs
    leaves = [v.requires_grad_() for v in (x, gate, first)]

    def step():
        h, last = gated_recurrence(*leaves)
        return (h, last, *torch.autograd.grad((h, last), leaves, (dy, dlast)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3):
        with torch.no_grad():
            for v, f in zip(inputs, make(2, 1100, 48, torch.bfloat16, seed=seed)):
                v.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, step()):
            assert torch.equal(got, want)


def test_refusals():
    x, gate, first, _, _ = make(2, 6, 8, torch.bfloat16)
    with pytest.raises(RuntimeError, match="supports float16, bfloat16 and float32"):
        gated_recurrence(x.double(), gate.double(), backend="native")
    with pytest.raises(RuntimeError, match=r"\[batch, tokens, channels\]"):
        gated_recurrence(x[0], gate[0])
    with pytest.raises(RuntimeError, match="gate must match"):
        gated_recurrence(x, gate[:, :3])
    with pytest.raises(RuntimeError, match="gate must match"):
        gated_recurrence(x, gate.float())
    with pytest.raises(RuntimeError, match="initial_state must be float32"):
        gated_recurrence(x, gate, first.bfloat16())
    with pytest.raises(RuntimeError, match="initial_state must be float32"):
        gated_recurrence(x, gate, first[:1])
    with pytest.raises(RuntimeError, match="lengths must be int32 or int64"):
        gated_recurrence(x, gate, lengths=torch.ones(2, device="cuda"))
    with pytest.raises(RuntimeError, match="lengths must be int32 or int64"):
        gated_recurrence(x, gate, lengths=torch.ones(3, device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError, match="lengths must be int32 or int64"):
        gated_recurrence(x, gate, lengths=torch.ones(2, dtype=torch.int32))
    h, _ = gated_recurrence(x.requires_grad_(), gate)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(h.float().sum(), x, create_graph=True)
