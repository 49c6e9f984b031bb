"""gated_recurrence in each of its kernels' forms over several tiles (so that the state is carried and
both LDS buffers are used) against the 64-bit definition: one and two channels a lane, 64, 32 and 16
lanes, chunks over several groups, the step kernel of large batches. Each case asserts the plans it is
there for. Inputs are the two slices of one projection, at an odd offset, with lengths."""

import pytest
import torch

from sequence_helpers import assert_within, recurrence_reference
from torch_convnd import _build, _capi, gated_recurrence, load_native

pytestmark = pytest.mark.gpu
HALF = (torch.bfloat16, torch.float16)
SINGLE = (torch.float32,)
ALL = (*HALF, *SINGLE)

# types, batch, tokens, channels, forward's and backward's kernel, channels a lane and lanes
CASES = [
    (HALF, 9, 700, 1022, ("whole", 2, 16), ("whole", 1, 32)),
    (HALF, 17, 300, 1022, ("whole", 2, 32), ("whole", 1, 64)),
    (HALF, 65, 140, 1022, ("whole", 2, 64), ("whole", 1, 64)),
    (HALF, 33, 140, 1022, ("whole", 1, 64), ("whole", 1, 64)),
    (HALF, 9, 300, 999, ("whole", 1, 32), ("whole", 1, 32)),
    (ALL, 3, 700, 333, ("whole", 1, 16), ("whole", 1, 16)),
    (SINGLE, 9, 300, 1000, ("whole", 1, 32), ("whole", 1, 32)),
    (SINGLE, 17, 140, 1000, ("whole", 1, 64), ("whole", 1, 64)),
    (HALF, 2, 9000, 130, ("chain", 2, 64), ("chain", 2, 64)),
    (ALL, 2, 9000, 65, ("chain", 1, 64), ("chain", 1, 64)),
    (HALF, 129, 1, 1022, ("step", 2, 64), ("whole", 1, 64)),
    (HALF, 65, 8, 1022, ("step", 2, 64), ("whole", 1, 64)),
    (ALL, 5, 8, 131, ("step", 1, 64), ("whole", 1, 64)),
]


@pytest.mark.parametrize(
    ("dtype", "batch", "tokens", "c", "forward", "backward"),
    [(dtype, *rest) for types, *rest in CASES for dtype in types],
)
def test_forms(dtype, batch, tokens, c, forward, backward):
    for plan in planned(dtype, batch, tokens, c, forward, backward):
        # More than one tile, or group of 32 chunks, in the kernels that have them.
        assert tokens > plan["tile"] * {"whole": 1, "chain": 32}.get(plan["kernel"], 0) or tokens <= 8, plan
    check(dtype, batch, tokens, c)


# A forward of whole sequences leaves the states that a backward of chunks starts from.
MIXED = [
    (HALF, 6, 1100, 1022, ("whole", 2, 16), ("chain", 2, 64)),
    (HALF, 12, 1100, 1022, ("whole", 2, 32), ("chain", 2, 64)),
    (HALF, 30, 1030, 1022, ("whole", 2, 64), ("chain", 2, 64)),
    (ALL, 3, 1100, 999, ("whole", 1, 16), ("chain", 1, 64)),
    (SINGLE, 7, 1100, 1000, ("whole", 1, 32), ("chain", 1, 64)),
    (SINGLE, 12, 1100, 1000, ("whole", 1, 64), ("chain", 1, 64)),
]


@pytest.mark.parametrize(
    ("dtype", "batch", "tokens", "c", "forward", "backward"),
    [(dtype, *rest) for types, *rest in MIXED for dtype in types],
)
def test_whole_forward_with_chunks_behind(dtype, batch, tokens, c, forward, backward):
    planned(dtype, batch, tokens, c, forward, backward)
    check(dtype, batch, tokens, c)


@pytest.mark.parametrize(("dtype", "c"), [(torch.bfloat16, 130), (torch.float32, 65)])
def test_graph_replays_of_chunks(dtype, c):
    """The words that chunks hand on are cleared in every replay."""
    per_lane = 2 if c == 130 else 1
    planned(dtype, 2, 9000, c, ("chain", per_lane, 64), ("chain", per_lane, 64))

    def make(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        return [randn(2, 9000, c).to(dtype), (randn(2, 9000, c) + 3).to(dtype), randn(2, c), randn(2, 9000, c).to(dtype), randn(2, c)]

    inputs = make(0)
    leaves = [v.requires_grad_() for v in inputs[:3]]

    def step():
        h, last = gated_recurrence(*leaves)
        return (h, last, *torch.autograd.grad((h, last), leaves, tuple(inputs[3:])))

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
            for held, fresh in zip(inputs, make(seed)):
                held.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, step()):
            assert torch.equal(got, want)


def planned(dtype, batch, tokens, c, forward, backward):
    """The forward's and the backward's plan, which have to be the expected ones."""
    load_native()
    plans = []
    for expected, back in ((forward, False), (backward, True)):
        plan = _capi.recurrence_plan(_build.hip_library(), batch, tokens, c, dtype, back)
        assert (plan["kernel"], plan["channels_per_lane"], plan["lanes"]) == expected, plan
        plans.append(plan)
    return plans


def check(dtype, batch, tokens, c):
    g = torch.Generator().manual_seed(tokens)
    both = torch.randn(batch, tokens, 2 * c + 1, generator=g)
    both[..., c + 1 :] += torch.linspace(-1, 8, c)
    both = both.clamp(-12, 12).to(dtype).cuda()
    first, dlast = (torch.randn(batch, c, generator=g).cuda() for _ in range(2))
    dy = torch.randn(batch, tokens, c, generator=g).to(dtype).cuda()
    lengths = torch.randint(0, tokens + 1, (batch,), generator=g).cuda()
    lengths[0], lengths[-1] = tokens, max(0, tokens - 1)
    x, gate = both[..., 1 : c + 1].detach(), both[..., c + 1 :].detach()
    leaves = [x.requires_grad_(), gate.requires_grad_(), first.requires_grad_()]
    h, last = gated_recurrence(*leaves, lengths=lengths, backend="native")
    grads = torch.autograd.grad((h, last), leaves, (dy, dlast))
    ref = recurrence_reference(x, gate, first, lengths, dy, dlast)
    for name, got in zip(("h", "last", "dx", "dgate", "dfirst"), (h, last, *grads)):
        assert_within(got, *ref[name], name)
    with torch.no_grad():
        again = gated_recurrence(*leaves, lengths=lengths)
    assert torch.equal(h, again[0]) and torch.equal(last, again[1])
