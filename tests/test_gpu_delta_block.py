"""The delta rule, the gated linear layer and what stands around them together on the GPU: the block against the
same block in float64 on the CPU, parts and steps of a prompt, ragged batches, graphs of a decoding step and of a
training step, and the example."""

import copy
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import torch_convnd

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent
# Norm, convolution and projection round q, k, v and the two gates three times each; an output depends on each of
# them (on k twice): 18 roundings, and its own, the heads' norm's, the projection's, the second norm's (whose result
# enters a product twice), the product's and the last one's: 7. Each is at most half a spacing, and the residual
# only adds to the size they are relative to: 25 roundings added up. Gradients pass twice as many. Every test starts
# from a state, as the first output of an empty one is a multiple of its value by q.k, which may be near zero and
# which the heads' norm takes to size one. float32's sums round more than once: as 8 halves of a spacing.
ROUND = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-21}
FORWARD, GRADIENTS = 25, 50


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def pair(dtype, channels=64, heads=2):
    """The block on the GPU and its float64 copy on the CPU."""
    torch.manual_seed(1)
    model = torch_convnd.GatedDeltaBlock(channels, heads, backend="native").to(dtype)
    wide = copy.deepcopy(model).double()
    for module in wide.modules():
        if hasattr(module, "backend"):
            module.backend = "torch"
    return model.cuda(), wide


def states(batch, dtype, channels=64, heads=2):
    window = randn(batch, 3, channels, seed=8).to(dtype)
    hidden = 0.3 * randn(batch, heads, channels // heads, channels // heads, seed=9)
    return (window.cuda(), hidden.cuda()), (window.double(), hidden.double())


def relative(actual, expected):
    a, e = actual.detach().double().cpu(), expected.detach().double().cpu()
    return ((a - e).norm() / e.norm()).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_block_against_float64(dtype):
    model, wide = pair(dtype)
    x, dy = (randn(3, 150, 64, seed=s).to(dtype) for s in (2, 3))
    state, wide_state = states(3, dtype)
    x_gpu, x_wide = x.cuda().requires_grad_(), x.double().requires_grad_()
    y, (window, hidden) = model(x_gpu, state)
    want, (want_window, want_hidden) = wide(x_wide, wide_state)
    assert y.dtype == dtype and hidden.dtype == torch.float32
    assert relative(y, want) <= FORWARD * ROUND[dtype]
    assert relative(window, want_window) <= FORWARD * ROUND[dtype]
    assert relative(hidden, want_hidden) <= FORWARD * ROUND[dtype]
    grads = torch.autograd.grad(y, [x_gpu, *model.parameters()], dy.cuda())
    wants = torch.autograd.grad(want, [x_wide, *wide.parameters()], dy.double())
    for (name, _), got, ref in zip([("input", None), *model.named_parameters()], grads, wants):
        assert relative(got, ref) <= GRADIENTS * ROUND[dtype], name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_then_steps(dtype):
    model, wide = pair(dtype, 128, 1)
    x = randn(2, 90, 128, seed=3).to(dtype)
    state, wide_state = states(2, dtype, 128, 1)
    want, _ = wide(x.double(), wide_state)
    with torch.no_grad():
        outputs = []
        for begin, end in ((0, 70), (70, 80), (80, 84), *((t, t + 1) for t in range(84, 90))):
            y, state = model(x[:, begin:end].cuda(), state)
            outputs.append(y)
    assert relative(torch.cat(outputs, 1), want) <= FORWARD * ROUND[dtype]


def test_ragged_batch():
    model, wide = pair(torch.float32)
    x = randn(4, 70, 64, seed=4)
    (window, hidden), (wide_window, wide_hidden) = states(4, torch.float32)
    lengths = torch.tensor([70, 1, 64, 33])
    y, (window, hidden) = model(x.cuda(), (window, hidden), lengths.cuda())
    for i, n in enumerate(lengths.tolist()):
        want, (want_window, want_hidden) = wide(x[i : i + 1, :n].double(), (wide_window[i : i + 1], wide_hidden[i : i + 1]))
        assert relative(y[i : i + 1, :n], want) <= FORWARD * ROUND[torch.float32]
        assert relative(window[i : i + 1], want_window) <= FORWARD * ROUND[torch.float32]
        assert relative(hidden[i : i + 1], want_hidden) <= FORWARD * ROUND[torch.float32]


def test_decoding_step_in_a_graph():
    """A captured step on static buffers, replayed with the state copied back, is the eager loop."""
    model, _ = pair(torch.bfloat16)
    x = randn(6, 2, 1, 64, seed=5).bfloat16().cuda()
    with torch.no_grad():
        token, state = x[0].clone(), model.initial_state(x[0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model(token, state)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, following = model(token, state)
            for held, new in zip(state, following):
                held.copy_(new)
        for held in state:
            held.zero_()
        eager = model.initial_state(x[0])
        for t in range(6):
            token.copy_(x[t])
            graph.replay()
            want, eager = model(x[t], eager)
            torch.cuda.synchronize()
            assert torch.equal(y, want)
            for held, new in zip(state, eager):
                assert torch.equal(held, new)


def test_training_step_in_a_graph():
    """Outputs and gradients of a captured forward and backward pass, replayed on other inputs beside eager ones."""
    model, _ = pair(torch.bfloat16)
    x, dy = (randn(2, 130, 64, seed=s).bfloat16().cuda() for s in (6, 7))
    weights = [model.gated.weight, model.gated.bias, model.down.weight, model.out.weight]

    def step():
        leaf = x.detach().requires_grad_()
        y, (_, hidden) = model(leaf)
        return y.detach(), hidden.detach(), *torch.autograd.grad(y, [leaf, *weights], dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (11, 12, 13):
        x.copy_(randn(2, 130, 64, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, step()):
            assert torch.equal(got, want)


def test_two_streams_at_once():
    """Blocks at work on two streams at the same time: the results of one after the other."""
    model, _ = pair(torch.bfloat16)
    inputs = [randn(2, 200, 64, seed=s).bfloat16().cuda() for s in (1, 2)]
    with torch.no_grad():
        expected = [model(x) for x in inputs]
        streams = [torch.cuda.Stream() for _ in inputs]
        got = [[], []]
        for stream in streams:
            stream.wait_stream(torch.cuda.current_stream())
        for _ in range(4):
            for stream, x, results in zip(streams, inputs, got):
                with torch.cuda.stream(stream):
                    results.append(model(x))
        torch.cuda.synchronize()
    for results, (want, (_, hidden)) in zip(got, expected):
        for y, (_, last) in results:
            assert torch.equal(y, want) and torch.equal(last, hidden)


def test_example_with_heads():
    command = [sys.executable, str(ROOT / "examples" / "byte_model.py"), "--steps", "20", "--channels", "64",
               "--blocks", "2", "--write", "20", "--heads", "2"]
    result = subprocess.run(command, capture_output=True, text=True, timeout=110)
    assert result.returncode == 0, result.stderr
    assert "bytes/s in writing" in result.stdout
