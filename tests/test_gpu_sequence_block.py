"""The sequence operators together on the GPU: the block against the same block in float64 on the CPU,
parts and steps of a prompt, ragged batches, a graph of a decoding step, and the example."""

import copy
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import torch_convnd

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent
# A block rounds its activations about ten times (norms, convolution, projections, recurrence,
# residuals), each by at most half a spacing: added up, 10 roundings of the output's magnitude. Its
# gradients pass twice as many.
ROUND = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-21}


def pair(dtype, channels=64):
    """The block on the GPU and its float64 copy on the CPU."""
    torch.manual_seed(1)
    model = torch_convnd.GatedConvBlock(channels, kernel_size=4, expansion=2, backend="native")
    model = model.to(dtype)
    wide = copy.deepcopy(model).double()
    for module in wide.modules():
        if hasattr(module, "backend"):
            module.backend = "torch"
    return model.cuda(), wide


def relative(actual, expected):
    a, e = actual.detach().double().cpu(), expected.detach().double().cpu()
    return ((a - e).norm() / e.norm()).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_block_against_float64(dtype):
    model, wide = pair(dtype)
    g = torch.Generator().manual_seed(2)
    x, dy = (torch.randn(3, 150, 64, generator=g).to(dtype) for _ in range(2))
    x_gpu, x_wide = x.cuda().requires_grad_(), x.double().requires_grad_()
    y, (window, hidden) = model(x_gpu)
    want, (want_window, want_hidden) = wide(x_wide)
    assert relative(y, want) <= 10 * ROUND[dtype]
    assert relative(window, want_window) <= 10 * ROUND[dtype]
    assert relative(hidden, want_hidden) <= 10 * ROUND[dtype]
    grads = torch.autograd.grad(y, [x_gpu, *model.parameters()], dy.cuda())
    wants = torch.autograd.grad(want, [x_wide, *wide.parameters()], dy.double())
    for (name, _), got, ref in zip([("input", None), *model.named_parameters()], grads, wants):
        assert relative(got, ref) <= 20 * ROUND[dtype], name


def test_prompt_then_steps():
    model, wide = pair(torch.float32)
    x = torch.randn(2, 40, 64, generator=torch.Generator().manual_seed(3))
    want, _ = wide(x.double())
    with torch.no_grad():
        first, state = model(x[:, :33].cuda())
        outputs = [first]
        for t in range(33, 40):
            y, state = model(x[:, t : t + 1].cuda(), state)
            outputs.append(y)
    assert relative(torch.cat(outputs, 1), want) <= 10 * ROUND[torch.float32]


def test_ragged_batch():
    model, wide = pair(torch.float32)
    x = torch.randn(4, 70, 64, generator=torch.Generator().manual_seed(4))
    lengths = torch.tensor([70, 1, 64, 33])
    y, (window, hidden) = model(x.cuda(), None, lengths.cuda())
    for i, n in enumerate(lengths.tolist()):
        want, (want_window, want_hidden) = wide(x[i : i + 1, :n].double())
        assert relative(y[i : i + 1, :n], want) <= 10 * ROUND[torch.float32]
        assert relative(window[i : i + 1], want_window) <= 10 * ROUND[torch.float32]
        assert relative(hidden[i : i + 1], want_hidden) <= 10 * ROUND[torch.float32]


def test_decoding_step_in_a_graph():
    """A captured step on static buffers, replayed with the state copied back, is the eager loop."""
    model, _ = pair(torch.bfloat16)
    x = torch.randn(6, 2, 1, 64, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
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


def test_example():
    command = [sys.executable, str(ROOT / "examples" / "byte_model.py"), "--steps", "61", "--channels", "64",
               "--blocks", "2", "--write", "20"]
    result = subprocess.run(command, capture_output=True, text=True, timeout=110)
    assert result.returncode == 0, result.stderr
    losses = [float(line.split()[-1]) for line in result.stdout.splitlines() if line.startswith("step")]
    assert losses[-1] < losses[0] - 1, result.stdout
