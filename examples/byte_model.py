"""A byte-level language model of convolution and recurrence blocks: trains on a text, then writes.

    python examples/byte_model.py [--text FILE] [--steps 200] [--channels 256] [--blocks 4] [--heads 0]

Training runs whole sequences through the blocks (layer norm, causal depthwise convolution, gated
recurrence and linear layers of ``torch_convnd``; with heads the gated delta rule and gated linear layers);
writing keeps each block's state and feeds one byte at a time. On a ROCm GPU all of it runs on the gfx950 kernels in bfloat16, elsewhere on PyTorch's
operations in float32.
"""

import argparse
import sys
import time
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "torch-convnd_amd"))

import torch_convnd  # noqa: E402


class ByteModel(nn.Module):
    def __init__(self, channels, blocks, device=None, dtype=None, backend="auto", heads=0):
        super().__init__()
        factory = {"device": device, "dtype": dtype, "backend": backend}
        self.embed = nn.Embedding(256, channels, device=device, dtype=dtype)
        self.blocks = nn.ModuleList(
            torch_convnd.GatedDeltaBlock(channels, heads, **factory)
            if heads
            else torch_convnd.GatedConvBlock(channels, **factory)
            for _ in range(blocks)
        )
        self.norm = torch_convnd.LayerNorm(channels, **factory)
        self.head = torch_convnd.LinearAct(channels, 256, **factory)

    def forward(self, tokens, states=None, lengths=None):
        x = self.embed(tokens)
        states = [None] * len(self.blocks) if states is None else states
        following = []
        for block, state in zip(self.blocks, states, strict=True):
            x, state = block(x, state, lengths)
            following.append(state)
        return self.head(self.norm(x)), following


def train(model, text, steps, batch, length, device):
    optimizer = torch.optim.AdamW(model.parameters(), lr=2e-3, weight_decay=0.01)
    g = torch.Generator().manual_seed(0)
    losses, started = [], None
    for step in range(steps):
        if step == min(10, steps - 1):
            started = (step, time.perf_counter())
        at = torch.randint(0, len(text) - length - 1, (batch, 1), generator=g)
        window = text[at + torch.arange(length + 1)].to(device)
        logits, _ = model(window[:, :-1])
        loss = nn.functional.cross_entropy(logits.float().flatten(0, 1), window[:, 1:].flatten())
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        if step % 20 == 0 or step == steps - 1:
            losses.append(loss.item())
            print(f"step {step:4d}  loss {losses[-1]:.3f}", flush=True)
    if steps - started[0] > 1:
        rate = (steps - 1 - started[0]) * batch * length / (time.perf_counter() - started[1])
        print(f"{rate:,.0f} bytes/s in training", flush=True)
    return losses


@torch.no_grad()
def write(model, prompt, count, device, temperature=0.7, seed=0):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.tensor(list(prompt), device=device)[None]
    logits, states = model(tokens)
    out, started = list(prompt), time.perf_counter()
    for _ in range(count):
        p = torch.softmax(logits[0, -1].float().cpu() / temperature, dim=0)
        token = int(torch.multinomial(p, 1, generator=g))
        out.append(token)
        logits, states = model(torch.tensor([[token]], device=device), states)
    print(f"{count / (time.perf_counter() - started):,.0f} bytes/s in writing", flush=True)
    return bytes(out)


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--text", default=__file__, help="training text (default: this file)")
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--channels", type=int, default=256)
    parser.add_argument("--blocks", type=int, default=4)
    parser.add_argument("--heads", type=int, default=0, help="heads of the delta rule (0: the gated recurrence)")
    parser.add_argument("--batch", type=int, default=16)
    parser.add_argument("--length", type=int, default=256)
    parser.add_argument("--write", type=int, default=200, help="bytes to write after training")
    options = parser.parse_args(argv)
    on_gpu = torch.cuda.is_available() and torch.version.hip is not None
    device, dtype = ("cuda", torch.bfloat16) if on_gpu else ("cpu", torch.float32)
    torch.manual_seed(0)
    text = torch.tensor(list(Path(options.text).read_bytes()))
    # "native": the convolution of one axis too runs on the gfx950 kernels ("auto" sends it to PyTorch's).
    backend = "native" if on_gpu else "auto"
    model = ByteModel(options.channels, options.blocks, device, dtype, backend, options.heads)
    losses = train(model, text, options.steps, options.batch, min(options.length, len(text) - 2), device)
    if options.write:
        print(write(model, b"def ", options.write, device).decode("utf-8", "replace"))
    return losses


if __name__ == "__main__":
    main()
