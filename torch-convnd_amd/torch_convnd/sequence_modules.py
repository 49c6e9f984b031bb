"""Modules of token sequences, [batch, tokens, channels]: the operators of ``sequence`` as layers, and
the block that joins them with a causal convolution. No counterpart in the reference."""

import math

import torch
from torch import Tensor, nn

from .functional import _ACTIVATIONS, conv_nd
from .modules import Conv1d
from .sequence import gated_recurrence, layer_norm, linear_act


class LayerNorm(nn.Module):
    """``layer_norm`` over the last dimension with a weight and (``bias=True``) a bias."""

    def __init__(self, channels: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=None, *, backend="auto"):
        super().__init__()
        if channels <= 0:
            raise ValueError("channels must be positive")
        self.channels = channels
        self.eps = eps
        self.backend = backend
        self.weight = nn.Parameter(torch.ones(channels, device=device, dtype=dtype))
        if bias:
            self.bias = nn.Parameter(torch.zeros(channels, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)

    def forward(self, input: Tensor) -> Tensor:
        return layer_norm(input, self.weight, self.bias, self.eps, backend=self.backend)

    def extra_repr(self) -> str:
        return f"{self.channels}, eps={self.eps}, bias={self.bias is not None}, backend={self.backend!r}"


class LinearAct(nn.Module):
    """``linear_act`` with its weight [out_features, in_features]; PyTorch's linear initialisation."""

    def __init__(
        self,
        in_features: int,
        out_features: int,
        bias: bool = True,
        activation: str | None = None,
        device=None,
        dtype=None,
        *,
        backend="auto",
    ):
        super().__init__()
        if in_features <= 0 or out_features <= 0:
            raise ValueError("in_features and out_features must be positive")
        if activation is not None and activation not in _ACTIVATIONS:
            raise ValueError(f"Invalid activation {activation!r}; expected 'relu', 'gelu' or 'gelu_tanh'")
        self.in_features, self.out_features = in_features, out_features
        self.activation = activation
        self.backend = backend
        bound = 1 / math.sqrt(in_features)
        self.weight = nn.Parameter(torch.empty(out_features, in_features, device=device, dtype=dtype))
        nn.init.uniform_(self.weight, -bound, bound)
        if bias:
            self.bias = nn.Parameter(torch.empty(out_features, device=device, dtype=dtype))
            nn.init.uniform_(self.bias, -bound, bound)
        else:
            self.register_parameter("bias", None)

    def forward(self, input: Tensor, residual: Tensor | None = None) -> Tensor:
        return linear_act(
            input, self.weight, self.bias, residual, activation=self.activation, backend=self.backend
        )

    def extra_repr(self) -> str:
        return (
            f"{self.in_features}, {self.out_features}, bias={self.bias is not None}, "
            f"activation={self.activation!r}, backend={self.backend!r}"
        )


class GatedConvBlock(nn.Module):
    """A residual block that mixes tokens by a causal depthwise convolution and a gated recurrence,
    then channels by a two-layer perceptron:

        x = x + out(recurrence(project(conv(norm(x)))))
        x = x + down(act(up(norm(x))))

    ``forward(x, state, lengths)`` returns ``(x, state)``; the state (the last ``kernel_size - 1``
    normalised tokens and the recurrence's state) starts the next call, so a prompt is followed by
    calls of one token. ``lengths`` [batch]: tokens at and past a sequence's length are padding.
    ``backend`` is that of every part; "auto" leaves the convolution, which has one axis, to PyTorch,
    as it does for ``Conv1d``, and "native" runs it on the gfx950 kernels too.
    """

    def __init__(
        self,
        channels: int,
        kernel_size: int = 4,
        expansion: int = 4,
        activation: str | None = "gelu",
        device=None,
        dtype=None,
        *,
        backend: str = "auto",
    ):
        super().__init__()
        if kernel_size <= 0 or expansion <= 0:
            raise ValueError("kernel_size and expansion must be positive")
        factory = {"device": device, "dtype": dtype, "backend": backend}
        self.channels, self.kernel_size, self.backend = channels, kernel_size, backend
        self.norm_tokens = LayerNorm(channels, **factory)
        self.conv = Conv1d(channels, channels, kernel_size, groups=channels, **factory)
        self.project = LinearAct(channels, 2 * channels, **factory)
        self.out = LinearAct(channels, channels, **factory)
        self.norm_channels = LayerNorm(channels, **factory)
        self.up = LinearAct(channels, expansion * channels, activation=activation, **factory)
        self.down = LinearAct(expansion * channels, channels, **factory)
        with torch.no_grad():  # gates from fast to slow channels: sigmoid 0.5 .. 0.998
            self.project.bias[channels:] = torch.linspace(0, 6, channels)

    def initial_state(self, input: Tensor) -> tuple[Tensor, Tensor]:
        batch = input.shape[0]
        window = input.new_zeros((batch, self.kernel_size - 1, self.channels))
        return window, input.new_zeros((batch, self.channels), dtype=torch.float32)

    def forward(
        self, input: Tensor, state: tuple[Tensor, Tensor] | None = None, lengths: Tensor | None = None
    ) -> tuple[Tensor, tuple[Tensor, Tensor]]:
        if input.dim() != 3 or input.shape[2] != self.channels:
            raise ValueError(f"expected an input of [batch, tokens, {self.channels}]")
        window, hidden = self.initial_state(input) if state is None else state
        tokens = torch.cat((window, self.norm_tokens(input)), dim=1)
        # [N, C, T] stored as [N, T, C]: the convolution reads and writes channels-last.
        mixed = conv_nd(
            tokens.transpose(1, 2),
            self.conv.weight,
            self.conv.bias,
            groups=self.channels,
            backend=self.backend,
            memory_format=torch.preserve_format,
        ).transpose(1, 2)
        update, gate = self.project(mixed).chunk(2, dim=2)
        states, hidden = gated_recurrence(update, gate, hidden, lengths=lengths, backend=self.backend)
        output = self.out(states, input)
        output = self.down(self.up(self.norm_channels(output)), output)
        kept = self.kernel_size - 1
        if lengths is None:
            window = tokens[:, tokens.shape[1] - kept :]
            if input.shape[1] > kept:  # a view would hold the whole prompt as long as the state lives
                window = window.clone(memory_format=torch.contiguous_format)
        else:  # the last tokens before each sequence's end
            first = lengths.clamp(0, input.shape[1]).long()[:, None, None]
            index = first + torch.arange(kept, device=input.device)[None, :, None]
            window = tokens.gather(1, index.expand(-1, -1, self.channels))
        return output, (window, hidden)

    def extra_repr(self) -> str:
        return f"{self.channels}, kernel_size={self.kernel_size}, backend={self.backend!r}"
