"""Operators of token sequences around the convolution: layer norm, the linear layer with its
activation and residual, the gated linear layer, the gated linear recurrence and the gated delta rule, over activations of
[..., channels]. No counterpart in the reference.

``backend`` as for ``conv_nd``: ``auto`` runs the gfx950 kernels for ROCm GPU tensors (float16,
bfloat16, float32; other types are refused there) and PyTorch operations for other devices and
under function transforms; ``native`` asks for the gfx950 kernels, ``torch`` for the PyTorch
operations. The gfx950 kernels keep statistics, states and sums in float32, give the same bits
on every call, run on the current stream and are differentiable once.
"""

import torch
from torch import Tensor
from torch.nn import functional as F

from . import _build
from ._compat import (
    autocast_disabled,
    autocast_dtype,
    is_autocast_enabled,
    is_compiling,
    is_onnx_exporting,
    transforms_active,
)
from ._dispatch import BACKENDS
from ._toolchain import native_unavailable_reason
from .functional import _ACTIVATIONS, _apply_activation

_NATIVE_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def _use_native(input, backend, name):
    """Whether a call runs on the gfx950 kernels; loads them, or raises where they cannot."""
    if (
        _build._LOADED
        and input.is_cuda
        and input.dtype in _NATIVE_DTYPES
        and (backend == "auto" or backend == "native")
        and not transforms_active()
        and torch._C._get_tracing_state() is None
    ):
        return True
    device = input.device
    if backend not in BACKENDS:
        raise ValueError(f"Invalid backend {backend!r}; expected 'auto', 'native' or 'torch'")
    if backend == "torch" or transforms_active() or is_onnx_exporting():
        return False
    if device.type != "cuda" or torch.version.hip is None:
        if backend == "native":
            raise RuntimeError(f"The native {name} runs on ROCm GPUs; use backend='torch' or 'auto'")
        return False
    if input.dtype not in _NATIVE_DTYPES:
        raise RuntimeError(
            f"native {name} supports float16, bfloat16 and float32, not {input.dtype}; use backend='torch'"
        )
    if not _build._LOADED and not is_compiling():
        reason = native_unavailable_reason(device.type)
        if reason is not None:
            raise RuntimeError(f"Cannot load the native torch_convnd kernels: {reason}")
        _build.load_native()
    return True


def _recording(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def layer_norm(
    input: Tensor,
    weight: Tensor | None = None,
    bias: Tensor | None = None,
    eps: float = 1e-5,
    *,
    backend: str = "auto",
) -> Tensor:
    """``(input - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    ``weight`` and ``bias`` are [channels], in the input's dtype or float32 (both the same), or
    None; the result has the input's dtype and is contiguous. Channels-last activations
    ([N, C, *spatial] stored as [N, *spatial, C]) are normalised over their channels without a
    copy as ``layer_norm(x.movedim(1, -1), ...)``; inputs whose rows are a fixed stride apart (a
    slice of a wider projection) are read in place too.
    """
    if _use_native(input, backend, "layer_norm"):
        keep = _recording(input, weight, bias)
        return torch.ops.torch_convnd.layer_norm.default(input, weight, bias, eps, keep)[0]
    if input.dim() == 0 or input.shape[-1] == 0:
        raise RuntimeError("layer_norm expects an input with channels in its last dimension")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (
            p.shape != input.shape[-1:] or p.device != input.device or p.dtype not in (input.dtype, torch.float32)
        ):
            raise RuntimeError(
                f"layer_norm {name} must match the input's channels and device, in its dtype or float32"
            )
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("layer_norm weight and bias must have the same dtype")
    wide = torch.float64 if input.dtype == torch.float64 else torch.float32
    cast = lambda t: None if t is None else t.to(wide)  # noqa: E731
    return F.layer_norm(cast(input), input.shape[-1:], cast(weight), cast(bias), eps).to(input.dtype)


def linear_act(
    input: Tensor,
    weight: Tensor,
    bias: Tensor | None = None,
    residual: Tensor | None = None,
    *,
    activation: str | None = None,
    backend: str = "auto",
) -> Tensor:
    """``act(input @ weight.T + bias) + residual`` over the last dimension of ``input`` [..., inputs].

    ``weight`` is [outputs, inputs], ``bias`` [outputs], ``residual`` of the output's shape
    [..., outputs]; all in the input's dtype. ``activation`` as for ``conv_nd``: "relu", "gelu",
    "gelu_tanh" or None. On the gfx950 path all of it is one rounding of the float32 sums (a training
    step also keeps the activation's slope, in 16 bits beside 16-bit types, else float32, and its
    backward rounds the gradient before the activation to the element type). ``input`` and
    ``residual`` may be slices of wider rows. Under autocast the operands are cast to its dtype, the
    residual too: a residual stream in float32 is added outside (``x + linear_act(...)``).
    """
    if activation is not None and activation not in _ACTIVATIONS:
        raise ValueError(f"Invalid activation {activation!r}; expected 'relu', 'gelu' or 'gelu_tanh'")
    if is_autocast_enabled(input.device.type):
        dtype = autocast_dtype(input.device.type)
        cast = lambda t: t.to(dtype) if t is not None and t.dtype in _NATIVE_DTYPES else t  # noqa: E731
        input, weight, bias, residual = cast(input), cast(weight), cast(bias), cast(residual)
    if _use_native(input, backend, "linear_act"):
        keep = _recording(input, weight, bias, residual)
        return torch.ops.torch_convnd.linear_act.default(
            input, weight, bias, residual, activation or "none", keep
        )[0]
    return _portable_linear(input, weight, bias, residual, activation)


def _portable_linear(input, weight, bias, residual, activation):
    if weight.dim() != 2 or input.dim() == 0 or input.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise RuntimeError("linear_act expects an input of [..., inputs] and a weight of [outputs, inputs]")
    if weight.device != input.device or weight.dtype != input.dtype:
        raise RuntimeError("input and weight must have the same device and dtype")
    if bias is not None and (
        bias.shape != weight.shape[:1] or bias.device != input.device or bias.dtype != input.dtype
    ):
        raise RuntimeError("bias must match the outputs, device and dtype")
    shape = (*input.shape[:-1], weight.shape[0])
    if residual is not None and (
        residual.shape != shape or residual.device != input.device or residual.dtype != input.dtype
    ):
        raise RuntimeError("residual must match the output's shape, device and dtype")
    wide = torch.float64 if input.dtype == torch.float64 else torch.float32
    with autocast_disabled(input.device.type):
        output = F.linear(input.to(wide), weight.to(wide), None if bias is None else bias.to(wide))
        output = _apply_activation(output, activation)
        if residual is not None:
            output = output + residual.to(wide)
    return output.to(input.dtype)


_GATED_ACTIVATIONS = ("silu", "relu", "gelu", "gelu_tanh")


def gated_linear(
    input: Tensor,
    weight: Tensor,
    bias: Tensor | None = None,
    *,
    activation: str = "silu",
    backend: str = "auto",
) -> Tensor:
    """``act(input @ Wg.T + bg) * (input @ Wu.T + bu)`` over the last dimension of ``input`` [..., inputs]:
    the two projections of a gated feed-forward block, its activation and the product.

    ``weight`` [2 * outputs, inputs] is Wg above Wu, ``bias`` [2 * outputs] bg before bu, in the input's
    dtype; ``activation`` is "silu", "relu", "gelu" or "gelu_tanh". On the gfx950 path all of it is one
    rounding of the float32 sums; a training step also keeps two factors an output (in 24 bits beside
    16-bit types, else float32), and its backward rounds the gradients before the product to the element
    type. ``input`` may be a slice of wider rows. Under autocast the operands are cast to its dtype.
    """
    if activation not in _GATED_ACTIVATIONS:
        raise ValueError(f"Invalid activation {activation!r}; expected 'silu', 'relu', 'gelu' or 'gelu_tanh'")
    if is_autocast_enabled(input.device.type):
        dtype = autocast_dtype(input.device.type)
        cast = lambda t: t.to(dtype) if t is not None and t.dtype in _NATIVE_DTYPES else t  # noqa: E731
        input, weight, bias = cast(input), cast(weight), cast(bias)
    if _use_native(input, backend, "gated_linear"):
        keep = _recording(input, weight, bias)
        return torch.ops.torch_convnd.gated_linear.default(input, weight, bias, activation, keep)[0]
    if (
        weight.dim() != 2
        or input.dim() == 0
        or input.shape[-1] != weight.shape[1]
        or weight.numel() == 0
        or weight.shape[0] % 2
    ):
        raise RuntimeError("gated_linear expects an input of [..., inputs] and a weight of [2 * outputs, inputs]")
    if weight.device != input.device or weight.dtype != input.dtype:
        raise RuntimeError("input and weight must have the same device and dtype")
    if bias is not None and (
        bias.shape != weight.shape[:1] or bias.device != input.device or bias.dtype != input.dtype
    ):
        raise RuntimeError("bias must match the weight's rows, device and dtype")
    wide = torch.float64 if input.dtype == torch.float64 else torch.float32
    with autocast_disabled(input.device.type):
        both = F.linear(input.to(wide), weight.to(wide), None if bias is None else bias.to(wide))
        gate, up = both.chunk(2, dim=-1)
        gate = F.silu(gate) if activation == "silu" else _apply_activation(gate, activation)
        return (gate * up).to(input.dtype)


def gated_recurrence(
    input: Tensor,
    gate: Tensor,
    initial_state: Tensor | None = None,
    *,
    lengths: Tensor | None = None,
    backend: str = "auto",
) -> tuple[Tensor, Tensor]:
    """``h[t] = a[t] * h[t-1] + (1 - a[t]) * input[t]`` with ``a = sigmoid(gate)`` over the tokens of
    ``input`` and ``gate`` [batch, tokens, channels]; returns ``(h, last_state)``.

    ``initial_state`` and ``last_state`` are float32 [batch, channels] (zeros if None), so that a
    prompt's last state starts the next call, of one token when decoding. ``lengths`` (int32 or
    int64 [batch]): tokens at and past a sequence's length leave its state as it is and give zeros,
    whatever the inputs hold there; a length below 0 counts as 0, one above ``tokens`` as
    ``tokens``. A gate of -inf closes it (``a`` = 0): a token that forgets all before it, where a
    packed document starts. Inputs may be strided (slices of one projection) as long as their
    channels are contiguous.
    """
    if is_autocast_enabled(input.device.type) and input.dtype != gate.dtype:
        dtype = autocast_dtype(input.device.type)
        input, gate = input.to(dtype), gate.to(dtype)
    if _use_native(input, backend, "gated_recurrence"):
        keep = _recording(input, gate, initial_state)
        h, last, _ = torch.ops.torch_convnd.gated_recurrence.default(input, gate, initial_state, lengths, keep)
        return h, last
    return _portable_recurrence(input, gate, initial_state, lengths)


def _portable_recurrence(input, gate, initial_state, lengths):
    """Token by token in float32 (float64 for float64 inputs)."""
    if input.dim() != 3 or input.shape[2] == 0:
        raise RuntimeError("gated_recurrence expects an input of [batch, tokens, channels]")
    if gate.shape != input.shape or gate.device != input.device or gate.dtype != input.dtype:
        raise RuntimeError("gated_recurrence gate must match the input's shape, device and dtype")
    batch, tokens, channels = input.shape
    wide = torch.float64 if input.dtype == torch.float64 else torch.float32
    if initial_state is not None and (
        initial_state.shape != (batch, channels)
        or initial_state.device != input.device
        or initial_state.dtype not in (torch.float32, wide)
    ):
        raise RuntimeError(
            "gated_recurrence initial_state must be float32 of [batch, channels] on the input's device"
        )
    if lengths is not None and (
        lengths.shape != (batch,)
        or lengths.device != input.device
        or lengths.dtype not in (torch.int32, torch.int64)
    ):
        raise RuntimeError(
            "gated_recurrence lengths must be int32 or int64 of [batch] on the input's device"
        )
    h = input.new_zeros((batch, channels), dtype=wide) if initial_state is None else initial_state.to(wide)
    x, g = input.to(wide), gate.to(wide)
    if lengths is not None:
        # An open gate and a zero before any arithmetic, so that nothing held past a length
        # reaches a state or a gradient.
        live = (torch.arange(tokens, device=input.device) < lengths[:, None])[..., None]
        x, g = torch.where(live, x, 0), torch.where(live, g, torch.inf)
    keep, take = torch.sigmoid(g), torch.sigmoid(-g)
    states = []
    for t in range(tokens):
        h = keep[:, t] * h + take[:, t] * x[:, t]
        states.append(h)
    output = torch.stack(states, dim=1) if states else x
    if lengths is not None:
        output = torch.where(live, output, 0)
    return output.to(input.dtype), h


def gated_delta_rule(
    query: Tensor,
    key: Tensor,
    value: Tensor,
    decay: Tensor,
    beta: Tensor,
    initial_state: Tensor | None = None,
    *,
    lengths: Tensor | None = None,
    scale: float | None = None,
    normalize: bool = False,
    backend: str = "auto",
) -> tuple[Tensor, Tensor]:
    """A matrix state a head, corrected towards each token's value; returns ``(output, last_state)``:

        S[t] = a[t] * S[t-1] + k[t] u[t]^T,  u[t] = beta[t] * (v[t] - a[t] * S[t-1]^T k[t])
        output[t] = scale * S[t]^T q[t],  a = exp(decay)

    ``query`` and ``key`` are [batch, tokens, key_heads, key_size], ``value`` [batch, tokens, heads,
    value_size] with ``heads`` a multiple of ``key_heads`` (value heads share the query and key head of
    their group, in order). ``decay`` (the logarithm of what a token keeps of the state) and ``beta``
    are [batch, tokens, heads], both in the inputs' dtype or float32. ``scale`` is ``key_size ** -0.5`` if
    None; ``normalize`` divides q and k by ``sqrt(|.|^2 + 1e-6)``, without which keys have to be of
    about unit length (a beta of more than 2 / |k|^2 makes the state grow without end).

    ``initial_state`` and ``last_state`` are float32 [batch, heads, key_size, value_size] (zeros if None), so
    that a prompt's last state starts the next call, of one token when decoding. ``lengths`` as for
    ``gated_recurrence``. A decay of -inf (below -104, where its exp in float32 is zero) forgets all before
    it (that is finite): where a packed document starts. The gfx950 kernels take key sizes up to 128. They read slices of
    wider rows in place, keep states in float32 and products within the last bits of the result's dtype, and
    take more than a few tokens in chunks: there a NaN reaches its whole chunk of 64 tokens, an infinity as a
    NaN, and beside float16 states, and what is added to them, have to be within its range. Their backward keeps
    states' gradients beside float16 in units of a head's largest cotangent, up to 2^13 times it.
    """
    if is_autocast_enabled(query.device.type):
        dtype = autocast_dtype(query.device.type)
        cast = lambda t: t.to(dtype) if t.dtype in _NATIVE_DTYPES else t  # noqa: E731
        query, key, value = cast(query), cast(key), cast(value)
        if decay.dtype != beta.dtype or decay.dtype != torch.float32:
            decay, beta = cast(decay), cast(beta)
    if scale is None:
        scale = query.shape[-1] ** -0.5 if query.dim() > 0 and query.shape[-1] > 0 else 1.0
    if _use_native(query, backend, "gated_delta_rule"):
        keep = _recording(query, key, value, decay, beta, initial_state)
        output, last, _ = torch.ops.torch_convnd.gated_delta_rule.default(
            query, key, value, decay, beta, initial_state, lengths, scale, normalize, keep
        )
        return output, last
    return _portable_delta(query, key, value, decay, beta, initial_state, lengths, scale, normalize)


def _portable_delta(query, key, value, decay, beta, initial_state, lengths, scale, normalize):
    """Token by token in float32 (float64 for float64 inputs)."""
    if query.dim() != 4 or key.shape != query.shape or query.shape[2] == 0 or query.shape[3] == 0:
        raise RuntimeError("gated_delta_rule expects query and key of [batch, tokens, key_heads, key_size]")
    batch, tokens, key_heads, key_size = query.shape
    if (
        value.dim() != 4
        or value.shape[:2] != query.shape[:2]
        or value.shape[2] == 0
        or value.shape[3] == 0
        or value.shape[2] % key_heads
    ):
        raise RuntimeError(
            "gated_delta_rule expects a value of [batch, tokens, heads, value_size], heads a multiple of key_heads"
        )
    heads, value_size = value.shape[2:]
    if decay.shape != value.shape[:3] or beta.shape != value.shape[:3]:
        raise RuntimeError("gated_delta_rule expects decay and beta of [batch, tokens, heads]")
    if any(t.device != query.device or t.dtype != query.dtype for t in (key, value)):
        raise RuntimeError("gated_delta_rule query, key and value must have the same device and dtype")
    if (
        decay.device != query.device
        or beta.device != query.device
        or beta.dtype != decay.dtype
        or decay.dtype not in (query.dtype, torch.float32)
    ):
        raise RuntimeError(
            "gated_delta_rule decay and beta must be on the inputs' device, both of their dtype or float32"
        )
    wide = torch.float64 if query.dtype == torch.float64 else torch.float32
    shape = (batch, heads, key_size, value_size)
    if initial_state is not None and (
        initial_state.shape != shape
        or initial_state.device != query.device
        or initial_state.dtype not in (torch.float32, wide)
    ):
        raise RuntimeError(
            "gated_delta_rule initial_state must be float32 of [batch, heads, key_size, value_size] on the "
            "inputs' device"
        )
    if lengths is not None and (
        lengths.shape != (batch,)
        or lengths.device != query.device
        or lengths.dtype not in (torch.int32, torch.int64)
    ):
        raise RuntimeError("gated_delta_rule lengths must be int32 or int64 of [batch] on the inputs' device")
    state = query.new_zeros(shape, dtype=wide) if initial_state is None else initial_state.to(wide)
    q, k, v, g, b = (t.to(wide) for t in (query, key, value, decay, beta))
    if lengths is not None:
        # Tokens that do nothing, before any arithmetic, so that nothing held past a length reaches a
        # state or a gradient.
        live = torch.arange(tokens, device=query.device) < lengths[:, None]
        q, k, v = (torch.where(live[..., None, None], t, 0) for t in (q, k, v))
        g, b = (torch.where(live[..., None], t, 0) for t in (g, b))
    if normalize:
        q = q / (q.square().sum(dim=-1, keepdim=True) + 1e-6).sqrt()
        k = k / (k.square().sum(dim=-1, keepdim=True) + 1e-6).sqrt()
    q = (q * scale).repeat_interleave(heads // key_heads, dim=2)
    k = k.repeat_interleave(heads // key_heads, dim=2)
    keep = torch.where(g < -104, 0, torch.exp(g))
    outputs = []
    for t in range(tokens):
        state = keep[:, t, :, None, None] * state
        update = b[:, t, :, None] * (v[:, t] - (k[:, t, :, :, None] * state).sum(dim=2))
        state = state + k[:, t, :, :, None] * update[:, :, None, :]
        outputs.append((q[:, t, :, :, None] * state).sum(dim=2))
    output = torch.stack(outputs, dim=1) if outputs else v
    if lengths is not None:
        output = torch.where(live[..., None, None], output, 0)
    return output.to(value.dtype), state
