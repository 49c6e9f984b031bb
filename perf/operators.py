"""Performance cases of the sequence operators: layer norm, the pointwise linear layer with its
epilogue, and the gated linear recurrence, as a model of convolutions over a token axis runs them.

A case is one call through the package's public entry points: a training pass (the operator, then
the gradients of every input and parameter), or an inference pass without autograd (a prompt, or
a decoding step of one token per sequence). Activations are channels-last, [..., channels].

    layer norm   y = (x - mean) / sqrt(var + eps) * weight + bias        over the last axis
    linear       y = act(x weight^T + bias) + residual
    recurrence   h_t = a_t h_(t-1) + (1 - a_t) x_t,  a_t = sigmoid(gate_t), h_0 the state given,
                 outputs past a sequence's length are 0; also the state after the last token
"""

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-5


def _norm(mode, dtype, rows, channels, name=None):
    case = {} if name is None else {"name": name}
    case.update(op="layer_norm", mode=mode, dtype=dtype, rows=rows, channels=channels)
    return case


def _linear(mode, dtype, rows, inputs, outputs, activation="none", bias=True, residual=False, name=None):
    case = {} if name is None else {"name": name}
    case.update(op="linear", mode=mode, dtype=dtype, rows=rows, inputs=inputs, outputs=outputs,
                activation=activation, bias=bias, residual=residual)
    return case


def _recurrence(mode, dtype, batch, tokens, channels, state=True, ragged=False, name=None):
    case = {} if name is None else {"name": name}
    case.update(op="recurrence", mode=mode, dtype=dtype, batch=batch, tokens=tokens, channels=channels,
                state=state, ragged=ragged)
    return case


def listed():
    return [
        # A decoding step's norm: one token of four sequences, bound by latency.
        _norm("infer", "bf16", 4, 512, name="norm_bf16_step"),
        # The norm of an ordinary training step.
        _norm("train", "bf16", 16384, 1024, name="norm_bf16_train"),
        # Single precision with odd channels: no row starts on a vector boundary.
        _norm("train", "fp32", 5003, 769, name="norm_fp32_odd_train"),
        # A wide model's training step over many tokens.
        _norm("train", "fp16", 65536, 2048, name="norm_fp16_large_train"),
        # A decoding step's expansion layer for four sequences: bound by reading the weight.
        _linear("infer", "bf16", 4, 1024, 4096, "gelu", name="linear_bf16_step"),
        # The expansion layer of a training step, activation in the epilogue.
        _linear("train", "bf16", 8192, 1024, 4096, "gelu_tanh", name="linear_bf16_train"),
        # Single precision, ragged sizes, with the residual added.
        _linear("train", "fp32", 1001, 333, 517, "gelu", residual=True, name="linear_fp32_ragged_train"),
        # The contraction layer over a batch of prompts, with the residual added.
        _linear("infer", "fp16", 16384, 4096, 1024, residual=True, name="linear_fp16_prompt"),
        # A decoding step: one token of 32 sequences from their states.
        _recurrence("infer", "bf16", 32, 1, 1024, name="recurrence_bf16_step"),
        # An ordinary training step.
        _recurrence("train", "bf16", 8, 2048, 1024, state=False, name="recurrence_bf16_train"),
        # One very long prompt of a narrow model: little to do side by side but the token axis.
        _recurrence("infer", "fp32", 1, 65536, 512, name="recurrence_fp32_long_prompt"),
        # Sequences of different lengths (some empty), odd sizes, documents packed by closed gates.
        _recurrence("train", "fp16", 13, 777, 300, ragged=True, name="recurrence_fp16_ragged_train"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _size(rng, low, high):
    """Spread over the logarithm of the range; whole eights and odd sizes alike."""
    n = _log(rng, low, high)
    n = max(8, n // 8 * 8) if rng.random() < 0.5 and n >= 8 else n
    return n + 8 if n == 3072 else n


def _draw_once(rng):
    mode = rng.choice(["train", "train", "infer"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    op = rng.choice(["layer_norm", "linear", "linear", "recurrence", "recurrence"])
    if op == "layer_norm":
        return _norm(mode, dtype, _log(rng, 1, 65536), _size(rng, 16, 8192))
    if op == "linear":
        return _linear(mode, dtype, _log(rng, 1, 16384), _size(rng, 16, 4096), _size(rng, 16, 4096),
                       rng.choice(["none", "relu", "gelu", "gelu_tanh"]), rng.random() < 0.7, rng.random() < 0.5)
    tokens = 1 if rng.random() < 0.15 else _log(rng, 2, 65536)
    return _recurrence(mode, dtype, _log(rng, 1, 64), tokens, _size(rng, 16, 4096), rng.random() < 0.6,
                       rng.random() < 0.4)


def draw(rng):
    limits = {}
    for case in listed():
        cost = work(case)
        key = case["op"]
        top = limits.get(key, (0, 0))
        limits[key] = (max(top[0], cost["bytes"]), max(top[1], cost["flops"]))
    while True:
        case = _draw_once(rng)
        cost, top = work(case), limits[case["op"]]
        # Single-precision products are several times as long as the listed 16-bit ones.
        scale = 8 if case["op"] == "linear" and case["dtype"] == "fp32" else 1
        if cost["bytes"] <= top[0] and cost["flops"] * scale <= top[1]:
            return case


def work(case):
    """Inputs once, outputs once; products and the operations of each element."""
    size = 4 if case["dtype"] == "fp32" else 2
    train = case["mode"] == "train"
    if case["op"] == "layer_norm":
        n, c = case["rows"] * case["channels"], case["channels"]
        # x (and dy) in, y (and dx) out; weight and bias in, their gradients out.
        return {"bytes": size * ((4 * n + 4 * c) if train else (2 * n + 2 * c)), "flops": (24 if train else 8) * n}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        elements = m * k + n * k + m * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        if train:  # dy in; dx, dweight and dbias out (the residual's gradient is dy itself)
            elements += m * n + m * k + n * k + (n if case["bias"] else 0)
        return {"bytes": size * elements, "flops": 2 * m * n * k * (3 if train else 1)}
    b, t, c = case["batch"], case["tokens"], case["channels"]
    states = 1 + (1 if case["state"] else 0)  # the last state, the first where one is given
    total = size * 3 * b * t * c + 4 * b * c * states
    if train:  # dy and the last state's gradient in; dx, dgate and the first state's gradient out
        total += size * 3 * b * t * c + 4 * b * c * states
    return {"bytes": total + (4 * b if case["ragged"] else 0), "flops": (30 if train else 10) * b * t * c}


def _package():
    path = str(Path(__file__).resolve().parent.parent / "torch-convnd_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import torch_convnd

    return torch_convnd


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    train = case["mode"] == "train"

    def normal(*shape, scale=1.0, offset=0.0):
        t = torch.empty(shape, device="cuda", dtype=torch.float32).normal_(generator=g)
        return t.mul_(scale).add_(offset)

    def uniform(*shape, bound=1.0):
        return torch.empty(shape, device="cuda", dtype=torch.float32).uniform_(-bound, bound, generator=g)

    def leaf(t, to=dtype):
        return t.to(to).requires_grad_(train)

    state = {"case": dict(case)}
    if case["op"] == "layer_norm":
        rows, c = case["rows"], case["channels"]
        # A residual stream: every channel has its own offset and spread, a few are large.
        spread = 1.0 + 3.0 * (normal(c) > 2).float()
        state["x"] = leaf(normal(rows, c) * spread + normal(c, scale=0.5))
        state["weight"] = leaf(normal(c, scale=0.1, offset=1.0))
        state["bias"] = leaf(normal(c, scale=0.1))
        if train:
            state["dy"] = normal(rows, c).to(dtype)
    elif case["op"] == "linear":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        bound = 1 / math.sqrt(k)
        state["x"] = leaf(normal(m, k))
        state["weight"] = leaf(uniform(n, k, bound=bound * math.sqrt(3)))
        state["bias"] = leaf(uniform(n, bound=bound)) if case["bias"] else None
        state["residual"] = leaf(normal(m, n)) if case["residual"] else None
        if train:
            state["dy"] = normal(m, n).to(dtype)
    else:
        b, t, c = case["batch"], case["tokens"], case["channels"]
        state["x"] = leaf(normal(b, t, c))
        # Channels that forget at once and channels that remember thousands of tokens.
        gate = normal(b, t, c) + torch.linspace(-1, 8, c, device="cuda")
        if case["ragged"]:  # a closed gate (sigmoid 0) is where a packed document starts
            gate[torch.rand((b, t), device="cuda", generator=g) < 0.01] = -math.inf
        state["gate"] = leaf(gate)
        state["first"] = leaf(normal(b, c), torch.float32) if case["state"] else None
        lengths = None
        if case["ragged"]:
            lengths = torch.randint(0, t + 1, (b,), device="cuda", dtype=torch.int32, generator=g)
            lengths[0] = t
            if b > 1:
                lengths[1] = 0
        state["lengths"] = lengths
        if train:
            state["dy"] = normal(b, t, c).to(dtype)
            state["dlast"] = normal(b, c)
    return state


def run(state):
    case = state["case"]
    call = {"layer_norm": _run_norm, "linear": _run_linear, "recurrence": _run_recurrence}[case["op"]]
    if own:
        return call(state, case, _package())
    plain = {"layer_norm": _plain_norm, "linear": _plain_linear, "recurrence": _plain_recurrence}[case["op"]]
    with torch.no_grad():
        return plain(state, case)


# ---- the framework's operators, as a user calls them ---------------------------------------


def _run_norm(s, case, convnd):
    if case["mode"] == "infer":
        with torch.no_grad():
            return convnd.layer_norm(s["x"], s["weight"], s["bias"], _EPS)
    y = convnd.layer_norm(s["x"], s["weight"], s["bias"], _EPS)
    return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"]))


def _run_linear(s, case, convnd):
    activation = None if case["activation"] == "none" else case["activation"]
    if case["mode"] == "infer":
        with torch.no_grad():
            return convnd.linear_act(s["x"], s["weight"], s["bias"], s["residual"], activation=activation)
    y = convnd.linear_act(s["x"], s["weight"], s["bias"], s["residual"], activation=activation)
    wanted = [t for t in (s["x"], s["weight"], s["bias"], s["residual"]) if t is not None]
    return (y.detach(), *torch.autograd.grad(y, wanted, s["dy"]))


def _run_recurrence(s, case, convnd):
    if case["mode"] == "infer":
        with torch.no_grad():
            return convnd.gated_recurrence(s["x"], s["gate"], s["first"], lengths=s["lengths"])
    h, last = convnd.gated_recurrence(s["x"], s["gate"], s["first"], lengths=s["lengths"])
    wanted = [t for t in (s["x"], s["gate"], s["first"]) if t is not None]
    return (h.detach(), last.detach(), *torch.autograd.grad((h, last), wanted, (s["dy"], s["dlast"])))


# ---- the plain forms: elementary operations in 32 bits, rounded once -------------------------


def _plain_norm(s, case):
    dtype = s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    centred = x - x.mean(dim=-1, keepdim=True)
    rstd = (centred.square().mean(dim=-1, keepdim=True) + _EPS).rsqrt()
    hat = centred * rstd
    y = (hat * w + b).to(dtype)
    if case["mode"] == "infer":
        return y
    dy = s["dy"].float()
    dhat = dy * w
    dx = rstd * (dhat - dhat.mean(dim=-1, keepdim=True) - hat * (dhat * hat).mean(dim=-1, keepdim=True))
    return y, dx.to(dtype), (dy * hat).sum(dim=0).to(dtype), dy.sum(dim=0).to(dtype)


def _activate(z, kind):
    """act(z) and act'(z)."""
    if kind == "none":
        return z, None
    if kind == "relu":
        return z.clamp(min=0), (z > 0).float()
    if kind == "gelu":
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _plain_linear(s, case):
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, slope = _activate(z, case["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    y = y.to(dtype)
    if case["mode"] == "infer":
        return y
    dz = s["dy"].float()
    if slope is not None:
        dz = dz * slope
    out = [y, (dz @ w).to(dtype), (dz.t() @ x).to(dtype)]
    if s["bias"] is not None:
        out.append(dz.sum(dim=0).to(dtype))
    if s["residual"] is not None:
        out.append(s["dy"])
    return tuple(out)


def _scan(a, u, reverse=False):
    """Every prefix of v_t = a_t v_(t-1) + u_t along axis 1, by doubling; from the end if reverse."""
    if reverse:
        return _scan(a.flip(1), u.flip(1)).flip(1)
    step, tokens = 1, a.shape[1]
    while step < tokens:
        u = torch.cat((u[:, :step], a[:, step:] * u[:, :-step] + u[:, step:]), dim=1)
        step *= 2
        if step < tokens:
            half = step // 2
            a = torch.cat((a[:, :half], a[:, half:] * a[:, :-half]), dim=1)
    return u


def _plain_recurrence(s, case):
    dtype = s["x"].dtype
    x, a = s["x"].float(), 1 / (1 + torch.exp(-s["gate"].float()))
    first = s["first"] if s["first"] is not None else x.new_zeros(x.shape[0], x.shape[2])
    valid = None
    if s["lengths"] is not None:
        valid = torch.arange(x.shape[1], device=x.device)[None, :, None] < s["lengths"][:, None, None]
    u = (1 - a) * x
    decay = a
    if valid is not None:  # past its length a sequence keeps its state
        u = torch.where(valid, u, 0)
        decay = torch.where(valid, a, 1)
    u[:, 0] += decay[:, 0] * first
    h = _scan(decay, u)
    last = h[:, -1].clone()
    y = h if valid is None else torch.where(valid, h, 0)
    if case["mode"] == "infer":
        return y.to(dtype), last
    dy = s["dy"].float()
    if valid is not None:
        dy = torch.where(valid, dy, 0)
    dy = torch.cat((dy[:, :-1], dy[:, -1:] + s["dlast"][:, None]), dim=1)
    after = torch.cat((decay[:, 1:], torch.ones_like(decay[:, :1])), dim=1)
    dh = _scan(after, dy, reverse=True)
    before = torch.cat((first[:, None], h[:, :-1]), dim=1)
    dgate = dh * (before - x) * a * (1 - a)
    dx = dh * (1 - a)
    if valid is not None:
        dgate, dx = torch.where(valid, dgate, 0), torch.where(valid, dx, 0)
    out = [y.to(dtype), last, dx.to(dtype), dgate.to(dtype)]
    if s["first"] is not None:
        out.append(dh[:, 0] * decay[:, 0])
    return tuple(out)


# ---- the definitions in 64 bits ----------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    train = case["mode"] == "train"
    wide = {k: v.detach().double().requires_grad_(train) if isinstance(v, torch.Tensor) and v.is_floating_point() else v
            for k, v in s.items()}
    if case["op"] == "layer_norm":
        with torch.set_grad_enabled(train):
            y = torch.nn.functional.layer_norm(wide["x"], (case["channels"],), wide["weight"], wide["bias"], _EPS)
        if not train:
            return y
        grads = torch.autograd.grad(y, (wide["x"], wide["weight"], wide["bias"]), wide["dy"].detach())
        return (y.detach(), *grads)
    if case["op"] == "linear":
        with torch.set_grad_enabled(train):
            y = torch.nn.functional.linear(wide["x"], wide["weight"], wide["bias"])
            if case["activation"] == "relu":
                y = torch.nn.functional.relu(y)
            elif case["activation"] != "none":
                y = torch.nn.functional.gelu(y, approximate="tanh" if case["activation"] == "gelu_tanh" else "none")
            if wide["residual"] is not None:
                y = y + wide["residual"]
        if not train:
            return y
        wanted = [wide[k] for k in ("x", "weight", "bias", "residual") if wide[k] is not None]
        return (y.detach(), *torch.autograd.grad(y, wanted, wide["dy"].detach()))
    return _exact_recurrence(case, wide)


def _exact_recurrence(case, wide):
    """Token by token, and back: each sequence stops at its own length."""
    with torch.no_grad():
        x, a = wide["x"], torch.sigmoid(wide["gate"])
        h = wide["first"].clone() if wide["first"] is not None else x.new_zeros(x.shape[0], x.shape[2])
        tokens = x.shape[1]
        live = None
        if wide["lengths"] is not None:
            live = [wide["lengths"][:, None] > t for t in range(tokens)]
        states, u = [h], (1 - a) * x
        for t in range(tokens):
            new = torch.addcmul(u[:, t], a[:, t], h)
            h = new if live is None else torch.where(live[t], new, h)
            states.append(h)
        y = torch.stack(states[1:], dim=1)
        if live is not None:
            y = torch.where(torch.stack(live, dim=1), y, 0)
        if case["mode"] == "infer":
            return y, h
        d, dy = wide["dlast"].clone(), wide["dy"]
        dhs = []
        for t in reversed(range(tokens)):
            total = d + dy[:, t]
            back = total * a[:, t]
            if live is not None:
                total, back = torch.where(live[t], total, 0), torch.where(live[t], back, d)
            dhs.append(total)
            d = back
        dh = torch.stack(dhs[::-1], dim=1)
        dgate = dh * (torch.stack(states[:-1], dim=1) - x) * a * (1 - a)
        out = [y, h, dh * (1 - a), dgate]
        if wide["first"] is not None:
            out.append(d)
        return tuple(out)
