"""Performance cases of the sequence operators of a delta-rule block: the gated delta rule (a matrix
state a head that is corrected towards each token's value) and the gated linear layer (two
projections, the activation of one times the other).

A case is one call through the package's public entry points: a training pass (the operator, then
the gradients of every input and parameter), or an inference pass without autograd (a prompt, or
a decoding step of one token per sequence).

    delta rule   S_t = a_t S_(t-1) + k_t u_t^T,  u_t = beta_t (v_t - a_t S_(t-1)^T k_t),  a_t = exp(log_decay_t)
                 o_t = scale S_t^T q_t, S_0 the state given; also the state after the last token.
                 q and k are divided by sqrt(|.|^2 + 1e-6) where `normalize` says so; value heads share the
                 query and key head of their group; outputs past a sequence's length are 0
    gated linear y = act(x Wg^T + bg) * (x Wu^T + bu), weight = [Wg; Wu]
"""

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_NORM_EPS = 1e-6


def _delta(mode, dtype, batch, tokens, key_heads, heads, key_size, value_size, normalize=True, state=True,
           ragged=False, name=None):
    case = {} if name is None else {"name": name}
    case.update(op="delta", mode=mode, dtype=dtype, batch=batch, tokens=tokens, key_heads=key_heads, heads=heads,
                key_size=key_size, value_size=value_size, normalize=normalize, state=state, ragged=ragged)
    return case


def _gated(mode, dtype, rows, inputs, outputs, activation="silu", bias=False, name=None):
    case = {} if name is None else {"name": name}
    case.update(op="gated", mode=mode, dtype=dtype, rows=rows, inputs=inputs, outputs=outputs,
                activation=activation, bias=bias)
    return case


def listed():
    return [
        # A decoding step: one token of 32 sequences from their states, bound by reading and writing them.
        _delta("infer", "bf16", 32, 1, 8, 8, 128, 128, name="delta_bf16_step"),
        # An ordinary training step of 1024 channels.
        _delta("train", "bf16", 8, 2048, 8, 8, 128, 128, state=False, name="delta_bf16_train"),
        # A wide model's training step, two value heads a key head.
        _delta("train", "bf16", 8, 4096, 8, 16, 128, 128, state=False, name="delta_bf16_large_train"),
        # One very long prompt: little to do side by side but the token axis.
        _delta("infer", "bf16", 1, 32768, 8, 8, 128, 128, name="delta_bf16_long_prompt"),
        # A batch of prompts of different lengths (some empty), small heads.
        _delta("infer", "fp16", 16, 517, 4, 8, 64, 64, ragged=True, name="delta_fp16_ragged_prompt"),
        # Single precision, odd sizes of everything, documents packed by decays of -inf.
        _delta("train", "fp32", 5, 333, 3, 6, 40, 71, normalize=False, ragged=True, name="delta_fp32_ragged_train"),
        # A decoding step's gated expansion for four sequences: bound by reading the weight.
        _gated("infer", "bf16", 4, 1024, 2736, name="gated_bf16_step"),
        # The gated expansion of a training step.
        _gated("train", "bf16", 8192, 1024, 2736, name="gated_bf16_train"),
        # Single precision, ragged sizes, biases.
        _gated("train", "fp32", 1001, 333, 259, "gelu", bias=True, name="gated_fp32_ragged_train"),
        # A batch of prompts.
        _gated("infer", "fp16", 4096, 2048, 5504, name="gated_fp16_prompt"),
        # A wide model's training step over many tokens.
        _gated("train", "bf16", 16384, 2048, 5504, "gelu_tanh", name="gated_bf16_large_train"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _size(rng, low, high):
    """Spread over the logarithm of the range; whole eights and odd sizes alike."""
    n = _log(rng, low, high)
    return max(8, n // 8 * 8) if rng.random() < 0.5 and n >= 8 else n


def _draw_once(rng):
    mode = rng.choice(["train", "train", "infer"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if rng.random() < 0.45:
        return _gated(mode, dtype, _log(rng, 1, 16384), _size(rng, 16, 2048), _size(rng, 16, 5504),
                      rng.choice(["silu", "silu", "relu", "gelu", "gelu_tanh"]), rng.random() < 0.4)
    tokens = 1 if mode == "infer" and rng.random() < 0.25 else _log(rng, 2, 32768)
    key_heads = _log(rng, 1, 8)
    heads = key_heads * rng.choice([1, 1, 2, 3])
    sizes = rng.choice([(64, 64), (128, 128), (128, 128), None])
    if sizes is None:
        sizes = (_size(rng, 16, 128), _size(rng, 16, 256))
    return _delta(mode, dtype, _log(rng, 1, 32), tokens, key_heads, heads, *sizes, rng.random() < 0.7,
                  rng.random() < 0.6, rng.random() < 0.4)


def draw(rng):
    limits = {}
    for case in listed():
        cost = work(case)
        top = limits.get(case["op"], (0, 0))
        limits[case["op"]] = (max(top[0], cost["bytes"]), max(top[1], cost["flops"]))
    while True:
        case = _draw_once(rng)
        cost, top = work(case), limits[case["op"]]
        # Single-precision products are several times as long as the listed 16-bit ones.
        scale = 8 if case["dtype"] == "fp32" else 1
        if cost["bytes"] <= top[0] and cost["flops"] * scale <= top[1]:
            return case


def work(case):
    """Inputs once, outputs once; the products of the definition."""
    size = 4 if case["dtype"] == "fp32" else 2
    train = case["mode"] == "train"
    if case["op"] == "gated":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        bias = 2 * n if case["bias"] else 0
        elements = m * k + 2 * n * k + m * n + bias
        if train:  # dy in; dx, dweight and dbias out
            elements += m * n + m * k + 2 * n * k + bias
        return {"bytes": size * elements, "flops": 4 * m * n * k * (3 if train else 1)}
    b, t, hk, h = case["batch"], case["tokens"], case["key_heads"], case["heads"]
    dk, dv = case["key_size"], case["value_size"]
    states = 4 * b * h * dk * dv * (1 + (1 if case["state"] else 0))
    # q, k, v, decays and betas in, o out.
    total = b * t * size * (2 * hk * dk + 2 * h * dv + 2 * h) + states
    if train:  # do in; dq, dk, dv and the decays' and betas' gradients out
        total += b * t * size * (2 * hk * dk + 2 * h * dv + 2 * h) + states
    # Three products of a state and a vector a token: S^T k, k u^T, S^T q.
    return {"bytes": total + (4 * b if case["ragged"] else 0), "flops": 6 * b * t * h * dk * dv * (3 if train else 1)}


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

    def uniform(*shape, low=-1.0, high=1.0):
        return torch.empty(shape, device="cuda", dtype=torch.float32).uniform_(low, high, generator=g)

    def leaf(t, to=dtype):
        return t.to(to).requires_grad_(train)

    state = {"case": dict(case)}
    if case["op"] == "gated":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        bound = 1 / math.sqrt(k)
        state["x"] = leaf(normal(m, k))
        state["weight"] = leaf(uniform(2 * n, k, low=-bound, high=bound).mul_(math.sqrt(3)))
        state["bias"] = leaf(uniform(2 * n, low=-bound, high=bound)) if case["bias"] else None
        if train:
            state["dy"] = normal(m, n).to(dtype)
        return state
    b, t, hk, h = case["batch"], case["tokens"], case["key_heads"], case["heads"]
    dk, dv = case["key_size"], case["value_size"]
    # Keys that share a direction, as a projection's keys do; of about unit length where they are not
    # normalised by the operator.
    spread = 1.0 if case["normalize"] else 1 / math.sqrt(1.25 * dk)
    state["query"] = leaf(normal(b, t, hk, dk))
    state["key"] = leaf((normal(b, t, hk, dk) + normal(1, 1, hk, dk, scale=0.5)).mul_(spread))
    state["value"] = leaf(normal(b, t, h, dv))
    # Heads that forget within a few tokens and heads that remember thousands.
    rate = torch.exp(torch.linspace(math.log(0.5), math.log(5e-4), h, device="cuda"))
    decay = -rate * torch.nn.functional.softplus(normal(b, t, h))
    if case["ragged"]:  # a decay of -inf is where a packed document starts
        decay[torch.rand((b, t), device="cuda", generator=g) < 0.01] = -math.inf
    state["decay"] = leaf(decay)
    state["beta"] = leaf(torch.sigmoid(normal(b, t, h)))
    state["first"] = leaf(normal(b, h, dk, dv, scale=0.3), torch.float32) if case["state"] else None
    state["lengths"] = None
    if case["ragged"]:
        lengths = torch.randint(0, t + 1, (b,), device="cuda", dtype=torch.int32, generator=g)
        lengths[0] = t
        if b > 1:
            lengths[1] = 0
        state["lengths"] = lengths
    if train:
        state["dy"] = normal(b, t, h, dv).to(dtype)
        state["dlast"] = normal(b, h, dk, dv, scale=0.1)
    return state


def run(state):
    case = state["case"]
    if own:
        call = {"delta": _run_delta, "gated": _run_gated}[case["op"]]
        return call(state, case, _package())
    with torch.no_grad():
        return (_plain_delta if case["op"] == "delta" else _plain_gated)(state, case)


# ---- the framework's operators, as a user calls them ---------------------------------------


def _run_gated(s, case, convnd):
    if case["mode"] == "infer":
        with torch.no_grad():
            return convnd.gated_linear(s["x"], s["weight"], s["bias"], activation=case["activation"])
    y = convnd.gated_linear(s["x"], s["weight"], s["bias"], activation=case["activation"])
    wanted = [t for t in (s["x"], s["weight"], s["bias"]) if t is not None]
    return (y.detach(), *torch.autograd.grad(y, wanted, s["dy"]))


def _run_delta(s, case, convnd):
    inputs = (s["query"], s["key"], s["value"], s["decay"], s["beta"], s["first"])
    options = {"lengths": s["lengths"], "normalize": case["normalize"]}
    if case["mode"] == "infer":
        with torch.no_grad():
            return convnd.gated_delta_rule(*inputs, **options)
    o, last = convnd.gated_delta_rule(*inputs, **options)
    wanted = [t for t in inputs if t is not None]
    return (o.detach(), last.detach(), *torch.autograd.grad((o, last), wanted, (s["dy"], s["dlast"])))


# ---- the plain forms: elementary operations in 32 bits, rounded once -------------------------


def _activate(z, kind):
    """act(z) and act'(z)."""
    if kind == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p + z * p * (1 - p)
    if kind == "relu":
        return z.clamp(min=0), (z > 0).float()
    if kind == "gelu":
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _plain_gated(s, case):
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    gate, up = z.chunk(2, dim=1)
    act, slope = _activate(gate, case["activation"])
    y = (act * up).to(dtype)
    if case["mode"] == "infer":
        return y
    dy = s["dy"].float()
    dz = torch.cat((dy * up * slope, dy * act), dim=1)
    out = [y, (dz @ w).to(dtype), (dz.t() @ x).to(dtype)]
    if s["bias"] is not None:
        out.append(dz.sum(dim=0).to(dtype))
    return tuple(out)


_CHUNK = 64


def _chunks(t, count, groups=1):
    """[batch, tokens, heads, ...] as [batch, heads, chunks, chunk, ...] in float, shared heads repeated."""
    t = t.float()
    pad = count * _CHUNK - t.shape[1]
    if pad:
        t = torch.cat((t, t.new_zeros(t.shape[0], pad, *t.shape[2:])), dim=1)
    t = t.reshape(t.shape[0], count, _CHUNK, *t.shape[2:]).movedim(3, 1)
    return t.repeat_interleave(groups, dim=1) if groups > 1 else t


def _plain_step(s, case):
    """One token a sequence: the definition itself."""
    groups = case["heads"] // case["key_heads"]
    q = s["query"][:, 0].float().repeat_interleave(groups, dim=1)
    k = s["key"][:, 0].float().repeat_interleave(groups, dim=1)
    if case["normalize"]:
        q = q * torch.rsqrt(q.square().sum(dim=-1, keepdim=True) + _NORM_EPS)
        k = k * torch.rsqrt(k.square().sum(dim=-1, keepdim=True) + _NORM_EPS)
    v, beta = s["value"][:, 0].float(), s["beta"][:, 0, :, None].float()
    first = s["first"] if s["first"] is not None else q.new_zeros(*k.shape, v.shape[-1])
    state = torch.exp(s["decay"][:, 0].float())[..., None, None] * first
    u = beta * (v - (k[..., None] * state).sum(dim=-2))
    state = state + k[..., None] * u[..., None, :]
    o = (q[..., None] * state).sum(dim=-2) / math.sqrt(case["key_size"])
    if s["lengths"] is not None:
        live = s["lengths"] > 0
        o, state = torch.where(live[:, None, None], o, 0), torch.where(live[:, None, None, None], state, first)
    return o[:, None].to(s["value"].dtype), state


def _plain_delta(s, case):
    """Chunks of the token axis: what tokens of a chunk do to each other as triangular matrices, then
    a walk over the chunks with the state, and one back."""
    if case["mode"] == "infer" and case["tokens"] == 1:
        return _plain_step(s, case)
    dtype, tokens, groups = s["value"].dtype, case["tokens"], case["heads"] // case["key_heads"]
    scale = 1 / math.sqrt(case["key_size"])
    n = (tokens + _CHUNK - 1) // _CHUNK
    decay = s["decay"]
    live = None
    inputs = [s["query"], s["key"], s["value"], decay, s["beta"]]
    if s["lengths"] is not None:  # a token past its sequence's length does nothing
        live = torch.arange(tokens, device=decay.device)[None, :] < s["lengths"][:, None]
        inputs = [torch.where(live.reshape(*live.shape, *(1,) * (t.dim() - 2)), t, 0) for t in inputs]
    q, k, v, decay, beta = inputs
    q, k, v = _chunks(q, n, groups), _chunks(k, n, groups), _chunks(v, n)
    decay, beta = _chunks(decay, n), _chunks(beta, n)
    q_raw, k_raw = q, k
    if case["normalize"]:
        rq = torch.rsqrt(q.square().sum(dim=-1, keepdim=True) + _NORM_EPS)
        rk = torch.rsqrt(k.square().sum(dim=-1, keepdim=True) + _NORM_EPS)
        q, k = q * rq, k * rk
    q = q * scale
    # Sums of decays in 64 bits; a closed gate is left out of them and counted.
    closed = torch.isneginf(decay)
    total = torch.where(closed, 0, decay).double().cumsum(dim=-1)
    document = closed.int().cumsum(dim=-1)
    row, col = torch.arange(_CHUNK, device=q.device)[:, None], torch.arange(_CHUNK, device=q.device)[None, :]
    ratio = torch.exp(total[..., :, None] - total[..., None, :]).float()
    ratio = torch.where((row >= col) & (document[..., :, None] == document[..., None, :]), ratio, 0)
    since = torch.where(document == 0, torch.exp(total).float(), 0)  # from the state before the chunk
    until = ratio[..., -1, :]  # to the state after it
    kk, qk = k @ k.transpose(-1, -2), q @ k.transpose(-1, -2)
    a = torch.where(row > col, beta[..., None] * ratio * kk, 0)
    inverse = torch.eye(_CHUNK, device=q.device).expand_as(a).clone()
    for i in range(1, _CHUNK):
        inverse[..., i, :i] = -(a[..., i : i + 1, :i] @ inverse[..., :i, :i])[..., 0, :]
    p = ratio * qk
    state = s["first"] if s["first"] is not None else q.new_zeros(*q.shape[:2], q.shape[-1], v.shape[-1])
    states, us, os, rs = [], [], [], []
    for c in range(n):
        states.append(state)
        r = v[:, :, c] - since[:, :, c, :, None] * (k[:, :, c] @ state)
        u = inverse[:, :, c] @ (beta[:, :, c, :, None] * r)
        os.append(since[:, :, c, :, None] * (q[:, :, c] @ state) + p[:, :, c] @ u)
        state = since[:, :, c, -1, None, None] * state + k[:, :, c].transpose(-1, -2) @ (until[:, :, c, :, None] * u)
        us.append(u)
        rs.append(r)

    def tokens_first(t, to=dtype):
        t = t.movedim(1, 3).reshape(t.shape[0], n * _CHUNK, t.shape[1], *t.shape[4:])[:, :tokens]
        if live is not None:
            t = torch.where(live.reshape(*live.shape, *(1,) * (t.dim() - 2)), t, 0)
        return t.to(to)

    o, last = tokens_first(torch.stack(os, dim=2)), state
    if case["mode"] == "infer":
        return o, last
    do = s["dy"]
    if live is not None:
        do = torch.where(live[..., None, None], do, 0)
    do = _chunks(do, n)
    dstate = s["dlast"]
    ys, dstates = [], []
    for c in reversed(range(n)):
        dstates.append(dstate)
        du = p[:, :, c].transpose(-1, -2) @ do[:, :, c] + until[:, :, c, :, None] * (k[:, :, c] @ dstate)
        y = inverse[:, :, c].transpose(-1, -2) @ du
        ys.append(y)
        dstate = (since[:, :, c, -1, None, None] * dstate
                  + q[:, :, c].transpose(-1, -2) @ (since[:, :, c, :, None] * do[:, :, c])
                  - k[:, :, c].transpose(-1, -2) @ ((since * beta)[:, :, c, :, None] * y))
    y, dstates = torch.stack(ys[::-1], dim=2), torch.stack(dstates[::-1], dim=2)
    u, r, states = torch.stack(us, dim=2), torch.stack(rs, dim=2), torch.stack(states, dim=2)
    dv = beta[..., None] * y
    dp = ratio * (do @ u.transpose(-1, -2))
    da = torch.where(row > col, -ratio * (y @ u.transpose(-1, -2)), 0)
    dq_state = since[..., None] * (do @ states.transpose(-1, -2))
    dk_value = -(since * beta)[..., None] * (y @ states.transpose(-1, -2))
    dk_state = until[..., None] * (u @ dstates.transpose(-1, -2))
    db = beta[..., None] * da
    dq = dq_state + dp @ k
    dk = dk_value + dk_state + dp.transpose(-1, -2) @ q + db @ k + db.transpose(-1, -2) @ k
    dbeta = (y * r).sum(dim=-1) + (da * kk).sum(dim=-1)
    # Gradients of the sums of decays, then of the decays.
    pairs = dp * qk + db * kk
    kept = (k * dk_state).sum(dim=-1)
    dtotal = (q * dq_state).sum(dim=-1) + (k * dk_value).sum(dim=-1) + pairs.sum(dim=-1) - pairs.sum(dim=-2) - kept
    dtotal[..., -1] += kept.sum(dim=-1) + since[..., -1] * (dstates * states).sum(dim=(-1, -2))
    ddecay = torch.where(closed, 0, dtotal.flip(-1).cumsum(dim=-1).flip(-1))
    dq = dq * scale
    if case["normalize"]:
        qn, kn = q_raw * rq, k_raw * rk
        dq = rq * (dq - qn * (qn * dq).sum(dim=-1, keepdim=True))
        dk = rk * (dk - kn * (kn * dk).sum(dim=-1, keepdim=True))
    if groups > 1:
        dq, dk = (t.reshape(t.shape[0], -1, groups, *t.shape[2:]).sum(dim=2) for t in (dq, dk))
    out = [o, last, tokens_first(dq), tokens_first(dk), tokens_first(dv),
           tokens_first(ddecay), tokens_first(dbeta)]
    if s["first"] is not None:
        out.append(dstate)
    return tuple(out)


# ---- the definitions in 64 bits ----------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "delta" and case["tokens"] > (8192 if case["mode"] == "train" else 40000):
        return None  # token by token: too long
    s = prepare(case, seed)
    train = case["mode"] == "train"
    wide = {k: v.detach().double().requires_grad_(train) if isinstance(v, torch.Tensor) and v.is_floating_point() else v
            for k, v in s.items()}
    if case["op"] == "delta":
        return _exact_delta(case, wide)
    with torch.set_grad_enabled(train):
        gate, up = torch.nn.functional.linear(wide["x"], wide["weight"], wide["bias"]).chunk(2, dim=1)
        if case["activation"] == "silu":
            gate = torch.nn.functional.silu(gate)
        elif case["activation"] == "relu":
            gate = torch.nn.functional.relu(gate)
        else:
            gate = torch.nn.functional.gelu(gate, approximate="tanh" if case["activation"] == "gelu_tanh" else "none")
        y = gate * up
    if not train:
        return y
    wanted = [wide[k] for k in ("x", "weight", "bias") if wide[k] is not None]
    return (y.detach(), *torch.autograd.grad(y, wanted, wide["dy"].detach()))


def _exact_delta(case, wide):
    """Token by token. The gradients segment by segment from the end, each segment run again from its
    first state."""
    tokens, groups = case["tokens"], case["heads"] // case["key_heads"]
    scale, first = 1 / math.sqrt(case["key_size"]), wide["first"]
    lengths = wide["lengths"]

    def walk(state, q, k, v, decay, beta, start):
        if case["normalize"]:
            q = q / (q.square().sum(dim=-1, keepdim=True) + _NORM_EPS).sqrt()
            k = k / (k.square().sum(dim=-1, keepdim=True) + _NORM_EPS).sqrt()
        q, k = (t.repeat_interleave(groups, dim=2) for t in (q * scale, k))
        keep = torch.exp(decay)
        outs = []
        for t in range(q.shape[1]):
            faded = keep[:, t, :, None, None] * state
            u = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, None, :] @ faded)[:, :, 0])
            new = torch.addcmul(faded, k[:, t, :, :, None], u[:, :, None, :])
            o = (q[:, t, :, None, :] @ new)[:, :, 0]
            if lengths is not None:
                alive = lengths > start + t
                new = torch.where(alive[:, None, None, None], new, state)
                o = torch.where(alive[:, None, None], o, 0)
            state = new
            outs.append(o)
        return torch.stack(outs, dim=1), state

    inputs = [wide[n] for n in ("query", "key", "value", "decay", "beta")]
    shape = (case["batch"], case["heads"], case["key_size"], case["value_size"])
    state = first.detach() if first is not None else inputs[0].new_zeros(shape)
    # Segments whose states (about five of them a token in the backward) stay within some gigabytes.
    segment = max(4, min(128, int(4e9 / (40 * math.prod(shape)))))
    starts, outs = [], []
    with torch.no_grad():
        for at in range(0, tokens, segment):
            starts.append((at, state))
            o, state = walk(state, *(t[:, at : at + segment] for t in inputs), at)
            outs.append(o)
    o, last = torch.cat(outs, dim=1), state
    if case["mode"] == "infer":
        return o, last
    grads, back = [], wide["dlast"].detach()
    for at, begin in reversed(starts):
        leaves = [begin.clone().requires_grad_()]
        leaves += [t.detach()[:, at : at + segment].clone().requires_grad_() for t in inputs]
        part, end = walk(*leaves, at)
        back, *rest = torch.autograd.grad((part, end), leaves, (wide["dy"].detach()[:, at : at + segment], back))
        grads.append(rest)
    out = [o, last, *(torch.cat(parts[::-1], dim=1) for parts in zip(*grads, strict=True))]
    if first is not None:
        out.append(back)
    return tuple(out)
