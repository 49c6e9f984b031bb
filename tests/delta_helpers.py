"""The gated delta rule's 64-bit definition, token by token, and how far the kernels may be from it.

Tolerances are relative to the size of a row (a token's head) plus the rows' mean square over the head,
since a row is a sum of terms of that size, plus the size of what a row is a small difference of (the part
across a normalised q or k; the state's product with its gradient, which is a decay's), and count
roundings, each at most ROUND of what is rounded:

* a result's own rounding: 1;
* float32 arithmetic: a sum of n products n of 2^-24, over the key size, the value size and the tokens of
  two chunks, and 32 operations besides (the triangular solve, exp, lengths); the terms of a sum are taken
  at up to four times its size;
* two-term operands (16 bits): two roundings leave ROUND^2 (and 2^-24) of a value; five products follow each
  other from a state to the next and a token's influence fades or is kept, not multiplied: 8 of them,
  again at four times the size;
* gradients of q, k, decay and beta take states, their gradients, the tokens' updates (two of them) and the
  pairs as one term: 5 roundings besides their own, of terms up to twice their sum.
"""

import torch

from sequence_helpers import ROUND


def delta_reference(q, k, v, decay, beta, first=None, lengths=None, scale=None, normalize=False, dy=None, dlast=None):
    """{name: value} of o, last and, with dy, every gradient, in float64 on the CPU, and under "terms" the
    size of what a gradient is the difference or the product of, where that may be larger than itself."""
    f = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    q, k, v, decay, beta, first, dy, dlast = (f(t) for t in (q, k, v, decay, beta, first, dy, dlast))
    batch, tokens, key_heads, key_size = q.shape
    heads, value_size = v.shape[2:]
    live = torch.ones(batch, tokens, dtype=torch.bool)
    if lengths is not None:
        live = torch.arange(tokens) < lengths.cpu()[:, None]
        q, k, v = (torch.where(live[..., None, None], t, 0) for t in (q, k, v))
        decay, beta = (torch.where(live[..., None], t, 0) for t in (decay, beta))
        if dy is not None:
            dy = torch.where(live[..., None, None], dy, 0)
    scale = key_size**-0.5 if scale is None else scale
    nq = nk = torch.ones(batch, tokens, key_heads, 1, dtype=torch.float64)
    if normalize:
        nq, nk = (1 / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
    share = lambda t: t.repeat_interleave(heads // key_heads, 2)  # noqa: E731
    qn, kn = share(q * nq), share(k * nk)
    keep = torch.where(decay < -104, 0, decay.exp())
    outer = lambda x, y: x[..., :, None] * y[..., None, :]  # noqa: E731
    state = torch.zeros(batch, heads, key_size, value_size, dtype=torch.float64) if first is None else first
    size, states, outputs = state.abs(), [], []
    for t in range(tokens):
        faded = keep[:, t, :, None, None] * state
        r = v[:, t] - (kn[:, t, :, None, :] @ faded)[:, :, 0]
        u = beta[:, t, :, None] * r
        states.append((state, size, r, u))
        state = faded + outer(kn[:, t], u)
        size = keep[:, t, :, None, None] * size + outer(kn[:, t], u).abs()
        outputs.append(scale * (qn[:, t, :, None, :] @ state)[:, :, 0])
    o = torch.stack(outputs, 1) if outputs else torch.zeros_like(v)
    out = {"o": torch.where(live[..., None, None], o, 0), "last": state}
    if dy is None:
        return out
    d = torch.zeros_like(state) if dlast is None else dlast
    dsize, after = d.abs(), state
    parts = {name: [None] * tokens for name in ("dq", "dk", "dv", "ddecay", "dbeta", "decay_terms")}
    for t in reversed(range(tokens)):
        before, size, r, u = states[t]
        a = keep[:, t, :, None, None]
        parts["dq"][t] = scale * (after @ dy[:, t, :, :, None])[..., 0]
        d = d + scale * outer(qn[:, t], dy[:, t])
        dsize = dsize + scale * outer(qn[:, t], dy[:, t]).abs()
        du = (kn[:, t, :, None, :] @ d)[:, :, 0]
        dr = beta[:, t, :, None] * du
        parts["dv"][t], parts["dbeta"][t] = dr, (du * r).sum(-1)
        parts["dk"][t] = (d @ u[..., None])[..., 0] - a[..., 0] * (before @ dr[..., None])[..., 0]
        d, dsize = d - outer(kn[:, t], dr), dsize + outer(kn[:, t], dr).abs()
        parts["ddecay"][t] = (a * d * before).sum((-1, -2))
        # Operands of the products it sums are rounded apart from each other: as squares.
        parts["decay_terms"][t] = (a * dsize * size).square().sum((-1, -2)).sqrt()
        d, dsize, after = a * d, a * dsize, before
    stack = lambda name, like: torch.stack(parts[name], 1) if tokens else torch.zeros_like(like)  # noqa: E731
    group = lambda t: t.unflatten(2, (key_heads, -1)).sum(3)  # noqa: E731
    dq, dk = (group(stack(name, share(q))) for name in ("dq", "dk"))
    out["terms"] = {"dq": (nq * dq).norm(dim=-1), "dk": (nk * dk).norm(dim=-1)}
    if normalize:
        dq, dk = (n * (g - n * n * x * (x * g).sum(-1, keepdim=True)) for n, g, x in ((nq, dq, q), (nk, dk, k)))
    dead = lambda t: torch.where(live.reshape(batch, tokens, *[1] * (t.dim() - 2)), t, 0)  # noqa: E731
    out.update(dq=dead(dq), dk=dead(dk), dv=stack("dv", v), dfirst=d)
    out.update(ddecay=dead(stack("ddecay", decay)), dbeta=dead(stack("dbeta", beta)))
    out["terms"]["ddecay"] = stack("decay_terms", decay)
    return out


def tolerance(name, dtype, key_size, value_size):
    arithmetic = 4 * (key_size + value_size + 160) * 2.0**-24
    if dtype != torch.float32:
        arithmetic += 4 * 8 * (ROUND[dtype] ** 2 + 2.0**-24)
    if name in ("last", "dfirst"):
        return arithmetic
    if name in ("o", "dv") or dtype == torch.float32:
        return ROUND[dtype] + arithmetic
    return ROUND[dtype] * (1 + 2 * 5) + arithmetic


def assert_rows(name, actual, reference, dtype, sizes):
    """Every row of a result within its tolerance: the last axis of o, dq, dk, dv; a value of ddecay, dbeta; a
    key's row of last and dfirst. ``sizes``: of a key and of a value."""
    expected = reference[name]
    assert actual.shape == expected.shape, f"{name}: {tuple(actual.shape)} != {tuple(expected.shape)}"
    if expected.numel() == 0:
        return
    a = actual.detach().double().cpu()
    assert torch.isfinite(a).all(), f"{name}: non-finite values"
    if name in ("last", "dfirst"):
        a, expected = a.transpose(1, 2), expected.transpose(1, 2)  # [batch, key, heads, value]
    if name in ("ddecay", "dbeta"):
        a, expected = a[..., None], expected[..., None]
    size = expected.norm(dim=-1)
    size = size + size.square().mean(1, keepdim=True).sqrt()  # over the tokens (keys) of a head
    size = size + reference.get("terms", {}).get(name, 0)
    rel = ((a - expected).norm(dim=-1) / (size + 1e-30)).max().item()
    tol = tolerance(name, dtype, *sizes)
    assert rel <= tol, f"{name}: off by {rel:.3g} of its size, {tol:.3g} allowed"


def make_delta(batch, tokens, key_heads, heads, key_size, value_size, dtype, seed=0, gates=torch.float32, normalize=False):
    """Inputs and cotangents on the CPU: q, k, v, decay, beta, first, dy, dlast."""
    g = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q = randn(batch, tokens, key_heads, key_size)
    k = randn(batch, tokens, key_heads, key_size) + 0.5 * randn(1, 1, key_heads, key_size)
    if not normalize:
        k = k / (1.25 * key_size) ** 0.5
    v = randn(batch, tokens, heads, value_size)
    decay = -torch.rand(batch, tokens, heads, generator=g) * torch.exp(torch.linspace(-6, 0, heads))
    beta = torch.sigmoid(randn(batch, tokens, heads))
    first = 0.3 * randn(batch, heads, key_size, value_size)
    dy = randn(batch, tokens, heads, value_size)
    dlast = 0.1 * randn(batch, heads, key_size, value_size)
    return q.to(dtype), k.to(dtype), v.to(dtype), decay.to(gates), beta.to(gates), first, dy.to(dtype), dlast
