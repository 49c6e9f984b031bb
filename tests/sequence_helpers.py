"""64-bit definitions of the sequence operators with bounds on what float32 arithmetic may be off.

Every bound is ROUND[dtype] * |value| for the one rounding of the result, plus a running bound of
the float32 operations before it: each operation's relative error is at most 2^-24 of its operands'
magnitudes, and the constants count the operations on a value's way (a sum of n terms in any order:
n of them; sigmoid through exp2 and a reciprocal: |gate| + 8).
"""

import torch

EPS32 = 2.0**-24
ROUND = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
# Smallest spacing of a type's values (results near zero round to multiples of it).
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}


def assert_within(actual, expected, noise, what=""):
    """|actual - expected| <= half a spacing of the type + the bound on the arithmetic."""
    dtype = actual.dtype
    a = actual.detach().double().cpu()
    e = expected.detach().double().cpu()
    n = noise.detach().double().cpu() if isinstance(noise, torch.Tensor) else noise
    assert a.shape == e.shape, f"{what}: shape {tuple(a.shape)} != {tuple(e.shape)}"
    if e.numel() == 0:
        return
    assert torch.isfinite(a).all(), f"{what}: non-finite values"
    bound = ROUND[dtype] * (e.abs() + n) + n + TINY[dtype]
    excess = (a - e).abs() - bound
    worst = excess.argmax()
    assert excess.max() <= 0, (
        f"{what}: {a.flatten()[worst].item():.9g} is not {e.flatten()[worst].item():.9g} within "
        f"{(bound.flatten()[worst] if bound.numel() > 1 else bound).item():.3g}"
    )


def norm_reference(x, w, b, eps, dy=None):
    """{name: (value, noise)} of y and, with dy, dx, dw, db in float64 (on the CPU)."""
    x = x.detach().double().cpu().reshape(-1, x.shape[-1])
    rows, c = x.shape
    w64 = torch.ones(c, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b64 = torch.zeros(c, dtype=torch.float64) if b is None else b.detach().double().cpu()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    hat = (x - mean) * rstd
    # The mean's sum: the terms a thread adds in turn (at most 40, or c / 1024 past 1024 threads'
    # registers), and the levels of the tree over the threads.
    depth = 40 + 16 + c / 1024
    hat_noise = EPS32 * depth * (rstd * x.abs().amax(1, keepdim=True) + 4 * hat.abs())
    out = {"y": (hat * w64 + b64, hat_noise * w64.abs() + 4 * EPS32 * ((hat * w64).abs() + b64.abs()))}
    if dy is not None:
        g = dy.detach().double().cpu().reshape(-1, c)
        wg = g * w64
        c1, c2 = wg.mean(1, keepdim=True), (wg * hat).mean(1, keepdim=True)
        dx = rstd * (wg - c1 - hat * c2)
        size = wg.abs().amax(1, keepdim=True)
        big = hat.abs().amax(1, keepdim=True)
        dx_noise = rstd * (EPS32 * depth * size * (4 + 4 * big * big) + 4 * hat_noise.amax(1, keepdim=True) * size * (1 + big))
        n = rows + 64
        out["dx"] = (dx, dx_noise)
        out["dw"] = ((g * hat).sum(0), (n * EPS32 * (g * hat).abs() + g.abs() * hat_noise).sum(0))
        out["db"] = (g.sum(0), n * EPS32 * g.abs().sum(0))
    return out


def recurrence_reference(x, gate, first=None, lengths=None, dy=None, dlast=None):
    """{name: (value, noise)} of h, last and, with dy, dx, dgate, dfirst in float64 (on the CPU)."""
    x, g = x.detach().double().cpu(), gate.detach().double().cpu()
    batch, tokens, c = x.shape
    h = torch.zeros(batch, c, dtype=torch.float64) if first is None else first.detach().double().cpu()
    n = None if lengths is None else lengths.cpu().clamp(0, tokens)
    live = torch.ones(batch, tokens, 1, dtype=torch.bool)
    if n is not None:
        live = (torch.arange(tokens) < n[:, None])[..., None]
    keep = torch.where(live, torch.sigmoid(g), 1)
    take = torch.where(live, torch.sigmoid(-g), 0)
    x = torch.where(live, x, 0)
    finite = torch.where(torch.isfinite(g) & live, g, 0)
    unit = EPS32 * (8 + finite.abs())  # of sigmoid and of the two operations with it
    hs, noises, before = [], [], []
    e = torch.zeros_like(h)
    for t in range(tokens):
        before.append((h, e))
        new = keep[:, t] * h + take[:, t] * x[:, t]
        e = keep[:, t] * e + 2 * unit[:, t] * (keep[:, t] * h.abs() + take[:, t] * x[:, t].abs())
        h = new
        hs.append(h)
        noises.append(e)
    out = {"last": (h, e)}
    stack = lambda parts: torch.stack(parts, 1) if parts else torch.zeros(batch, 0, c, dtype=torch.float64)  # noqa: E731
    out["h"] = (torch.where(live, stack(hs), 0), torch.where(live, stack(noises), 0))
    if dy is None:
        return out
    d = torch.where(live, dy.detach().double().cpu(), 0)
    back = torch.zeros(batch, c, dtype=torch.float64) if dlast is None else dlast.detach().double().cpu()
    size = back.abs()  # the same sums with every term's magnitude: what rounding is relative to
    noise = torch.zeros_like(back)
    dx, dg = [None] * tokens, [None] * tokens
    for t in reversed(range(tokens)):
        (hp, he), u = before[t], unit[:, t]
        total, tsize, tnoise = back + d[:, t], size + d[:, t].abs(), noise
        tnoise = tnoise + 2 * EPS32 * tsize
        slope = keep[:, t] * take[:, t]
        spread = hp.abs() + x[:, t].abs()
        dx[t] = (take[:, t] * total, take[:, t] * (tnoise + 2 * u * tsize))
        dg[t] = (
            total * (hp - x[:, t]) * slope,
            slope * (tnoise * spread + tsize * he + 4 * u * tsize * spread),
        )
        back, size = keep[:, t] * total, keep[:, t] * tsize
        noise = keep[:, t] * (tnoise + 2 * u * tsize)
    for name, parts in (("dx", dx), ("dgate", dg)):
        out[name] = tuple(torch.where(live, stack([p[i] for p in parts]), 0) for i in range(2))
    out["dfirst"] = (back, noise)
    return out


def activation_reference(z, kind):
    """act(z) and act'(z) in float64."""
    if kind is None:
        return z, torch.ones_like(z)
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double()
    if kind == "gelu":
        phi = 0.5 * (1 + torch.erf(z / 2**0.5))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5
    c = (2 / torch.pi) ** 0.5
    t = torch.tanh(c * (z + 0.044715 * z**3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def linear_reference(x, w, b, residual, kind, dy=None):
    """{name: (value, noise)} of y and, with dy, dx, dw, db in float64 (on the CPU).

    Sums of n products in any order: n roundings of the magnitudes' sum. The activations and their
    slopes vary by at most 1.13 of their argument's error (1.2 for a slope); their own evaluation
    adds 16 roundings of |z| + 1. Beside 16-bit values the slope is kept in steps of 1 / 28672, dz is
    rounded to the element type, and relu's slope may be either side of the step where z is within its
    error of zero.
    """
    dtype = x.dtype
    f = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    x, w, b, r = f(x).reshape(-1, x.shape[-1]), f(w), f(b), f(residual)
    z = x @ w.T
    size = x.abs() @ w.abs().T
    if b is not None:
        z, size = z + b, size + b.abs()
    z_noise = EPS32 * (x.shape[1] + 8) * size
    y, slope = activation_reference(z, kind)
    y_noise = z_noise
    if kind is not None:
        y_noise = 1.13 * z_noise + 16 * EPS32 * (z.abs() + 1)
    if r is not None:
        r = r.reshape(y.shape)
        y_noise = y_noise + 2 * EPS32 * (y.abs() + r.abs())
        y = y + r
    out = {"y": (y, y_noise)}
    if dy is None:
        return out
    g = f(dy).reshape(y.shape)
    dz = g * slope
    if kind is None:
        dz_noise = torch.zeros_like(dz)
    else:
        slope_noise = 1.2 * z_noise + 16 * EPS32 * (z.abs() + 1)
        if kind == "relu":
            slope_noise = (z.abs() <= z_noise).double()
        elif dtype != torch.float32:
            slope_noise = slope_noise + 0.5 / 28672
        dz_noise = g.abs() * slope_noise
        dz_noise = dz_noise + ROUND[dtype] * (dz.abs() + dz_noise) + TINY[dtype]
    dz_size = dz.abs() + dz_noise
    rows, outputs = dz.shape
    out["dx"] = (dz @ w, dz_noise @ w.abs() + EPS32 * (outputs + 8) * (dz_size @ w.abs()))
    out["dw"] = (dz.T @ x, dz_noise.T @ x.abs() + EPS32 * (rows + 8) * (dz_size.T @ x.abs()))
    out["db"] = (dz.sum(0), dz_noise.sum(0) + EPS32 * (rows + 8) * dz_size.sum(0))
    return out
