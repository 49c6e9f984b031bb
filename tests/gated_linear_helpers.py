"""The gated linear layer's 64-bit definition with bounds on what the kernels may be off, as in
sequence_helpers."""

import torch

from sequence_helpers import EPS32, ROUND, TINY, activation_reference


def gated_activation(z, kind):
    """act(z) and act'(z) in float64."""
    if kind != "silu":
        return activation_reference(z, kind)
    s = torch.sigmoid(z)
    return z * s, s + z * s * torch.sigmoid(-z)


def gated_reference(x, w, b, kind, dy=None):
    """{name: (value, noise)} of y and, with dy, dx, dw, db in float64 (on the CPU).

    Sums of n products in any order: n roundings of the magnitudes' sum. The activations vary by at most
    1.13 of their argument's error, their slopes by 1.2 (of relu's, either side of the step where z is within
    its error of zero); their own evaluation adds 16 roundings of |z| + 1. Products of two such values: each
    one's error times the other. Beside 16-bit types the factors kept for the backward have 16 significant bits
    (half a step: 2^-16), and dz is rounded to the element type.
    """
    dtype = x.dtype
    f = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    x, w, b = f(x).reshape(-1, x.shape[-1]), f(w), f(b)
    z = x @ w.T
    size = x.abs() @ w.abs().T
    if b is not None:
        z, size = z + b, size + b.abs()
    noise = EPS32 * (x.shape[1] + 8) * size
    gate, up = z.chunk(2, 1)
    gate_noise, up_noise = noise.chunk(2, 1)
    act, slope = gated_activation(gate, kind)
    act_noise = 1.13 * gate_noise + 16 * EPS32 * (gate.abs() + 1)
    if kind == "relu":
        act_noise = gate_noise
    times = lambda p, q, dp, dq: dp * q.abs() + p.abs() * dq + dp * dq + EPS32 * (p * q).abs()  # noqa: E731
    out = {"y": (act * up, times(act, up, act_noise, up_noise))}
    if dy is None:
        return out
    g = f(dy).reshape(act.shape)
    slope_noise = 1.2 * gate_noise + 16 * EPS32 * (gate.abs() + 1)
    if kind == "relu":
        slope_noise = (gate.abs() <= gate_noise).double()
    keep = 0 if dtype == torch.float32 else 2.0**-16
    halves, noises = [], []
    for value, error in ((up * slope, times(up, slope, up_noise, slope_noise)), (act, act_noise)):
        error = error + keep * (value.abs() + error)
        dz = g * value
        error = g.abs() * error + EPS32 * dz.abs()
        halves.append(dz)
        noises.append(error + ROUND[dtype] * (dz.abs() + error) + TINY[dtype])
    dz, dz_noise = torch.cat(halves, 1), torch.cat(noises, 1)
    dz_size = dz.abs() + dz_noise
    rows, outputs = dz.shape
    out["dx"] = (dz @ w, dz_noise @ w.abs() + EPS32 * (outputs + 8) * (dz_size @ w.abs()))
    out["dw"] = (dz.T @ x, dz_noise.T @ x.abs() + EPS32 * (rows + 8) * (dz_size.T @ x.abs()))
    out["db"] = (dz.sum(0), dz_noise.sum(0) + EPS32 * (rows + 8) * dz_size.sum(0))
    return out
