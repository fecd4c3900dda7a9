"""64-bit definitions of the plaintext operators, for the tests."""

from __future__ import annotations

import torch


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def rope64(x, positions, freqs, factor, rotary, layout, gradient=False):
    """x [batch, seq, heads, dim], positions [batch, seq] -> (y, |x0| + |x1| of each element)."""

    f = torch.tensor(freqs, dtype=torch.float64, device=x.device)
    ang = positions.double()[..., None] * f
    c, s = torch.cos(ang)[:, :, None] * factor, torch.sin(ang)[:, :, None] * factor
    s = -s if gradient else s
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    lo, hi = (slice(0, rotary // 2), slice(rotary // 2, rotary)) if layout == "half" else \
        (slice(0, rotary, 2), slice(1, rotary, 2))
    a, b = x.double()[..., lo], x.double()[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    size[..., lo] = size[..., hi] = (a.abs() + b.abs()) * abs(factor)
    return y, size


def q4_weight64(codes, scales, zeros, group):
    idx = torch.arange(codes.shape[1], device=codes.device) // group
    z = 8.0 if zeros is None else zeros.double()[:, idx]
    return (codes.double() - z) * scales.double()[:, idx]


def loss64(hidden, weight, labels, ignore):
    """(loss, lse, logits) in binary64; NaN for labels outside the vocabulary."""

    z = hidden.double() @ weight.double().T
    lse = torch.logsumexp(z, dim=1)
    v = z.shape[1]
    bad = (labels < 0) | (labels >= v)
    own = z.gather(1, labels.clamp(0, v - 1)[:, None])[:, 0]
    loss = torch.where(bad, torch.full_like(lse, float("nan")), lse - own)
    return torch.where(labels == ignore, torch.zeros_like(loss), loss), lse, z


def loss_grad64(hidden, weight, labels, ignore, grad):
    """dz [tokens, words] in binary64, rows of ignored tokens zero."""

    _, lse, z = loss64(hidden, weight, labels, ignore)
    dz = torch.exp(z - lse[:, None])
    dz[torch.arange(z.shape[0]), labels.clamp(0, z.shape[1] - 1)] -= 1.0
    dz = dz * grad.double()[:, None]
    return torch.where((labels == ignore)[:, None], torch.zeros_like(dz), dz)
