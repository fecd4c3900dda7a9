"""Rotary positions of binary32 heads: sines and cosines rounded once.

y0 = a c - b s with c and s half a step (2^-24) of themselves off, one product rounded and
the sum (a fused multiply-add): 2^-24 (|a c| + |b s| + max(|a c|, |b s|) + |y|).  The angle is
off by 4 steps of 2^-53 of itself at most (its two products, 1 / 2 pi, and the definition's
own).  y1 likewise."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (96, 64), (6, 6), (37, 34)])
@pytest.mark.parametrize("first", [0, 1000, 1000000])
@pytest.mark.parametrize("gradient", [False, True])
def test_no_more_than_the_roundings(layout, dim, rotary, first, gradient):
    from easyfhe import plain

    plan = plain.RopePlan(dim, rotary_dim=rotary, layout=layout,
                          scaling={"type": "yarn", "factor": 16.0, "original": 4096,
                                   "fast": 32.0, "slow": 1.0} if dim == 96 else None)
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn((2, 700, 6, dim), generator=g, device="cuda")
    pos = torch.arange(700, device="cuda") * 3 + first
    y = (plain.rope_grad if gradient else plain.rope)(x, positions=pos, plan=plan).double()
    angle = pos.double()[:, None] * plan.freqs
    c = (torch.cos(angle) * plan.factor)[:, None]
    s = (torch.sin(angle) * (-plan.factor if gradient else plan.factor))[:, None]
    off = (4 * 2.0 ** -53 * abs(plan.factor) * angle.abs())[:, None]
    lo, hi = (slice(0, rotary // 2), slice(rotary // 2, rotary)) if layout == "half" else \
        (slice(0, rotary, 2), slice(1, rotary, 2))
    a, b = x.double()[..., lo], x.double()[..., hi]
    for got, p, q in ((y[..., lo], a * c, -(b * s)), (y[..., hi], b * c, a * s)):
        want = p + q
        tol = 2.0 ** -24 * (p.abs() + q.abs() + torch.maximum(p.abs(), q.abs()) + want.abs())
        tol = 1.001 * tol + off * (a.abs() + b.abs()) + 2.0 ** -126
        diff = (got - want).abs()
        assert bool((diff <= tol).all()), float((diff / tol).max())
