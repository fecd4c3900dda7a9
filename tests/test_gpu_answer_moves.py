"""answer_check on states that are moved along the score's gradient, by enough that its
first-order change is far above what rounding and curvature leave."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import llama3_layer
from _plain import loss64, loss_grad64

pytestmark = pytest.mark.gpu

HIDDEN, WORDS, TOKENS = 128, 700, 30


@pytest.mark.parametrize("towards", [-1.0, 1.0])
def test_first_order_change_and_scores(towards):
    """States whose normed form moves by half a unit against (along) the gradient.

    The first-order change is the sum of error times gradient: the gradient of the states as
    the head takes them (rounded to bf16), itself rounded to bf16 (2^-8 of each term, and
    2^-12 for all else).  The scores are of states rounded to bf16: a logit is off by 2^-8 of
    sum |h w| at most, a loss by twice that, a change of the score by that of both states."""

    rng = np.random.default_rng(21)
    w32 = rng.standard_normal((WORDS, HIDDEN)).astype(np.float32) / HIDDEN ** 0.5
    head = llama3_layer.ClientHead(1 + 0.1 * rng.standard_normal(HIDDEN), w32)
    reference = rng.standard_normal((TOKENS, HIDDEN))
    tokens = rng.integers(0, WORDS, TOKENS)
    w, labels = head.weight.double(), head.labels(tokens)
    each = torch.full((TOKENS,), 1.0 / (TOKENS - 1), device="cuda", dtype=torch.float64)

    def nll(states):
        return float((loss64(states, w, labels, -100)[0] * each).sum())

    def gradient(states):
        return loss_grad64(states, w, labels, -100, each) @ w

    plain = head.norm(reference)
    g = gradient(plain)
    step = 0.5 * g / g.norm(dim=1, keepdim=True).clamp(min=1e-30)
    decoded = ((plain + towards * step) / head.gamma).cpu().numpy()
    error = head.norm(decoded) - plain
    got = llama3_layer.answer_check(decoded, reference, head, tokens)

    terms = error * gradient(plain.to(torch.bfloat16).double())
    first = float(terms.sum())
    tol = (2.0 ** -8 + 2.0 ** -12) * float(terms.abs().sum())
    assert abs(got["nll_change_first_order"] - first) <= tol < 0.02 * abs(first)

    change = nll(plain + error) - nll(plain)
    assert towards * change > 0.2 and abs(first - change) <= 0.1 * abs(change)

    rounding = [2 * 2.0 ** -8 * (s.abs() @ w.abs().T).amax(1) for s in (plain, plain + error)]
    rounding = [float((r * each)[labels != -100].sum()) for r in rounding]
    assert abs(got["nll_plain"] - nll(plain)) <= rounding[0]
    assert abs(got["nll_decoded"] - nll(plain + error)) <= rounding[1]
    assert abs(got["nll_decoded"] - got["nll_plain"] - change) <= sum(rounding) < 0.5 * abs(change)
