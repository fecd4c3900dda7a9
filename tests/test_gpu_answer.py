"""The plaintext operators together, as a client uses them: a plain decoder
layer on the GPU (rotary positions), the head's score with its gradient
(vocabulary cross entropy) and the next token (4-bit head)."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

import llama3_layer
from _plain import loss64, loss_grad64, q4_weight64

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, HIDDEN, INNER = 8, 2, 16, 128, 256
GEOMETRY = {"query_heads": HEADS, "kv_heads": KV, "head_dim": DIM}


def _layer(seed=0):
    rng = np.random.default_rng(seed)
    draw = lambda *s: (rng.standard_normal(s) * 0.2).astype(np.float32)  # noqa: E731
    return SimpleNamespace(
        input_layernorm=1 + 0.1 * rng.standard_normal(HIDDEN),
        post_attention_layernorm=1 + 0.1 * rng.standard_normal(HIDDEN),
        q_proj=draw(HEADS * DIM, HIDDEN), k_proj=draw(KV * DIM, HIDDEN),
        v_proj=draw(KV * DIM, HIDDEN), o_proj=draw(HIDDEN, HEADS * DIM),
        gate_proj=draw(INNER, HIDDEN), up_proj=draw(INNER, HIDDEN),
        down_proj=draw(HIDDEN, INNER))


def _fits():
    x = np.cos(np.pi * (np.arange(24) + 0.5) / 24)

    def fit(f, lo, hi):
        c = np.polynomial.chebyshev.chebfit(x, f((lo + hi) / 2 + (hi - lo) / 2 * x), 20)
        c[0] *= 2
        return {"fit_interval": [lo, hi], "coefficients": c.tolist()}

    norm = fit(lambda t: 1 / np.sqrt(t + 1e-5), 0.3, 40.0)
    return SimpleNamespace(input_norm=norm, post_attention_norm=norm,
                           silu=fit(lambda t: t / (1 + np.exp(-t)), -12.0, 12.0))


@pytest.mark.parametrize("seq", [1, 5, 128])
@pytest.mark.parametrize("poly", [False, True])
def test_layer_on_the_gpu_is_the_numpy_layer(seq, poly):
    """Both in binary64 on the same formulas: sums in another order, 1e-12 of the
    largest value (a few thousand roundings of 1.1e-16)."""

    rng = np.random.default_rng(seq)
    x, w = rng.standard_normal((seq, HIDDEN)), _layer()
    ap = _fits() if poly else None
    want = llama3_layer.layer_fp64(x, w, approximations=ap, **GEOMETRY)
    got = llama3_layer.layer_fp64(x, w, approximations=ap, device="cuda", **GEOMETRY)
    assert got.dtype == np.float64 and got.shape == want.shape
    assert np.max(np.abs(got - want)) < 1e-12 * np.max(np.abs(want))


def _head(words=700):
    rng = np.random.default_rng(3)
    w = rng.standard_normal((words, HIDDEN)).astype(np.float32) / HIDDEN ** 0.5
    return llama3_layer.ClientHead(1 + 0.1 * rng.standard_normal(HIDDEN), w), w


def test_score_gradient_and_next_token_of_a_prompt():
    head, _ = _head()
    rng = np.random.default_rng(4)
    x, w = rng.standard_normal((40, HIDDEN)), _layer()
    hidden = llama3_layer.layer_fp64(x, w, device="cuda", **GEOMETRY)
    tokens = rng.integers(0, 700, 40)
    # the score on the operands that the head uses (bf16): the loss test's bound on a logit
    h = head.norm(hidden).to(torch.bfloat16)
    labels = head.labels(tokens)
    loss, lse, z = loss64(h, head.weight, labels, -100)
    tol = (HIDDEN / 16 + 2) * 2.0 ** -22 * float(z.abs().max()) + 2.0 ** -19 * float(lse.max())
    want = float(loss.sum() / 39)
    assert abs(head.score(hidden, tokens) - want) <= 2 * tol
    score, dh, dw = head.gradient(hidden, tokens)
    assert abs(score - want) <= 2 * tol
    dz = loss_grad64(h, head.weight, labels, -100, torch.full((40,), 1 / 39, device="cuda"))
    for got, full, size in ((dh, dz @ head.weight.double(), dz.abs() @ head.weight.double().abs()),
                            (dw, dz.T @ h.double(), dz.abs().T @ h.double().abs())):
        # dz and the result are rounded to bf16 (2^-8 each), p is off by twice a logit's bound
        assert bool(((got.double() - full).abs() <= (2.1 * 2.0 ** -8 + 8 * tol) * size).all())
    assert not dh[-1].any()  # the last position predicts nothing
    # the next token: the 4-bit head's own logits in binary64
    from easyfhe import plain

    w64 = q4_weight64(*plain.q4_codes(head.weight), 128)
    row = head.norm(hidden[-1:]).float()
    want = (row.double() @ w64.T)[0]
    logits = head.next_logits(hidden)
    assert float((logits - want).abs().max()) < 1e-4 * float(want.abs().max())
    top = torch.topk(want, 2).values
    assert float(top[0] - top[1]) < 1e-4 or head.next_token(hidden) == int(want.argmax())


def test_answer_check_sees_the_error():
    """No error, no change; a small one moves the score by its first-order change:
    what is left is second order in the error (1e-3 of a unit hidden state) and
    the bf16 rounding of both normed states, 2^-8 of each term."""

    head, _ = _head()
    rng = np.random.default_rng(6)
    plain_hidden = rng.standard_normal((30, HIDDEN))
    tokens = rng.integers(0, 700, 30)
    same = llama3_layer.answer_check(plain_hidden, plain_hidden, head, tokens)
    assert same["nll_decoded"] == same["nll_plain"] and same["nll_change_first_order"] == 0.0
    assert same["logits_max_abs"] == 0.0
    assert same["next_token_decoded"] == same["next_token_plain"]
    error = 0.05 * rng.standard_normal(plain_hidden.shape)
    moved = llama3_layer.answer_check(plain_hidden + error, plain_hidden, head, tokens)
    # the same in binary64, without any rounding to bf16
    w = head.weight.double()
    labels = head.labels(tokens)

    def nll(h):
        return float(loss64(head.norm(h), w, labels, -100)[0].sum() / 29)

    change = nll(plain_hidden + error) - nll(plain_hidden)
    _, dh, _ = head.gradient(plain_hidden, tokens, need_weight=False)
    delta = (head.norm(plain_hidden + error) - head.norm(plain_hidden)).abs()
    # second order: p (1 - p) <= 1/4 of the squared change of a logit, |dlogit| <= |delta| |w|
    second = float(((delta @ w.abs().T).amax(1) ** 2).mean()) / 2
    rounding = float((dh.double().abs() * delta).sum()) * 2.0 ** -7
    assert abs(moved["nll_change_first_order"] - change) <= second + rounding + 1e-3
    assert moved["logits_max_abs"] > 0


def test_training_the_head_on_decrypted_states_runs():
    head, w0 = _head()
    rng = np.random.default_rng(8)
    hidden, tokens = rng.standard_normal((64, HIDDEN)), rng.integers(0, 700, 64)
    before = head.weight.clone()
    _, _, dw = head.gradient(hidden, tokens)
    logits = head.next_logits(hidden)
    head.weight -= 0.5 * dw
    assert torch.equal(head.next_logits(hidden), logits)  # the 4-bit head as it was
    head.quantize()
    assert not torch.equal(head.next_logits(hidden), logits)
    assert torch.isfinite(head.weight).all() and not torch.equal(head.weight, before)
    score, dh, dw = head.gradient(hidden, tokens)
    assert np.isfinite(score) and torch.isfinite(dh).all() and torch.isfinite(dw).all()


def test_refusals():
    with pytest.raises(ValueError):
        llama3_layer.ClientHead(np.ones(64), np.zeros((10, 128), np.float32))


def test_synthetic_head():
    head = llama3_layer.synthetic_head(words=1000, hidden=256)
    again = llama3_layer.synthetic_head(words=1000, hidden=256)
    assert torch.equal(head.weight, again.weight) and head.four_bit.shape == (1000, 256)
