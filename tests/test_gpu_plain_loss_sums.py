"""What the sums of the vocabulary loss's gradients keep (csrc/vocab_loss.cu), against
binary64."""

from __future__ import annotations

import pytest
import torch

from _plain import half_step, loss64, loss_grad64

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _inputs(t, v, d, dtype, ignored=0.2, seed=0, lean=12.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn((v, d), generator=g, device="cuda") / d ** 0.5).to(dtype)
    labels = torch.randint(0, v, (t,), generator=g, device="cuda")
    h = torch.randn((t, d), generator=g, device="cuda")
    h = (h + lean * torch.rand((t, 1), generator=g, device="cuda") * w[labels]).to(dtype)
    off = torch.rand((t,), generator=g, device="cuda") < ignored
    labels = torch.where(off, torch.full_like(labels, -100), labels)
    grad = torch.randn((t,), generator=g, device="cuda") / t
    return h, w, labels, grad


def _weight_gradient_is_exact_at_labels(h, w, labels, grad, dw):
    """dz is rounded by up to half a step at every word but the label, whose remainder is
    added in binary32: there only half a step squared is lost (2^-24 of it), and each token
    of a word costs its row of dW one rounding more.  A p is off by twice a logit's error e
    ((d / 16 + 2) accumulations of 2^-22 max|z|, and lse's 16 steps) and by 2^-20 for the
    exponential and its argument; a sum by a step of 2^-22 of its terms for every 16 tokens;
    the output by half a step.  Below 2^-126 nothing keeps its relative precision, in fp16
    below 2^-38 max|g| (dz under its scale) and 2^-25 (the output)."""

    t, d = h.shape
    dz = loss_grad64(h, w, labels, -100, grad)
    _, lse, z = loss64(h, w, labels, -100)
    e = (d / 16 + 2) * 2.0 ** -22 * float(z.abs().max())
    e = e + 16 * 2.0 ** -23 * lse.abs().clamp(min=1.0)
    counted = labels != -100
    g = torch.where(counted, grad.double().abs(), 0.0)[:, None]
    step = half_step(h.dtype)
    lost = torch.full_like(dz, 1.01 * step)
    lost[torch.arange(t), labels.clamp(min=0)] = 2.0 ** -24
    size = dz.abs() * (lost + 2.0 ** -20) + 2 * e[:, None] * torch.exp(z - lse[:, None]) * g
    size += 2.0 ** -126
    if h.dtype == FP:
        size += 2.0 ** -38 * float(g.max()) * counted[:, None]
    hc = torch.where(counted[:, None], h.double(), 0.0)
    want, total = dz.T @ hc, dz.abs().T @ hc.abs()
    each = torch.bincount(labels[counted], minlength=w.shape[0])[:, None]
    tol = size.T @ hc.abs() + ((t / 16 + 16) * 2.0 ** -22 + (each + 1) * 2.0 ** -24) * total
    tol = tol + 1.01 * step * want.abs() + 2.0 ** -126 + (2.0 ** -25 if h.dtype == FP else 0.0)
    diff = (dw.double() - want).abs()
    assert bool((diff <= tol).all()), float((diff / tol).max())


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,v,d", [(65, 300, 64), (130, 2000, 200), (300, 40, 72), (1100, 700, 72),
                                   (1024, 70000, 64), (1025, 255, 8), (9000, 70001, 24)])
def test_weight_gradient_keeps_the_labels_dz(dtype, t, v, d):
    from easyfhe import plain

    h, w, labels, grad = _inputs(t, v, d, dtype)
    _, lse = plain.vocab_loss(h, w, labels)
    dh, dw = plain.vocab_loss_grad(h, w, labels, lse, grad)
    _weight_gradient_is_exact_at_labels(h, w, labels, grad, dw)
    again = plain.vocab_loss_grad(h, w, labels, lse, grad, need_hidden=False)[1]
    assert torch.equal(again, dw)


@pytest.mark.parametrize("t", [70, 1000, 3000])
@pytest.mark.parametrize("which", ["one", "ends", "few", "last counted"])
def test_labels_that_many_tokens_share(t, which):
    from easyfhe import plain

    v = 777
    h, w, labels, grad = _inputs(t, v, 200, BF, lean=0.0)
    at = torch.arange(t, device="cuda")
    labels = {"one": torch.full_like(labels, 5), "ends": torch.where(at % 3 == 0, 0, v - 1),
              "few": 31 + at % 4,
              "last counted": torch.where(at == t - 1, 256, -100)}[which]
    _, lse = plain.vocab_loss(h, w, labels)
    dh, dw = plain.vocab_loss_grad(h, w, labels, lse, grad)
    _weight_gradient_is_exact_at_labels(h, w, labels, grad, dw)


def test_labels_outside_the_vocabulary_among_many():
    """A label that is no word makes every row of dW NaN (its token's dz is), and leaves the
    other tokens' rows of dh what they are without it."""
    from easyfhe import plain

    for t in (100, 2000):
        h, w, labels, grad = _inputs(t, 300, 64, BF)
        labels[7] = -100
        _, lse = plain.vocab_loss(h, w, labels)
        clean, dw = plain.vocab_loss_grad(h, w, labels, lse, grad)
        assert torch.isfinite(dw).all()
        for bad in (300, -3, 2 ** 40):
            labels[7] = bad
            _, lse = plain.vocab_loss(h, w, labels)
            dh, dw = plain.vocab_loss_grad(h, w, labels, lse, grad)
            assert torch.isnan(dw).all() and torch.isnan(dh[7]).all()
            keep = torch.arange(t, device="cuda") != 7
            assert torch.equal(dh[keep], clean[keep])


def _is_unbiased(got, want, steps):
    """The mean relative error of n values of one sign: at most `steps` steps (2^-23) of the
    sums, and what n roundings to nearest, each half a step of the type at most, leave of
    their mean: more than 6 / sqrt(n) of that once in 3e7 draws (Hoeffding's bound)."""

    n = want.numel()
    mean = float(((got.double() - want) / want).mean())
    tol = steps * 2.0 ** -23 + 6 * half_step(got.dtype) / n ** 0.5
    assert abs(mean) <= tol, (mean, tol)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_weight_gradient_of_a_million_tokens(dtype):
    """Sums of 2^20 products of one sign: a tensor core's accumulator truncates at every 16 of
    them, so one over all would lose up to 65536 steps.  At most 16384 products run in one
    accumulator here: 1024 steps, and 64 roundings where the sums are joined.  W is zero, so
    that each p is 2^-6 and each dz exact."""
    from easyfhe import plain

    t, v, d = 1 << 20, 64, 2048
    g = torch.Generator(device="cuda").manual_seed(1)
    h = torch.empty((t, d), dtype=dtype, device="cuda")
    want = torch.zeros(d, dtype=torch.float64, device="cuda")
    for part in h.split(1 << 16):
        part.copy_(torch.rand(part.shape, generator=g, device="cuda") + 0.5)
        want += part.double().sum(0)
    want /= t
    w = torch.zeros((v, d), dtype=dtype, device="cuda")
    labels = torch.full((t,), 3, device="cuda")
    _, lse = plain.vocab_loss(h, w, labels)
    _, dw = plain.vocab_loss_grad(h, w, labels, lse, torch.full((t,), 1.0 / t, device="cuda"),
                                  need_hidden=False)
    _is_unbiased(dw[0], want / 64, 1024 + 64)
    _is_unbiased(dw[3], want * (-63 / 64), 1024 + 64)
    assert torch.equal(dw[0], dw[63])


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,d", [(120, 4096), (200, 4096), (250, 8192)])
def test_hidden_gradient_over_half_a_million_words(dtype, t, d):
    """As above, over the words: hidden states of zero, so that each p is 2^-19, and a label
    whose word is zero.  Up to 1024 steps in one accumulator, and 32 joined."""
    from easyfhe import plain

    v = 1 << 19
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.empty((v, d), dtype=dtype, device="cuda")
    want = torch.zeros(d, dtype=torch.float64, device="cuda")
    for part in w.split(1 << 15):
        part.copy_(torch.rand(part.shape, generator=g, device="cuda") + 0.5)
    w[5] = 0.0
    for part in w.split(1 << 15):
        want += part.double().sum(0)
    h = torch.zeros((t, d), dtype=dtype, device="cuda")
    labels = torch.full((t,), 5, device="cuda")
    _, lse = plain.vocab_loss(h, w, labels)
    dh, _ = plain.vocab_loss_grad(h, w, labels, lse, torch.ones(t, device="cuda"),
                                  need_weight=False)
    _is_unbiased(dh[0], want / v, 1024 + 32)
    _is_unbiased(dh[t - 1], want / v, 1024 + 32)


@pytest.mark.parametrize("t", [9, 64, 100, 300, 1100])
def test_no_upstream_gradient_no_gradient(t):
    """A token whose finite operands overflow its logits, under an upstream gradient of zero:
    its rows are zero and the others' what they are beside a harmless token."""
    from easyfhe import plain

    h, w, labels, grad = _inputs(t, 400, 64, BF, ignored=0.0)
    grad[2] = 0.0
    _, lse = plain.vocab_loss(h, w, labels)
    want = plain.vocab_loss_grad(h, w, labels, lse, grad)
    assert not want[0][2].any()
    h[2] = 3e38
    _, lse = plain.vocab_loss(h, w, labels)
    assert not torch.isfinite(lse[2])
    got = plain.vocab_loss_grad(h, w, labels, lse, grad)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [BF, FP])
def test_labels_among_more_than_2_to_24_words(dtype):
    """Four passes of the labels' sort.  dW at the labels and some other words, from the lse
    that the loss returned: p is off by that one's own rounding (2^-23 of about 17) besides."""
    from easyfhe import plain

    t, v, d = 1100, (1 << 24) + 77, 8
    g = torch.Generator(device="cuda").manual_seed(4)
    w = torch.empty((v, d), dtype=dtype, device="cuda")
    for part in w.split(1 << 20):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") / d ** 0.5)
    h = torch.randn((t, d), generator=g, device="cuda").to(dtype)
    labels = torch.randint(0, v, (t,), generator=g, device="cuda")
    labels[:6] = torch.tensor([0, v - 1, 1 << 24, (1 << 24) - 1, v - 1, 255], device="cuda")
    labels[::9] = -100
    grad = torch.randn((t,), generator=g, device="cuda") / t
    _, lse = plain.vocab_loss(h, w, labels)
    _, dw = plain.vocab_loss_grad(h, w, labels, lse, grad, need_hidden=False)
    counted = labels != -100
    words = torch.cat([labels[counted], torch.randint(0, v, (500,), generator=g, device="cuda"),
                       torch.arange(v - 300, v, device="cuda")]).unique()
    z = h.double() @ w[words].double().T
    dz = torch.exp(z - lse.double()[:, None]) - (labels[:, None] == words[None, :]).double()
    gc = torch.where(counted, grad.double(), 0.0)[:, None]
    dz, step = dz * gc, half_step(dtype)
    hit = labels[:, None] == words[None, :]
    lost = torch.where(hit, 2.0 ** -24, 1.01 * step)
    e = (d / 16 + 2) * 2.0 ** -22 * float(z.abs().max()) + 2.0 ** -18
    size = dz.abs() * (lost + 2.0 ** -20) + 2 * e * torch.exp(z - lse.double()[:, None]) * gc.abs()
    size += 2.0 ** -126
    if dtype == FP:
        size += 2.0 ** -38 * float(gc.abs().max()) * counted[:, None]
    want, total = dz.T @ h.double(), dz.abs().T @ h.double().abs()
    tol = size.T @ h.double().abs() + (t / 16 + 16) * 2.0 ** -22 * total + 1.01 * step * want.abs()
    tol = tol + 2.0 ** -126 + (2.0 ** -25 if dtype == FP else 0.0)
    diff = (dw[words].double() - want).abs()
    assert bool((diff <= tol).all()), float((diff / tol).max())


@pytest.mark.parametrize("t", [100, 900, 3000])
def test_a_captured_step_follows_its_labels(t):
    """The order of the labels is found again at every replay."""
    from easyfhe import plain

    h, w, labels, grad = _inputs(t, 1200, 64, BF)

    def step():
        loss, lse = plain.vocab_loss(h, w, labels)
        return (loss, *plain.vocab_loss_grad(h, w, labels, lse, grad))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed, ignored in ((1, 0.9), (2, 0.0), (3, 1.0), (4, 0.3)):
        for dst, src in zip((h, w, labels, grad), _inputs(t, 1200, 64, BF, ignored, seed)):
            dst.copy_(src)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), seed
