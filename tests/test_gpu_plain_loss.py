"""Cross entropy over the vocabulary (csrc/vocab_loss.cu) against binary64.

Tolerances.  A logit is a binary32 sum of D / 16 accumulations, each off by at
most a step (2^-23) of a partial sum; partial sums of these inputs stay below
twice the largest logit: e = (D / 16 + 2) 2^-22 max|z| in all.  lse is off by e
and the binary32 of the maximum, the exponentials and the logarithm: 16 steps
of 2^-23 of max(1, |lse|) covers those.  A dz is g (p - [label]) with p off by
2 (e + that) relative, rounded to the operand type (half a step, and for fp16
half a step of its subnormals under the power-of-two scale: 2^-38 max|g|); the
gradients' sums add their accumulations' steps and the output's half step.
Below 2^-126 bf16 and binary32 lose their relative precision (a value there is
rounded to a multiple of 2^-133 or taken as zero), so every dz and every output
may be off by 2^-126 besides: a word of probability e^-88 has such a dz."""

from __future__ import annotations

import pytest
import torch

from _plain import half_step, loss64, loss_grad64

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _inputs(t, v, d, dtype, ignored=0.3, seed=0, lean=12.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn((v, d), generator=g, device="cuda") / d ** 0.5).to(dtype)
    labels = torch.randint(0, v, (t,), generator=g, device="cuda")
    h = torch.randn((t, d), generator=g, device="cuda")
    h = (h + lean * torch.rand((t, 1), generator=g, device="cuda") * w[labels]).to(dtype)
    off = torch.rand((t,), generator=g, device="cuda") < ignored
    labels = torch.where(off, torch.full_like(labels, -100), labels)
    grad = torch.randn((t,), generator=g, device="cuda") / t
    return h, w, labels, grad


def _errors(h, w, labels, ignore):
    loss, lse, z = loss64(h, w, labels, ignore)
    top = float(z.abs().max()) if z.numel() else 0.0
    e = (h.shape[1] / 16 + 2) * 2.0 ** -22 * top
    return loss, lse, e + 16 * 2.0 ** -23 * lse.abs().clamp(min=1.0)


def _check_loss(h, w, labels, ignore=-100):
    from easyfhe import plain

    loss, lse = plain.vocab_loss(h, w, labels, ignore_index=ignore)
    want, want_lse, tol = _errors(h, w, labels, ignore)
    assert loss.dtype == lse.dtype == torch.float32 and loss.shape == labels.shape
    assert torch.equal(torch.isnan(loss), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert bool(((loss.double() - want).abs() <= 2 * tol)[ok].all()), float(
        ((loss.double() - want).abs() - 2 * tol)[ok].max())
    kept = labels != ignore
    assert bool(((lse.double() - want_lse).abs() <= tol)[kept].all())
    assert not loss[~kept].any() and not lse[~kept].any()
    return loss, lse


def _check_grad(h, w, labels, grad, lse, ignore=-100, need=(True, True), got=None):
    from easyfhe import plain

    dh, dw = got if got is not None else plain.vocab_loss_grad(
        h, w, labels, lse, grad, ignore_index=ignore, need_hidden=need[0], need_weight=need[1])
    assert (dh is not None, dw is not None) == need
    t, d = h.shape
    v = w.shape[0]
    if t == 0:
        assert dw is None or not dw.any()
        return dh, dw
    dz = loss_grad64(h, w, labels, ignore, grad)
    _, _, e = _errors(h, w, labels, ignore)
    step = half_step(h.dtype)
    counted = (labels != ignore)
    hc = torch.where(counted[:, None], h.double(), 0.0)
    # p's own error at the label is absolute: 2 e g p, which |dz| need not cover
    p = torch.exp(loss64(h, w, labels, ignore)[2] - loss64(h, w, labels, ignore)[1][:, None])
    size = (dz.abs() * (step + 2.0 ** -20)
            + 2 * e[:, None] * p * torch.where(counted, grad.double().abs(), 0.0)[:, None])
    size = size + 2.0 ** -126  # of every dz: no relative precision below
    gmax = float(torch.where(counted, grad.abs(), 0.0).max())
    if h.dtype == FP:
        size = size + torch.where(counted[:, None], 2.0 ** -38 * gmax, 0.0)
    for got_, want, tol, terms in (
            (dh, dz @ w.double(), size @ w.double().abs(), (v, dz.abs() @ w.double().abs())),
            (dw, dz.T @ hc, size.T @ hc.abs(), (t, dz.abs().T @ hc.abs()))):
        if got_ is None:
            continue
        n, total = terms
        tol = tol + (n / 16 + 16) * 2.0 ** -22 * total + 1.01 * step * want.abs() + 2.0 ** -126
        if h.dtype == FP:
            tol = tol + 2.0 ** -25
        diff = (got_.double() - want).abs()
        assert got_.dtype == h.dtype and got_.is_contiguous()
        assert bool((diff <= tol).all()), float((diff - tol).max())
    if dh is not None:
        assert not dh[~counted].any()
    return dh, dw


SHAPES = [(1, 1, 8), (1, 300, 8), (2, 255, 16), (5, 257, 64), (45, 1003, 200), (127, 256, 72),
          (128, 512, 128), (129, 511, 136), (130, 2000, 1000), (300, 777, 256)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,v,d", SHAPES)
def test_loss_and_gradients(dtype, t, v, d):
    h, w, labels, grad = _inputs(t, v, d, dtype)
    _, lse = _check_loss(h, w, labels)
    _check_grad(h, w, labels, grad, lse)
    _check_grad(h, w, labels, grad, lse, need=(True, False))
    _check_grad(h, w, labels, grad, lse, need=(False, True))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,v,d", [(16400, 9001, 16), (4100, 33000, 24), (700, 5000, 512)])
def test_many_pieces_and_tiles(dtype, t, v, d):
    """More words than one piece of dz holds, and many tiles per block."""
    h, w, labels, grad = _inputs(t, v, d, dtype, ignored=0.1)
    _, lse = _check_loss(h, w, labels)
    _check_grad(h, w, labels, grad, lse)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,v,d", [(1, 300, 8), (2, 700, 64), (31, 1003, 200), (33, 500, 72),
                                   (64, 2000, 136)])
def test_few_tokens_lose_nothing_but_the_outputs_rounding(dtype, t, v, d):
    """dz in two parts: off by the square of half a step instead of half a step.  An output
    may differ from its value by its own half step, the steps of its sum (2^-22 of the terms
    for each accumulation), dz's p (2 e, and 2^-20 for the exponential and its argument),
    what the second part cannot hold, and fp16's subnormals (2^-25 and, of dz under its
    scale, 2^-38 max|g|)."""
    from easyfhe import plain

    h, w, labels, grad = _inputs(t, v, d, dtype, ignored=0.2 if t > 2 else 0.0)
    _, lse = plain.vocab_loss(h, w, labels)
    dh, dw = plain.vocab_loss_grad(h, w, labels, lse, grad)
    dz = loss_grad64(h, w, labels, -100, grad)
    _, want_lse, e = _errors(h, w, labels, -100)
    counted = labels != -100
    g = torch.where(counted, grad.double().abs(), 0.0)[:, None]
    p = torch.exp(h.double() @ w.double().T - want_lse[:, None])
    step = half_step(dtype)
    size = dz.abs() * (2 * step ** 2 + 2.0 ** -20) + 2 * e[:, None] * p * g + 2.0 ** -126
    if dtype == FP:
        size = size + 2.0 ** -38 * float(g.max()) * counted[:, None]
    hc = torch.where(counted[:, None], h.double(), 0.0)
    for got, want, tol, n, total in (
            (dh, dz @ w.double(), size @ w.double().abs(), v, dz.abs() @ w.double().abs()),
            (dw, dz.T @ hc, size.T @ hc.abs(), 128, dz.abs().T @ hc.abs())):
        tol = tol + (n / 16 + 16) * 2.0 ** -22 * total + 1.01 * step * want.abs() + 2.0 ** -126
        if dtype == FP:
            tol = tol + 2.0 ** -25
        diff = (got.double() - want).abs()
        assert bool((diff <= tol).all()), float((diff / tol).max())


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,v,d", [(65, 300, 64), (130, 2000, 200), (1100, 700, 72)])
def test_hidden_gradient_keeps_the_labels_dz(dtype, t, v, d):
    """dz is rounded by up to half a step at every word but the label, whose remainder is
    added in binary32: there only half a step squared is lost (2^-24 of it).  The rest as for
    few tokens."""
    from easyfhe import plain

    h, w, labels, grad = _inputs(t, v, d, dtype, ignored=0.2)
    _, lse = plain.vocab_loss(h, w, labels)
    dh, _ = plain.vocab_loss_grad(h, w, labels, lse, grad, need_weight=False)
    dz = loss_grad64(h, w, labels, -100, grad)
    _, want_lse, e = _errors(h, w, labels, -100)
    counted = labels != -100
    g = torch.where(counted, grad.double().abs(), 0.0)[:, None]
    p = torch.exp(h.double() @ w.double().T - want_lse[:, None])
    step = half_step(dtype)
    lost = torch.full_like(dz, step)
    lost[torch.arange(t), labels.clamp(min=0)] = 2.0 ** -24
    size = dz.abs() * (1.01 * lost + 2.0 ** -20) + 2 * e[:, None] * p * g + 2.0 ** -126
    if dtype == FP:
        size = size + 2.0 ** -38 * float(g.max()) * counted[:, None]
    want, total = dz @ w.double(), dz.abs() @ w.double().abs()
    tol = size @ w.double().abs() + (v / 16 + 16) * 2.0 ** -22 * total
    tol = tol + 1.01 * step * want.abs() + 2.0 ** -126 + (2.0 ** -25 if dtype == FP else 0.0)
    diff = (dh.double() - want).abs()
    assert bool((diff <= tol).all()), float((diff / tol).max())
    assert not dh[~counted].any()


def test_a_last_piece_of_fewer_words():
    """Many tokens over a vocabulary whose last piece holds 64 words: fewer K blocks than
    the sum over a full piece is split into."""

    h, w, labels, grad = _inputs(38400, 49984, 64, BF, ignored=0.992)
    from easyfhe import plain

    _, lse = plain.vocab_loss(h, w, labels)
    dh, _ = plain.vocab_loss_grad(h, w, labels, lse, grad, need_weight=False)
    kept = labels != -100
    assert 200 < int(kept.sum()) < 400 and not dh[~kept].any()
    _check_grad(h[kept], w, labels[kept], grad[kept], lse[kept], need=(True, False),
                got=(dh[kept], None))


def test_offsets_past_32_bits():
    """A head of more than 2^31 values, labels among its first and last words."""
    from easyfhe import plain

    t, v, d = 7, 530000, 4096
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.empty((v, d), dtype=BF, device="cuda")
    for v0 in range(0, v, 50000):
        part = w[v0:v0 + 50000]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") / 64)
    labels = torch.tensor([0, v - 1, v - 2, -100, 3, v // 2, v - 1], device="cuda")
    h = (torch.randn((t, d), generator=g, device="cuda")
         + 9 * w[labels.clamp(min=0)].float()).to(BF)
    grad = torch.rand((t,), generator=g, device="cuda")
    loss, lse = plain.vocab_loss(h, w, labels)
    z = torch.cat([h.double() @ w[v0:v0 + 50000].double().T for v0 in range(0, v, 50000)], dim=1)
    counted = labels != -100
    want = torch.logsumexp(z, dim=1)
    tol = (d / 16 + 2) * 2.0 ** -22 * float(z.abs().max()) + 2.0 ** -18 * float(want.max())
    own = z.gather(1, labels.clamp(min=0)[:, None])[:, 0]
    assert bool(((lse - want).abs() <= tol)[counted].all())
    assert bool(((loss - (want - own)).abs() <= 2 * tol)[counted].all())
    dh, dw = plain.vocab_loss_grad(h, w, labels, lse, grad)
    dz = torch.exp(z - want[:, None])
    dz[torch.arange(t), labels.clamp(min=0)] -= 1.0
    dz *= torch.where(counted, grad, 0.0)[:, None]
    ends = torch.cat([torch.arange(300), torch.arange(v - 300, v)]).cuda()
    full = dz[:, ends].T @ h.double()
    size = dz[:, ends].abs().T @ h.double().abs()
    assert bool(((dw[ends] - full).abs() <= (2.1 * 2.0 ** -8 + 4 * tol) * size + 2.0 ** -126).all())
    full = sum(dz[:, v0:v0 + 50000] @ w[v0:v0 + 50000].double() for v0 in range(0, v, 50000))
    size = sum(dz[:, v0:v0 + 50000].abs() @ w[v0:v0 + 50000].double().abs()
               for v0 in range(0, v, 50000))
    assert bool(((dh - full).abs() <= (2.1 * 2.0 ** -8 + 4 * tol) * size).all())


def test_every_token_ignored_and_none():
    h, w, labels, grad = _inputs(70, 400, 64, BF)
    none = torch.full_like(labels, -100)
    loss, lse = _check_loss(h, w, none)
    dh, dw = _check_grad(h, w, none, grad, lse)
    assert not loss.any() and not dh.any() and not dw.any()
    h, w, labels, grad = _inputs(70, 400, 64, BF, ignored=0.0)
    _, lse = _check_loss(h, w, labels)
    _check_grad(h, w, labels, grad, lse)


@pytest.mark.parametrize("ignore", [-1, 7, 10 ** 12])
def test_another_ignored_label(ignore):
    h, w, labels, grad = _inputs(33, 300, 64, BF, ignored=0.0)
    labels[3:9] = ignore
    labels[0], labels[32] = 0, 299  # the borders of the vocabulary
    _, lse = _check_loss(h, w, labels, ignore)
    _check_grad(h, w, labels, grad, lse, ignore)


@pytest.mark.parametrize("t", [1, 33, 129, 300, 1030])
def test_ignored_label_is_a_word(t):
    """Rows past the last token are no token's: with a word as the ignored label they
    must leave no logit anywhere (many words: many entries beside the logits)."""
    h, w, labels, grad = _inputs(t, 20011, 64, BF, ignored=0.0)
    for ignore in (0, 7, 20010):
        lab = labels.clone()
        lab[lab == ignore] = 3
        lab[::5] = ignore
        _, lse = _check_loss(h, w, lab, ignore)
        _check_grad(h, w, lab, grad, lse, ignore)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_garbage_in_ignored_rows_reaches_nothing(dtype):
    from easyfhe import plain

    h, w, labels, grad = _inputs(140, 600, 128, dtype, ignored=0.0)
    labels[[0, 5, 139]] = -100
    clean = plain.vocab_loss(h, w, labels)
    clean_grad = plain.vocab_loss_grad(h, w, labels, clean[1], grad)
    h[0], h[5, 3], h[139, 100] = float("nan"), float("inf"), -float("inf")
    grad[5] = float("nan")
    loss, lse = plain.vocab_loss(h, w, labels)
    assert torch.equal(loss, clean[0])
    kept = labels != -100
    assert torch.equal(lse[kept], clean[1][kept])
    for a, b in zip(plain.vocab_loss_grad(h, w, labels, lse, grad), clean_grad):
        assert torch.equal(a, b)


def test_labels_outside_the_vocabulary_are_nan():
    from easyfhe import plain

    h, w, labels, grad = _inputs(20, 300, 64, BF, ignored=0.0)
    clean, _ = plain.vocab_loss(h, w, labels)
    labels[4], labels[11], labels[12] = 300, -3, 2 ** 40
    loss, lse = _check_loss(h, w, labels)
    good = torch.ones(20, dtype=torch.bool, device="cuda")
    good[[4, 11, 12]] = False
    assert torch.equal(loss[good], clean[good]) and torch.isnan(loss[~good]).all()
    dh, dw = plain.vocab_loss_grad(h, w, labels, lse, grad)
    assert torch.isnan(dh[~good]).all() and torch.isfinite(dh[good]).all()
    assert torch.isnan(dw).all()


def test_nan_and_infinite_logits():
    from easyfhe import plain

    h, w, labels, _ = _inputs(9, 700, 64, BF, ignored=0.0)
    clean, _ = plain.vocab_loss(h, w, labels)
    h[2, 0], h[6, 1] = float("nan"), float("inf")
    loss, lse = plain.vocab_loss(h, w, labels)
    keep = torch.tensor([0, 1, 3, 4, 5, 7, 8], device="cuda")
    assert torch.equal(loss[keep], clean[keep])
    assert torch.isnan(loss[[2, 6]]).all() and torch.isnan(lse[[2, 6]]).all()
    # words that cannot occur: a row of the type's lowest value drives its logit to -inf
    h, w, labels, grad = _inputs(9, 700, 64, BF, ignored=0.0)
    h[:, 0] = 3.0
    w[100:400] = 0.0
    w[100:400, 0] = torch.finfo(BF).min
    labels[:] = 5
    loss, lse = plain.vocab_loss(h, w, labels)
    keep = torch.cat([w[:100], w[400:]])
    want, want_lse, tol = _errors(h, keep, labels, -100)
    assert bool(((loss.double() - want).abs() <= 2 * tol).all())
    dh, _ = plain.vocab_loss_grad(h, w, labels, lse, grad, need_weight=False)
    ref, _ = plain.vocab_loss_grad(h, keep, labels, lse, grad, need_weight=False)
    assert torch.isfinite(dh).all()
    assert bool(((dh - ref).abs() <= 4 * half_step(BF) * (ref.abs() + dh.abs()) + 1e-6).all())


@pytest.mark.parametrize("dtype", [BF, FP])
def test_confident_and_hopeless_tokens(dtype):
    """p(label) from nearly 1 (where p - 1 cancels) to e^-60."""
    h, w, labels, grad = _inputs(64, 500, 256, dtype, ignored=0.0)
    lean = torch.linspace(-40, 40, 64, device="cuda")[:, None]
    h = (h.float() + lean * w[labels].float()).to(dtype)
    _, lse = _check_loss(h, w, labels)
    _check_grad(h, w, labels, grad, lse)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("v", [3, 300, 5000])
def test_a_small_loss_keeps_its_precision(dtype, v):
    """Losses down to 1e-9.  The others' share of the sum is exp(z_v - z_label), each off by
    2 e relative with e a logit's error (D / 16 + 2 accumulations of 2^-22 max|z|), the
    exponential's argument (its own step, 2^-23 of up to 64) and the sums: 32 terms a group
    and at most 100 joins of three roundings, 2^-24 each."""
    from easyfhe import plain

    h, w, labels, _ = _inputs(40, v, 64, dtype, ignored=0.0)
    lean = torch.linspace(0, 32, 40, device="cuda")[:, None]
    h = (0.2 * h.float() + lean * w[labels].float()).to(dtype)
    loss, _ = plain.vocab_loss(h, w, labels)
    z = h.double() @ w.double().T
    own = z.gather(1, labels[:, None])
    others = torch.exp(z - own).scatter(1, labels[:, None], 0.0).sum(1)
    want = torch.log1p(others)
    e = (64 / 16 + 2) * 2.0 ** -22 * float(z.abs().max())
    tol = want * (2 * e + 64 * 2.0 ** -22 + (32 + 300) * 2.0 ** -24)
    small = (z - own).max(1).values <= 0  # the label's word is the likeliest
    assert int(small.sum()) > 20 and float(want[small].min()) < 1e-6
    assert bool(((loss.double() - want).abs() <= tol)[small].all()), float(
        ((loss.double() - want).abs() / tol)[small].max())


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t", [3, 200])
def test_long_sums_of_one_sign(dtype, t):
    """8192 positive products: an accumulation over all of them would lose up to 512 steps of
    the sum.  Chunks of 512 products lose 32 steps (2^-23) of their own sums, which add up to
    the logit, and 16 half steps where they are joined; lse and loss have 16 steps besides."""
    from easyfhe import plain

    g = torch.Generator(device="cuda").manual_seed(3)
    h = (0.5 + torch.rand((t, 8192), generator=g, device="cuda")).to(dtype)
    w = ((0.5 + torch.rand((700, 8192), generator=g, device="cuda")) / 200).to(dtype)
    labels = torch.randint(0, 700, (t,), generator=g, device="cuda")
    loss, lse = plain.vocab_loss(h, w, labels)
    want, want_lse, z = loss64(h, w, labels, -100)
    tol = (34 * 2.0 ** -23 + 16 * 2.0 ** -24 + 16 * 2.0 ** -23) * float(z.abs().max())
    assert bool(((lse.double() - want_lse).abs() <= tol).all()), float(
        (lse.double() - want_lse).abs().max() / tol)
    assert bool(((loss.double() - want).abs() <= 2 * tol).all())


def test_gradients_span_types_ranges():
    """Upstream gradients from 1e-8 to 1e4 in fp16: the scale keeps what the
    outputs can hold, and zeros give zeros."""
    h, w, labels, grad = _inputs(50, 300, 64, FP, ignored=0.0)
    _, lse = _check_loss(h, w, labels)
    for scale in (1e-6, 1.0, 1e4):
        _check_grad(h, w, labels, grad * scale, lse)
    dh, dw = _check_grad(h, w, labels, grad * 0, lse)
    assert not dh.any() and not dw.any()


def test_views_and_odd_offsets():
    h, w, labels, grad = _inputs(60, 500, 64, BF)
    wide = torch.randn((500, 200), device="cuda").to(BF)
    tall = torch.randn((60, 203), device="cuda").to(BF)
    g2 = torch.stack([grad, grad], 1)[:, 0]
    l2 = torch.stack([labels, labels], 1)[:, 1]
    for hh in (h, tall[:, :64], tall[:, 5:69], h.T.contiguous().T, h[:1].expand(60, 64)):
        for ww in (w, wide[:, 8:72], wide[:, 3:67], wide[::2, :64]):
            lab = torch.where(l2 >= 0, l2 % ww.shape[0], l2)
            _, lse = _check_loss(hh, ww, lab)
            _check_grad(hh, ww, lab, g2, lse)


def test_no_tokens():
    from easyfhe import plain

    h, w, labels, grad = _inputs(4, 50, 32, BF)
    loss, lse = plain.vocab_loss(h[:0], w, labels[:0])
    assert loss.shape == lse.shape == (0,)
    dh, dw = plain.vocab_loss_grad(h[:0], w, labels[:0], lse, grad[:0])
    assert dh.shape == (0, 32) and not dw.any()


def test_gradient_against_differences():
    """Directional derivatives of the binary64 loss: central differences of
    step 2^-8 are off by the third derivative's 2^-16 / 6, far below the
    gradient's own rounding (half a step per component, summed absolutely)."""
    from easyfhe import plain

    h, w, labels, grad = _inputs(30, 200, 64, BF, ignored=0.2)
    _, lse = plain.vocab_loss(h, w, labels)
    dh, dw = plain.vocab_loss_grad(h, w, labels, lse, grad)
    gen = torch.Generator(device="cuda").manual_seed(8)
    eps = 2.0 ** -8

    def total(hh, ww):
        return float((loss64(hh, ww, labels, -100)[0] * grad.double()).sum())

    for which, d in ((0, dh), (1, dw)):
        u = torch.randn(d.shape, generator=gen, device="cuda", dtype=torch.float64)
        a = [h.double(), w.double()]
        b = [h.double(), w.double()]
        a[which] = a[which] + eps * u / u.norm()
        b[which] = b[which] - eps * u / u.norm()
        diff = (total(*a) - total(*b)) / (2 * eps)
        mine = float((d.double() * u).sum() / u.norm())
        # dz's rounding spreads over a row: its sum is bounded by that of |dz| |w|
        dz = loss_grad64(h, w, labels, -100, grad).abs()
        reach = dz @ w.double().abs() if which == 0 else dz.T @ h.double().abs()
        tol = float((u.abs() * reach).sum() / u.norm()) * 2 * half_step(BF) + 2.0 ** -16
        assert abs(diff - mine) <= tol, (which, diff, mine, tol)


def test_repeated_calls_are_equal():
    from easyfhe import plain

    h, w, labels, grad = _inputs(200, 3000, 256, BF)
    runs = []
    for _ in range(3):
        loss, lse = plain.vocab_loss(h, w, labels)
        runs.append((loss, lse, *plain.vocab_loss_grad(h, w, labels, lse, grad)))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_two_streams_and_two_graphs():
    from easyfhe import plain

    h, w, labels, grad = _inputs(90, 1500, 128, FP)
    h2, w2, labels2, grad2 = _inputs(150, 900, 64, BF, seed=3)

    def step(h, w, labels, grad):
        loss, lse = plain.vocab_loss(h, w, labels)
        return (loss, *plain.vocab_loss_grad(h, w, labels, lse, grad))

    want, want2 = step(h, w, labels, grad), step(h2, w2, labels2, grad2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, args in zip(streams, ((h, w, labels, grad), (h2, w2, labels2, grad2))):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([step(*args) for _ in range(3)][-1])
    torch.cuda.synchronize()
    for a, b in zip(got, (want, want2)):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs, outs = [], []
    for args in ((h, w, labels, grad), (h2, w2, labels2, grad2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*args))
        graphs.append(g)
    for g, s in zip(graphs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, (want, want2)):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    # new inputs in the captured buffers
    n = _inputs(90, 1500, 128, FP, seed=11)
    for dst, src in zip((h, w, labels, grad), n):
        dst.copy_(src)
    graphs[0].replay()
    _, lse = plain.vocab_loss(h, w, labels)
    _check_grad(h, w, labels, grad, lse, got=outs[0][1:])


def test_refusals():
    from easyfhe import plain

    h, w, labels, grad = _inputs(6, 40, 32, BF)
    _, lse = plain.vocab_loss(h, w, labels)
    for args in ((h.float(), w, labels), (h.half(), w, labels), (h[:, :24], w, labels),
                 (h[:, :20], w[:, :20], labels), (h, w[:0], labels), (h, w, labels.int()),
                 (h, w, labels[:5]), (h, w.cpu(), labels), (h[0], w, labels),
                 (h.clone().requires_grad_(), w, labels)):
        with pytest.raises(ValueError):
            plain.vocab_loss(*args)
    for kw in ({"lse": lse.double()}, {"lse": lse[:3]}, {"grad": grad.half()},
               {"grad": grad[:2]}, {"grad": grad.cpu()},
               {"need": (False, False)}):
        need = kw.pop("need", (True, True))
        with pytest.raises(ValueError):
            plain.vocab_loss_grad(h, w, labels, kw.get("lse", lse), kw.get("grad", grad),
                                  need_hidden=need[0], need_weight=need[1])


def test_a_small_workspace_is_refused():
    from easyfhe import _native

    h, w, labels, grad = _inputs(6, 40, 32, BF)
    out = torch.full((4, 40, 32), 3.0, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    args = (h.data_ptr(), 32, w.data_ptr(), 32, 3, 6, 40, 32, labels.data_ptr(), -100)
    need = _native.lib.b2f_vocab_loss_workspace(6, 40, 32)
    need_grad = _native.lib.b2f_vocab_loss_grad_workspace(6, 40, 32, 1)
    with pytest.raises(ValueError, match="too small"):
        _native.call("b2f_vocab_loss", *args, out[0].data_ptr(), out[1].data_ptr(),
                     ws.data_ptr(), need - 1, None)
    with pytest.raises(ValueError, match="too small"):
        _native.call("b2f_vocab_loss_grad", *args, out[0].data_ptr(), out[1].data_ptr(),
                     out[2].data_ptr(), out[3].data_ptr(), ws.data_ptr(), need_grad - 1, None)
    torch.cuda.synchronize()
    assert bool((out == 3.0).all())


def test_no_wait_ran_out():
    from easyfhe import _native

    torch.cuda.synchronize()
    assert _native.lib.b2f_vocab_loss_wait_errors() == 0
