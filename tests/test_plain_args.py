"""The plaintext operators' refusals that need no GPU: the C ABI checks its
arguments before anything touches a device, and the host-side plans theirs."""

from __future__ import annotations

import math

import pytest

P = 1 << 20  # an aligned address; every call below is refused before it is used


def _refused(name, *args, match, kind=ValueError):
    from easyfhe import _native

    with pytest.raises(kind, match=match):
        _native.call(name, *args)


def test_rope_refusals():
    from easyfhe import plain

    def heads(where, count):
        return plain._HEADS.pack(where, P, 0, 64, 64, 0, 64, 64, count)

    def bad(match, p=heads(P, 1), parts=1, dtype=3, batch=1, seq=1, dim=64, rotary=64, pos=P, freqs=P):
        _refused("b2f_rope", p, parts, dtype, batch, seq, dim,
                 rotary, 0, pos, 1, 0, 1, freqs, 1.0, 0, None, match=match)

    bad("one or two", p=None)
    bad("one or two", parts=3)
    bad("dtype", dtype=4)
    bad("batch", batch=-1)
    bad("head of", dim=1025, rotary=64)
    bad("head of", rotary=63)
    bad("head of", rotary=66)
    bad("tokens", batch=2, seq=1 << 31)
    bad("null", pos=None)
    bad("null", freqs=None)
    bad("misaligned", p=heads(P + 1, 1))
    bad("heads", p=heads(P, 0))


def test_q4_refusals():
    def pack(match, codes=P, scales=P, zeros=None, n=16, k=64, group=64, out=P):
        _refused("b2f_q4_pack", codes, scales, zeros, n, k, group, out, None, match=match)

    pack("weight of", n=0)
    pack("weight of", k=131073)
    pack("group of", group=96 + 1)
    pack("group of", group=48)
    pack("null", codes=None)
    pack("null", out=None)
    pack("misaligned", out=P + 16)
    pack("misaligned", scales=P + 1)

    def quant(match, dtype=1, ld=64, symmetric=1, scale=3, zeros=None):
        _refused("b2f_q4_quantize", P, dtype, ld, 16, 64, 64, symmetric, scale, P, P, zeros, None,
                 match=match)

    quant("dtype", dtype=0)
    quant("apart", ld=63)
    quant("scale dtype", scale=1)
    quant("null", symmetric=0)

    def mv(match, x=P, dtype=3, ldx=64, rows=1, scale=3, group=64, y=P):
        _refused("b2f_q4_matvec", x, dtype, ldx, rows, P, scale, 0, 16, 64, group, y, 0, None,
                 match=match)

    mv("rows", rows=1025)
    mv("dtype", dtype=0)
    mv("scale dtype", scale=1)
    mv("null", x=None)
    mv("apart", rows=2, ldx=32)
    mv("misaligned", x=P + 1)
    mv("group of", group=16)


def test_vocab_loss_refusals():
    def loss(match, h=P, ldh=64, ldw=64, dtype=3, t=4, v=9, d=64, ws=P):
        _refused("b2f_vocab_loss", h, ldh, P, ldw, dtype, t, v, d, P, -100, P, P, ws,
                 1 << 20, None, match=match)

    loss("dtype", dtype=1)
    loss("hidden size", d=60)
    loss("words", v=0)
    loss("apart", ldh=56)
    loss("apart", ldw=68)
    loss("null", h=None)
    loss("null", ws=None)
    loss("misaligned", h=P + 8)
    loss("misaligned", ws=P + 16)

    def grad(match, dh=P, dw=P, lse=P):
        _refused("b2f_vocab_loss_grad", P, 64, P, 64, 3, 4, 9, 64, P, -100, lse, P, dh, dw, P, 0,
                 None, match=match)

    grad("no gradient", dh=None, dw=None)
    grad("null", lse=None)
    grad("misaligned", dw=P + 8)


def test_rope_frequencies():
    from easyfhe.plain import rope_frequencies

    f, m = rope_frequencies(128, 500000.0)
    assert m == 1.0 and f[0] == 1.0 and f[-1] == 500000.0 ** (-126 / 128)
    lin, _ = rope_frequencies(128, 500000.0, {"type": "linear", "factor": 4.0})
    assert lin == [x / 4.0 for x in f]
    bands, _ = rope_frequencies(128, 500000.0, {"type": "bands", "factor": 8.0, "low": 1.0,
                                                "high": 4.0, "original": 8192})
    for x, y in zip(f, bands):
        turns = 8192 * x / (2 * math.pi)
        assert (y == x) if turns >= 4 else (y == x / 8) if turns <= 1 else x / 8 < y < x
    yarn, m = rope_frequencies(64, 10000.0, {"type": "yarn", "factor": 16.0, "original": 4096,
                                             "fast": 32.0, "slow": 1.0})
    assert yarn[0] == 1.0 and yarn[-1] == 10000.0 ** (-62 / 64) / 16.0
    assert m == 0.1 * math.log(16.0) + 1.0
    assert all(a > b for a, b in zip(yarn, yarn[1:]))
    for kw in ({"rotary_dim": 63}, {"theta": 0.0}, {"theta": math.inf},
               {"scaling": {"type": "other"}}, {"scaling": {"type": "linear"}},
               {"scaling": {"type": "linear", "factor": -1.0}},
               {"scaling": {"type": "bands", "factor": 8.0, "low": 4.0, "high": 4.0,
                            "original": 8192}}):
        with pytest.raises(ValueError):
            rope_frequencies(**{"rotary_dim": 64, **kw})


def test_host_tensors_are_refused():
    import torch

    from easyfhe import plain

    with pytest.raises(ValueError, match="CUDA"):
        plain.RopePlan(64, device="cpu")
    for args in ((63,), (0,), (2048,)):
        with pytest.raises(ValueError):
            plain.RopePlan(*args, device="cpu")
    with pytest.raises(ValueError, match="layout"):
        plain.RopePlan(64, layout="pairs", device="cpu")
    h = torch.zeros(2, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        plain.vocab_loss(h, h, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        plain.pack_q4(torch.zeros(2, 64, dtype=torch.uint8), h[:, :1])
    with pytest.raises(ValueError, match="weight"):
        plain.q4_matvec(h, h)


def test_dual_tensors_are_refused():
    """A tangent would be lost without a word: the output would have none."""
    import torch
    from torch.autograd import forward_ad

    from easyfhe import plain

    x = torch.zeros(2, 8)
    assert plain._plain_tensor(x, -1)  # as on a device of that number
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        assert not plain._plain_tensor(dual, -1)
        assert plain._plain_tensor(forward_ad.unpack_dual(dual).primal, -1)
        assert plain._plain_tensor(x, -1)
        with torch.no_grad():
            assert not plain._plain_tensor(dual, -1)
    assert plain._plain_tensor(x, -1)


@pytest.mark.parametrize("run", ["run_layer0", "run_prefill"])
def test_an_answer_that_cannot_be_given_is_refused_first(run, monkeypatch):
    """Before the encrypted layers run: a head without tokens, with tokens that are not the
    prompt's, or with the checks off."""
    from types import SimpleNamespace

    import torch

    import llama3_layer

    def reached():
        raise AssertionError("the layers would have run")

    monkeypatch.setattr(llama3_layer, "import_reference", reached)
    run = getattr(llama3_layer, run)
    head = SimpleNamespace(weight=torch.empty((1000, 4096), device="meta"))
    small = SimpleNamespace(weight=torch.empty((1000, 64), device="meta"))
    tokens = torch.arange(128)
    for kw in ({"head": head}, {"tokens": tokens}, {"head": head, "tokens": tokens, "check": False},
               {"head": head, "tokens": tokens[:127]}, {"head": head, "tokens": tokens + 873},
               {"head": head, "tokens": tokens - 1}, {"head": head, "tokens": tokens.float()},
               {"head": small, "tokens": tokens}):
        with pytest.raises(ValueError):
            run(**kw)
    for kw in ({}, {"head": head, "tokens": tokens}, {"head": head, "tokens": list(range(128))}):
        with pytest.raises(AssertionError, match="would have run"):
            run(**kw)
