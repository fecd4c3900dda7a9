"""Waits inside the vocabulary loss that run out (csrc/vocab_loss.cu): one thread block that
loads nothing, so that nothing of its sums arrives."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent

# In a process of its own: the counter is the process's.
CODE = """
import sys
sys.path[:0] = [{root!r}, {pkg!r}]
import torch
from easyfhe import _native, plain

T, V, D = {t}, 3000, 320
g = torch.Generator(device="cuda").manual_seed(T)
h = torch.randn((T, D), generator=g, device="cuda").to(torch.{dtype})
w = (torch.randn((V, D), generator=g, device="cuda") / D ** 0.5).to(torch.{dtype})
labels = torch.randint(0, V, (T,), generator=g, device="cuda")
labels[::7] = -100
kept = labels != -100
up = torch.rand((T,), generator=g, device="cuda") + 0.5
_, lse = plain.vocab_loss(h, w, labels)

def step():
    return (*plain.vocab_loss(h, w, labels), *plain.vocab_loss_grad(h, w, labels, lse, up))

want = step()
assert all(torch.isfinite(x).all() for x in want) and plain.wait_errors() == 0
before = 0
for product in range(4):
    _native.call("b2f_vocab_loss_idle_block", product, 0)
    loss, lse_, dh, dw = got = step()
    _native.call("b2f_vocab_loss_idle_block", product, -1)
    torch.cuda.synchronize()
    assert plain.wait_errors("cuda") > before, product
    before = plain.wait_errors()
    # what is not NaN is what it should be, and there is NaN where the block's tiles were
    for a, b in zip(got, want):
        ok = ~torch.isnan(a)
        assert torch.equal(a[ok], b[ok]), product
    nan = [bool(torch.isnan(x).any()) for x in got]
    assert nan == {{0: [True, True, False, False], 1: [False, False, True, True],
                   2: [False, False, True, False], 3: [False, False, False, True]}}[product], nan
    if product == 0:  # a token whose logits are not all there has no loss
        assert torch.equal(torch.isnan(loss), torch.isnan(lse_))
        assert bool(torch.isnan(loss[kept][:60]).all())
    assert not loss[~kept].any() and not dh[~kept].any()
    again = step()  # the next call is whole
    assert all(torch.equal(a, b) for a, b in zip(again, want)), product
assert plain.wait_errors() == before
print("whole")
"""


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("t", [40, 100, 700, 1500])
def test_what_a_lost_wait_owes_is_nan(t, dtype):
    code = CODE.format(root=str(ROOT), pkg=str(ROOT / "easyfhe-llama3-8b_b200"), t=t, dtype=dtype)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "whole" in r.stdout, r.stderr[-2000:]


def test_a_healthy_device_counts_none():
    from easyfhe import plain

    h = torch.randn((5, 64), device="cuda").bfloat16()
    plain.vocab_loss(h, h, torch.arange(5, device="cuda"))
    assert plain.wait_errors() == 0 == plain.wait_errors("cuda:0")
