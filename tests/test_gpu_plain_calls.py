"""Calls that the operators' documentation allows and their own tests do not
make: first use inside a capture, several threads at once, inference mode."""

from __future__ import annotations

import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent

FIRST = """
import sys
sys.path[:0] = [{root!r}, {pkg!r}]
import torch
from easyfhe import plain
q = torch.randn(5, 3, 64, device="cuda").bfloat16()
pos = torch.arange(5, device="cuda")
plan = plain.RopePlan(64)
codes = torch.randint(0, 16, (100, 128), device="cuda", dtype=torch.uint8)
w4 = plain.pack_q4(codes, torch.ones((100, 1), device="cuda").half())
x = torch.randn(2, 128, device="cuda")
h = torch.randn(150, 64, device="cuda").bfloat16()
w = torch.randn(300, 64, device="cuda").bfloat16()
lab = torch.randint(0, 300, (150,), device="cuda")
g = torch.ones(150, device="cuda")

def step():
    loss, lse = plain.vocab_loss(h, w, lab)
    return (plain.rope(q, positions=pos, plan=plan), plain.q4_matvec(x, w4), loss, lse,
            *plain.vocab_loss_grad(h, w, lab, lse, g))

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = step()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(captured, step()):
    assert torch.equal(a, b)
print("same")
"""


def test_first_use_inside_a_capture():
    code = FIRST.format(root=str(ROOT), pkg=str(ROOT / "easyfhe-llama3-8b_b200"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def _work(seed):
    from easyfhe import plain

    g = torch.Generator(device="cuda").manual_seed(seed)
    t, v, d = 40 + 50 * seed, 700 + 90 * seed, 64 + 8 * seed
    h = torch.randn((t, d), generator=g, device="cuda").bfloat16()
    w = torch.randn((v, d), generator=g, device="cuda").bfloat16()
    lab = torch.randint(0, v, (t,), generator=g, device="cuda")
    grad = torch.rand((t,), generator=g, device="cuda")
    q = torch.randn((t, 4, 64), generator=g, device="cuda")
    pos = torch.arange(t, device="cuda")
    plan = plain.RopePlan(64, rotary_dim=32)
    w4 = plain.quantize_q4(w.float(), group=32)

    def run():
        loss, lse = plain.vocab_loss(h, w, lab)
        return (loss, *plain.vocab_loss_grad(h, w, lab, lse, grad),
                plain.rope(q, positions=pos, plan=plan), plain.q4_matvec(h[:3], w4))

    return run


def test_threads_at_once():
    runs = [_work(s) for s in range(4)]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def body(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = runs[i]()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # shown below, in the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=body, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_inference_mode_and_parameters():
    run = _work(2)
    want = run()
    with torch.inference_mode():
        got = run()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    from easyfhe import plain

    w = torch.nn.Parameter(torch.randn((90, 64), device="cuda").bfloat16())
    h = torch.randn((5, 64), device="cuda").bfloat16()
    lab = torch.arange(5, device="cuda")
    with pytest.raises(ValueError, match="gradient"):
        plain.vocab_loss(h, w, lab)
    with torch.no_grad():
        loss, lse = plain.vocab_loss(h, w, lab)
        dh, dw = plain.vocab_loss_grad(h, w, lab, lse, torch.ones_like(loss))
    assert not (loss.requires_grad or dh.requires_grad or dw.requires_grad)
    w.grad = dw
    torch.optim.SGD([w], lr=0.1).step()
    assert torch.isfinite(w).all()


def test_copies_of_plans_and_weights_stand_alone():
    import copy

    from easyfhe import plain

    plan = plain.RopePlan(64)
    w = plain.quantize_q4(torch.randn((50, 128), device="cuda"))
    q, x = torch.randn((4, 2, 64), device="cuda"), torch.randn((2, 128), device="cuda")
    pos = torch.arange(4, device="cuda")
    want = plain.rope(q, positions=pos, plan=plan), plain.q4_matvec(x, w)
    plan2, w2 = copy.deepcopy(plan), copy.deepcopy(w)
    plan.freqs.zero_()
    w.packed.zero_()
    assert torch.equal(plain.rope(q, positions=pos, plan=plan2), want[0])
    assert torch.equal(plain.q4_matvec(x, w2), want[1])


def test_dual_tensors_are_refused():
    from torch.autograd import forward_ad

    from easyfhe import plain

    plan = plain.RopePlan(64)
    w4 = plain.quantize_q4(torch.randn((50, 64), device="cuda"), group=64)
    h, lab = torch.randn((5, 64), device="cuda").bfloat16(), torch.arange(5, device="cuda")
    loss, lse = plain.vocab_loss(h, h, lab)
    one = torch.ones_like(loss)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: plain.rope(dual(h)[None], positions=lab[:1], plan=plan),
                     lambda: plain.rope(h[None], dual(h)[None], positions=lab[:1], plan=plan),
                     lambda: plain.rope_grad(dual(h)[None], positions=lab[:1], plan=plan),
                     lambda: plain.q4_matvec(dual(h), w4), lambda: plain.q4_codes(dual(h)),
                     lambda: plain.vocab_loss(dual(h), h, lab),
                     lambda: plain.vocab_loss(h, dual(h), lab),
                     lambda: plain.vocab_loss_grad(h, h, lab, dual(lse), one),
                     lambda: plain.vocab_loss_grad(h, h, lab, lse, dual(one))):
            with pytest.raises(ValueError, match="dual"):
                call()
        assert torch.equal(plain.vocab_loss(h, h, lab)[0], loss)
