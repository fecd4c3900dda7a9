"""Rotary positions (csrc/rope.cu) against the formula in binary64.

Tolerance: the output's rounding, half a step of its type, and the binary32
product: the angle's fraction of a turn is rounded to binary32 (2^-25 turns,
times 2 pi: 1.9e-7), sine and cosine are off by up to 2 steps (2.4e-7), the two
products and their sum add 3 half steps (1.8e-7): below 1e-6 of (|x0| + |x1|)
times the factor.  Binary64 inputs: the same angle product on both sides, two
sines within 2 steps each and three roundings: 8 x 2^-53.  Elements that only
pass through are equal."""

from __future__ import annotations

import pytest
import torch

from _plain import half_step, rope64

pytestmark = pytest.mark.gpu

SCALINGS = [None, {"type": "linear", "factor": 4.0},
            {"type": "bands", "factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192},
            {"type": "yarn", "factor": 16.0, "original": 4096, "fast": 32.0, "slow": 1.0}]


def _check(y, x, pos, plan, gradient=False):
    from easyfhe import plain

    freqs, factor = plan.freqs.tolist(), plan.factor
    if x.dim() == 3:
        y, x = y[None], x[None]
    pos = pos.expand(x.shape[0], x.shape[1])
    want, size = rope64(x, pos, freqs, factor, plan.rotary_dim, plan.layout, gradient)
    rel = 8 * 2.0 ** -53 if x.dtype == torch.float64 else 1e-6
    tol = half_step(y.dtype) * want.abs() + rel * size
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step of its subnormals
    assert y.dtype == x.dtype and y.is_contiguous()
    assert bool(((y.double() - want).abs() <= tol).all()), float(
        ((y.double() - want).abs() - tol).max())
    r = plan.rotary_dim
    assert torch.equal(y[..., r:], x[..., r:])
    assert plain is not None


def _x(*shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (96, 64), (2, 2), (6, 6), (80, 20), (37, 34),
                                        (256, 250), (1024, 1024)])
def test_rope_and_gradient(dtype, layout, dim, rotary):
    from easyfhe import plain

    for i, gradient in enumerate((False, True)):
        plan = plain.RopePlan(dim, rotary_dim=rotary, theta=10000.0, layout=layout,
                              scaling=SCALINGS[(dim + i) % 4])
        q, k = _x(2, 19, 5, dim, dtype=dtype, seed=1), _x(2, 19, 3, dim, dtype=dtype, seed=2)
        pos = torch.tensor([[3], [100000]], device="cuda") + torch.arange(19, device="cuda")
        f = plain.rope_grad if gradient else plain.rope
        yq, yk = f(q, k, positions=pos, plan=plan)
        _check(yq, q, pos, plan, gradient)
        _check(yk, k, pos, plan, gradient)


@pytest.mark.parametrize("seq", [1, 2, 3, 4, 5, 63, 128, 1001])
def test_lengths_and_one_tensor(seq):
    from easyfhe import plain

    plan = plain.RopePlan(128)
    q = _x(seq, 7, 128, dtype=torch.bfloat16)
    pos = torch.arange(seq, device="cuda", dtype=torch.int32)
    _check(plain.rope(q, positions=pos, plan=plan), q, pos[None], plan)


def test_rotation_of_position_zero_and_no_tokens():
    from easyfhe import plain

    plan = plain.RopePlan(64)
    q = _x(1, 2, 64, dtype=torch.float32)
    zero = torch.zeros(1, device="cuda", dtype=torch.int64)
    assert torch.equal(plain.rope(q, positions=zero, plan=plan), q)
    e, k = plain.rope(q[:0], q[:0, :1], positions=zero[:0], plan=plan)
    assert e.shape == (0, 2, 64) and k.shape == (0, 1, 64)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_views(layout):
    """Views of a fused buffer, transposed and expanded tensors, odd offsets."""
    from easyfhe import plain

    plan = plain.RopePlan(64, rotary_dim=48, layout=layout)
    buf = _x(2, 33, 12, 64, dtype=torch.bfloat16)
    pos = torch.arange(33, device="cuda").expand(2, 33)
    q, k = buf[:, :, :6], buf[:, :, 6:9]
    for t, y in zip((q, k), plain.rope(q, k, positions=pos, plan=plan)):
        _check(y, t, pos, plan)
    t = buf.transpose(1, 2).contiguous().transpose(1, 2)  # heads outermost
    _check(plain.rope(t, positions=pos, plan=plan), t, pos, plan)
    one = buf[:, :, :1].expand(2, 33, 4, 64)  # one head read four times
    _check(plain.rope(one, positions=pos, plan=plan), one, pos, plan)
    last = buf.transpose(2, 3).contiguous().transpose(2, 3)  # last stride not 1
    _check(plain.rope(last, positions=pos, plan=plan), last, pos, plan)
    odd = _x(1 + 2 * 5 * 65, dtype=torch.bfloat16)[1:].view(2, 5, 65)[:, :, :64]
    _check(plain.rope(odd, positions=pos[0, :2], plan=plan), odd, pos[:1, :2], plan)
    every = torch.arange(66, device="cuda")[::2]  # strided positions
    _check(plain.rope(q, positions=every, plan=plan), q, every[None], plan)


def test_far_and_negative_positions():
    from easyfhe import plain

    plan = plain.RopePlan(128, theta=500000.0)
    pos = torch.tensor([2 ** 31 - 1, -5, 2 ** 33 + 7, 10 ** 6], device="cuda")
    for dtype in (torch.float32, torch.float64):
        q = _x(4, 3, 128, dtype=dtype)
        _check(plain.rope(q, positions=pos, plan=plan), q, pos[None], plan)


def test_offsets_past_32_bits():
    from easyfhe import plain

    plan = plain.RopePlan(64)
    buf = torch.empty(2 ** 31 + 4096, dtype=torch.bfloat16, device="cuda")
    q = buf.as_strided((2, 2, 2, 64), (2 ** 31, 128, 64, 1))
    q.copy_(_x(2, 2, 2, 64, dtype=torch.bfloat16))
    pos = torch.arange(2, device="cuda")
    _check(plain.rope(q, positions=pos, plan=plan), q, pos[None], plan)


def test_infinities_stay_in_their_pair():
    from easyfhe import plain

    plan = plain.RopePlan(64)
    q = _x(3, 2, 64, dtype=torch.float32)
    want = plain.rope(q, positions=torch.arange(3, device="cuda"), plan=plan)
    q[1, 1, 5], q[1, 1, 7] = float("inf"), float("nan")
    y = plain.rope(q, positions=torch.arange(3, device="cuda"), plan=plan)
    touched = torch.zeros_like(y, dtype=torch.bool)
    touched[1, 1, [5, 37, 7, 39]] = True
    assert torch.equal(y[~touched], want[~touched])
    assert not torch.isfinite(y[touched]).any()


def test_capture_and_another_stream():
    from easyfhe import plain

    plan = plain.RopePlan(128)
    q, k = _x(40, 4, 128, dtype=torch.bfloat16), _x(40, 2, 128, dtype=torch.bfloat16, seed=3)
    pos = torch.arange(40, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = plain.rope(q, k, positions=pos, plan=plan)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b = plain.rope(q, k, positions=pos, plan=plan)
    for step in range(2):
        graph.replay()
        for x, y in zip((q, k), b):
            _check(y, x, pos[None], plan)
        if step == 0:
            assert all(torch.equal(x, y) for x, y in zip(a, b))
            q.neg_()
            pos += 11


def test_in_place_through_the_c_abi():
    from easyfhe import _native, plain

    for dtype, layout in ((torch.bfloat16, "half"), (torch.float32, "interleaved")):
        plan = plain.RopePlan(96, rotary_dim=64, layout=layout)
        q = _x(9, 3, 96, dtype=dtype)
        pos = torch.arange(9, device="cuda")
        want = plain.rope(q, positions=pos, plan=plan)
        part = plain._HEADS.pack(q.data_ptr(), q.data_ptr(), 0, 288, 96, 0, 288, 96, 3)
        _native.call("b2f_rope", part, 1, plain._DTYPES[dtype], 1, 9, 96, 64,
                     int(layout == "interleaved"), pos.data_ptr(), 1, 0, 1,
                     plan.freqs.data_ptr(), plan.factor, 0,
                     torch.cuda.current_stream().cuda_stream)
        assert torch.equal(q, want)


def test_refusals():
    from easyfhe import plain

    plan = plain.RopePlan(64)
    q = _x(3, 2, 64, dtype=torch.float32)
    pos = torch.arange(3, device="cuda")

    def bad(match, q=q, k=None, positions=pos, plan=plan):
        with pytest.raises(ValueError, match=match):
            plain.rope(q, k, positions=positions, plan=plan)

    bad("head", q=q[..., :32])
    bad("CUDA device", q=q.cpu())
    bad("CUDA device", positions=pos.cpu())
    bad("shape", positions=pos[:2])
    bad("int64", positions=pos.float())
    bad("beside", k=q[:2])
    bad("is torch", k=q.half())
    bad("is torch", q=q.int())
    bad("gradient", q=q.clone().requires_grad_())
    bad("plan", plan=None)
    bad("heads", q=q[:, :0])
    assert plain.rope(q, positions=pos, plan=plan).shape == q.shape
