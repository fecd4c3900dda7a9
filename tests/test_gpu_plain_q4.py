"""Matrix-vector products with 4-bit weights (csrc/q4.cu) against binary64.

Tolerance: the products are exact (an integer below 16 times a value of at most
24 bits, split exactly); every addition into a binary32 accumulator is off by
at most a step, 2^-23, of a partial sum that is at most S = sum |w x|.  A
product of 16 columns adds once per column and at most K / 16 of them follow
one another, then the groups' scaled sums (2 roundings each) and the warps'
(at most 16) and 4 planes: below (K + 2 groups + 32) 2^-23 S in all, taken in
full.  Rows may be fixed-point numbers, off by at most 2^-30 of the largest of
their 64 columns, times |w|.  The output's own rounding is half a step of
its type."""

from __future__ import annotations

import pytest
import torch

from _plain import half_step, q4_weight64

pytestmark = pytest.mark.gpu


def _weight(n, k, group, zeros, scale_dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.randn((n, groups), generator=g, device="cuda") * 0.02).to(scale_dtype)
    z = torch.randint(0, 16, (n, groups), generator=g, device="cuda", dtype=torch.uint8) \
        if zeros else None
    return codes, scales, z


def _x(rows, k, dtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((rows, k), generator=g, device="cuda", dtype=torch.float64).to(dtype)


def _check(y, x, codes, scales, zeros, group):
    w = q4_weight64(codes, scales, zeros, group)
    k, groups = w.shape[1], scales.shape[1]
    x64 = x.double().reshape(-1, k)
    want, size = x64 @ w.T, x64.abs() @ w.abs().T
    pad = torch.nn.functional.pad(x64.abs(), (0, -k % 64)).unflatten(1, (-1, 64))
    top = pad.amax(2).repeat_interleave(64, dim=1)[:, :k]
    size = size + 2.0 ** -30 / ((k + 2 * groups + 32) * 2.0 ** -23) * (top @ w.abs().T)
    tol = (k + 2 * groups + 32) * 2.0 ** -23 * size + half_step(y.dtype) * want.abs() * 1.01
    if y.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    d = (y.double().reshape(want.shape) - want).abs()
    assert bool((d <= tol).all()), float((d - tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,k,group,zeros,scale", [
    (1, 1, 32, False, torch.bfloat16), (16, 64, 64, True, torch.float16),
    (17, 65, 64, True, torch.bfloat16), (31, 33, 32, True, torch.float16),
    (40, 96, 32, False, torch.bfloat16), (5, 130, 128, True, torch.float16),
    (1001, 1000, 32, True, torch.float16), (250, 1000, 1024, False, torch.bfloat16),
    (300, 4096, 128, False, torch.bfloat16), (64, 14336, 64, True, torch.float16),
    (2500, 576, 192, True, torch.bfloat16), (28500, 200, 64, True, torch.bfloat16),
    (30005, 300, 32, False, torch.float16), (29999, 640, 32, True, torch.bfloat16),
    (20000, 1100, 128, False, torch.bfloat16), (30001, 300, 64, True, torch.float16),
    (18, 70001, 128, False, torch.float16), (33, 131072, 32, True, torch.bfloat16)])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 8, 11, 33])
def test_matvec(dtype, n, k, group, zeros, scale, rows):
    from easyfhe import plain

    codes, scales, z = _weight(n, k, group, zeros, scale)
    w = plain.pack_q4(codes, scales, z, group=group)
    x = _x(rows, k, dtype)
    for out in (None, torch.float32):
        y = plain.q4_matvec(x, w, out_dtype=out)
        assert y.shape == (rows, n) and y.dtype == (dtype if out is None else out)
        _check(y, x, codes, scales, z, group)
        assert torch.equal(y, plain.q4_matvec(x, w, out_dtype=out))


@pytest.mark.parametrize("n,rows", [(128, 2), (128, 7), (16000, 1), (32000, 3), (32000, 9)])
def test_binary32_rows_keep_24_bits(n, rows):
    """Identity-like weights (code 9 at row % columns, 8 elsewhere, scale 1) give x
    back bit for bit: any binary32 number for few weight rows, and those within a
    factor of 2^6 of the largest of their 64 columns for many."""
    from easyfhe import plain

    k = 128
    codes = torch.full((n, k), 8, dtype=torch.uint8, device="cuda")
    codes[torch.arange(n), torch.arange(n) % k] = 9
    w = plain.pack_q4(codes, torch.ones((n, 1), dtype=torch.bfloat16, device="cuda"))
    g = torch.Generator(device="cuda").manual_seed(5)
    x = 1.0 + torch.rand((rows, k), generator=g, device="cuda")
    x *= torch.randint(0, 2, (rows, k), generator=g, device="cuda") * 2 - 1
    if n == k:
        shift = torch.randint(-90, 127, (rows, k), generator=g, device="cuda")
    else:
        shift = torch.randint(-90, 121, (rows, k // 64, 1), generator=g, device="cuda") + \
            torch.randint(0, 7, (rows, k // 64, 64), generator=g, device="cuda")
    x *= torch.exp2(shift.reshape(rows, k).float())
    assert torch.equal(plain.q4_matvec(x, w), x[:, torch.arange(n) % k])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_views_shapes_and_rows_apart(dtype):
    from easyfhe import plain

    codes, scales, z = _weight(70, 200, 64, True, torch.float16)
    w = plain.pack_q4(codes, scales, z, group=64)
    wide = _x(6, 407, dtype)
    for x in (wide[:, :200], wide[:, 3:203], wide[::2, 1:201], wide[:1, 5:205],
              wide[:4, :200].T.contiguous().T, wide[:1, :200].expand(5, 200),
              wide[:, :400].reshape(3, 4, 200), wide[0, 7:207]):
        y = plain.q4_matvec(x, w)
        assert y.shape == (*x.shape[:-1], 70)
        _check(y, x, codes, scales, z, 64)
    assert plain.q4_matvec(wide[:0, :200], w).shape == (0, 70)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,rows", [(50, 5), (32000, 4), (32000, 2)])
def test_infinity_and_nan_stay_in_their_row(dtype, n, rows):
    from easyfhe import plain

    codes, scales, _ = _weight(n, 256, 128, False, torch.bfloat16)
    w = plain.pack_q4(codes, scales)
    x = _x(rows, 256, dtype)
    clean = plain.q4_matvec(x, w)
    x[1, 17] = float("inf")
    if rows > 3:
        x[3, 200] = float("nan")
    y = plain.q4_matvec(x, w)
    for r in range(rows):
        if r == 3:
            assert torch.isnan(y[3]).all()
        elif r != 1:
            assert torch.equal(y[r], clean[r])
    col = codes[:, 17].double() - 8  # inf times a zero weight is NaN, else a signed infinity
    want = (col * scales[:, 0].double()) * float("inf")
    assert torch.equal(torch.isnan(y[1]), torch.isnan(want))
    assert torch.equal(y[1].double()[~torch.isnan(want)], want[~torch.isnan(want)])


def test_rows_past_the_last_one_are_not_written():
    from easyfhe import _native, plain

    codes, scales, _ = _weight(19, 64, 64, False, torch.bfloat16)
    w = plain.pack_q4(codes, scales, group=64)
    x = _x(2, 64, torch.bfloat16)
    y = torch.full((3 * 19 + 5,), 7.0, device="cuda")
    _native.call("b2f_q4_matvec", x.data_ptr(), 3, 64, 2, w.packed.data_ptr(), 3, 0, 19, 64, 64,
                 y.data_ptr(), 1, torch.cuda.current_stream().cuda_stream)
    assert bool((y[2 * 19:] == 7.0).all())
    _check(y[:38].view(2, 19), x, codes, scales, None, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("scale", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,k,group", [(33, 200, 64), (8, 128, 128), (3, 31, 32), (5, 70, 32)])
def test_codes_are_the_formulas(dtype, symmetric, scale, n, k, group):
    """The same roundings in the same order in torch's binary32: equal codes."""
    from easyfhe import plain

    w = _x(n, k, dtype, seed=4)
    w[0, :group] = 0.0  # an empty range
    w[1, :] = w[1].abs()  # one sign only
    codes, scales, zeros = plain.q4_codes(w, group=group, symmetric=symmetric, scale_dtype=scale)
    groups = -(-k // group)
    for g in range(groups):
        c = slice(g * group, min((g + 1) * group, k))
        x = w[:, c].float()
        lo, hi = x.amin(1).clamp(max=0), x.amax(1).clamp(min=0)
        s = (torch.maximum(hi, -lo) / 7 if symmetric else (hi - lo) / 15).to(scale)
        sf = s.float()
        safe = torch.where(sf > 0, sf, 1.0)
        z = torch.full_like(sf, 8.0) if symmetric else \
            torch.where(sf > 0, (-lo / safe).round().clamp(0, 15), 0.0)
        q = torch.where(sf[:, None] > 0, (x / safe[:, None]).round() + z[:, None], z[:, None])
        assert torch.equal(scales[:, g], s)
        assert torch.equal(codes[:, c], q.clamp(0, 15).to(torch.uint8))
        assert (zeros is None) == symmetric
        if zeros is not None:
            assert torch.equal(zeros[:, g], z.to(torch.uint8))


def test_quantized_product_is_near_the_weight():
    """A weight rounds to within half a scale of itself (its extreme, on the
    symmetric grid, to the scale's own rounding), and the product follows."""
    from easyfhe import plain

    w = _x(64, 512, torch.float32, seed=9)
    x = _x(2, 512, torch.float32)
    codes, scales, zeros = plain.q4_codes(w)
    w64 = q4_weight64(codes, scales, zeros, 128)
    step = scales.double().repeat_interleave(128, dim=1)
    assert bool(((w64 - w.double()).abs() <= step * (0.5 + 8 * half_step(torch.bfloat16))).all())
    _check(plain.q4_matvec(x, plain.quantize_q4(w)), x, codes, scales, zeros, 128)


def test_offsets_past_32_bits():
    """More than 2^32 codes: the last rows, in the last records, are the formula's."""
    from easyfhe import plain

    n, k = (1 << 20) + 21, 4096
    g = torch.Generator(device="cuda").manual_seed(2)
    codes = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.rand((n, 1), generator=g, device="cuda").half()
    w = plain.pack_q4(codes, scales, group=k)
    last = slice(n - 50, n)
    for dtype, rows in ((torch.float32, 2), (torch.bfloat16, 9)):
        x = _x(rows, k, dtype)
        _check(plain.q4_matvec(x, w)[:, last], x, codes[last], scales[last], None, k)


def test_capture_replays_on_new_rows():
    from easyfhe import plain

    codes, scales, z = _weight(100, 320, 32, True, torch.bfloat16)
    w = plain.pack_q4(codes, scales, z, group=32)
    x = _x(3, 320, torch.float16)
    plain.q4_matvec(x, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = plain.q4_matvec(x, w)
    for seed in (2, 3):
        x.copy_(_x(3, 320, torch.float16, seed=seed))
        graph.replay()
        _check(y, x, codes, scales, z, 32)


def test_refusals():
    from easyfhe import plain

    codes, scales, z = _weight(20, 64, 64, True, torch.bfloat16)
    w = plain.pack_q4(codes, scales, z, group=64)
    x = _x(1, 64, torch.bfloat16)
    bad = pytest.raises(ValueError)
    with bad:
        plain.pack_q4(codes + 1, scales, z, group=64)  # a code of 16
    with bad:
        plain.pack_q4(codes, scales.float(), z, group=64)
    with bad:
        plain.pack_q4(codes, scales, z, group=32)  # scales of another group
    with bad:
        plain.pack_q4(codes, scales, z.int(), group=64)
    with bad:
        plain.pack_q4(codes, scales, z.cpu(), group=64)
    with bad:
        plain.q4_codes(x.double())
    with bad:
        plain.q4_codes(x, group=48)
    with bad:
        plain.q4_codes(x, scale_dtype=torch.float32)
    with bad:
        plain.q4_matvec(x[:, :32], w)
    with bad:
        plain.q4_matvec(x.double(), w)
    with bad:
        plain.q4_matvec(x.cpu(), w)
    with bad:
        plain.q4_matvec(x, w, out_dtype=torch.float16)
    with bad:
        plain.q4_matvec(x.expand(1025, 64), w)
    with bad:
        plain.q4_matvec(x.clone().requires_grad_(), w)
    with torch.no_grad():
        assert plain.q4_matvec(x.clone().requires_grad_(), w).shape == (1, 20)
