"""4-bit matrix-vector products (csrc/q4.cu) whose result is known without a tolerance."""

from __future__ import annotations

import pytest
import torch

from _plain import q4_weight64

pytestmark = pytest.mark.gpu

INF = float("inf")
# infinities (column: sign) of a row: alone, beside others in 32, 64 and 128 columns, over
# tiles, with one sign and with both
PATTERNS = [{17: 1}, {17: 1, 20: 1}, {17: 1, 50: 1}, {17: -1, 50: 1}, {3: 1, 17: 1, 21: -1, 60: 1},
            {17: 1, 100: 1}, {17: 1, 100: -1, 101: 1}, {64: -1, 65: -1, 127: -1, 255: -1},
            {254: 1, 255: -1}, dict.fromkeys(range(64, 128), 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
@pytest.mark.parametrize("n,rows", [(70, 2), (70, 9), (32011, 1), (32011, 2), (32011, 4)])
def test_infinities_are_the_sum_of_products(dtype, group, zeros, n, rows):
    """A product with an infinity is an infinity or, with a zero weight, NaN, and infinities
    of both signs sum to NaN, in every form that x enters the products in."""
    from easyfhe import plain

    g = torch.Generator(device="cuda").manual_seed(n + rows)
    codes = torch.randint(5, 12, (n, 256), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randn((n, 256 // group), generator=g, device="cuda").to(torch.bfloat16)
    scales[5] = 0.0  # a zero weight whatever its codes
    z = torch.randint(7, 10, scales.shape, generator=g, device="cuda", dtype=torch.uint8) \
        if zeros else None
    w = plain.pack_q4(codes, scales, z, group=group)
    w64 = q4_weight64(codes, scales, z, group)
    clean = torch.randn((rows, 256), generator=g, device="cuda").to(dtype)
    for first in range(0, len(PATTERNS), rows):
        x = clean.clone()
        for r, at in enumerate(PATTERNS[first:first + rows]):
            for column, sign in at.items():
                x[r, column] = sign * INF
        y = plain.q4_matvec(x, w, out_dtype=torch.float32)
        for r in range(rows):
            hit = torch.isinf(x[r])
            if not hit.any():
                assert torch.isfinite(y[r]).all()
                continue
            want = (w64[:, hit] * x[r, hit].double()).sum(1)
            assert torch.equal(torch.isnan(y[r]), torch.isnan(want)), (first, r)
            ok = ~torch.isnan(want)
            assert torch.equal(y[r, ok].double(), want[ok]), (first, r)
    x = clean.clone()
    x[0, 9], x[0, 10] = INF, float("nan")
    assert torch.isnan(plain.q4_matvec(x, w)[0]).all()


@pytest.mark.parametrize("rows", [1, 4])
def test_infinities_in_long_rows(rows):
    """Columns over a cluster's blocks: infinities met by one of them, by several, by none."""
    from easyfhe import plain

    n, k = 28500, 24000
    g = torch.Generator(device="cuda").manual_seed(rows)
    codes = torch.randint(5, 12, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randn((n, -(-k // 128)), generator=g, device="cuda").half()
    w = plain.pack_q4(codes, scales)
    clean = torch.randn((rows, k), generator=g, device="cuda")
    for at in ({}, {5: 1}, {23999: -1}, {5: 1, 23999: -1}, {700: 1, 15000: 1, 20000: 1}):
        x = clean.clone()
        for column, sign in at.items():
            x[rows - 1, column] = sign * INF
        y = plain.q4_matvec(x, w)
        assert torch.isfinite(y[:rows - 1 if at else rows]).all()
        if at:
            cols = torch.tensor(sorted(at), device="cuda")
            w64 = (codes[:, cols].double() - 8) * scales[:, cols // 128].double()
            want = (w64 * x[rows - 1, cols].double()).sum(1)
            assert torch.equal(torch.isnan(y[-1]), torch.isnan(want)), at
            ok = ~torch.isnan(want)
            assert torch.equal(y[-1, ok].double(), want[ok]), at


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,k,group,zeros", [
    (33, 14336, 64, True), (33, 70001, 128, False), (18, 131072, 32, True), (33, 131072, 64, False),
    (1001, 4096, 128, False), (14300, 14336, 128, False), (28500, 4097, 64, True),
    (28500, 24000, 32, False), (14300, 131072, 128, False)])
@pytest.mark.parametrize("rows", [1, 2, 4, 11, 33])
def test_integers_are_exact(dtype, n, k, group, zeros, rows):
    """Integers from -4 to 4 times weights from -15 to 15 under scales of 1: every sum of them
    is an integer below 2^24, which binary32 holds in whatever order it is formed.  A lost or
    doubled column, tile, warp or block shows."""
    from easyfhe import plain

    g = torch.Generator(device="cuda").manual_seed(k + rows)
    codes = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.ones((n, -(-k // group)), device="cuda", dtype=torch.float16)
    z = torch.randint(0, 16, scales.shape, generator=g, device="cuda", dtype=torch.uint8) \
        if zeros else None
    x = torch.randint(-4, 5, (rows, k), generator=g, device="cuda")
    assert 4 * 15 * k < 2 ** 24
    w = plain.pack_q4(codes, scales, z, group=group)
    y = plain.q4_matvec(x.to(dtype), w, out_dtype=torch.float32)
    for n0 in range(0, n, 2000):
        part = slice(n0, n0 + 2000)
        want = x.double() @ q4_weight64(codes[part], scales[part],
                                        None if z is None else z[part], group).T
        assert torch.equal(y[:, part].double(), want), n0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinities_in_rows_and_results_of_16_bits(dtype):
    """As above with y in x's type, from rows that are views."""
    from easyfhe import plain

    n, k = 40001, 320
    g = torch.Generator(device="cuda").manual_seed(3)
    codes = torch.randint(6, 11, (n, k), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.full((n, k // 64), 2.0 ** -6, device="cuda", dtype=torch.float16)
    w = plain.pack_q4(codes, scales, group=64)
    w64 = q4_weight64(codes, scales, None, 64)
    wide = torch.randn((2, 407), generator=g, device="cuda").to(dtype)
    for at in ({300: 1}, {0: -1, 319: -1}, {7: 1, 9: 1, 200: -1}):
        x = wide.clone()[:, 3:323]
        clean = plain.q4_matvec(x, w)
        for column, sign in at.items():
            x[1, column] = sign * INF
        y = plain.q4_matvec(x, w)
        assert y.dtype == dtype and torch.equal(y[0], clean[0])
        cols = torch.tensor(sorted(at), device="cuda")
        want = (w64[:, cols] * x[1, cols].double()).sum(1)
        assert torch.equal(torch.isnan(y[1]), torch.isnan(want)), at
        ok = ~torch.isnan(want)
        assert torch.equal(y[1, ok].double(), want[ok]), at
