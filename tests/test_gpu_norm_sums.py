"""Layer normalisation where sums lose most: rows far from zero, long rows, many rows (GPU).

u = 2^-24 is half a step of fp32, h_t = finfo(t).eps / 2 half a step of the stored type."""

import pytest
import torch

import sparse_embedding_b200 as se

pytestmark = pytest.mark.gpu

U = 2.0**-24
DIMS = [8, 24, 35, 64, 96, 129, 300, 301, 512, 701, 1032, 1037, 4096, 9001]  # every layout of rows


def half(t):
    return torch.finfo(t).eps / 2


def within(got, want, tol, what):
    d = (got.double() - want).abs()
    assert got.shape == want.shape and bool((d <= tol).all()), (what, float((d / tol).max()))


@pytest.mark.parametrize("dt, offset", [(torch.float32, 1000.0), (torch.float16, 200.0), (torch.bfloat16, 64.0)])
@pytest.mark.parametrize("dim", DIMS)
def test_backward_of_rows_far_from_zero(dim, dt, offset):
    """With the mean that is given, h = (x - mean) rstd has two roundings, 2 u |h|, however far the row lies from zero.
    A column's sum of three rows rounds at most three times more (a product is exact within its fused add; zeros add
    without rounding): 6 u sum|g h| and second-order terms. dx as in the other tests, with |h| in place of the sizes
    of x and mean."""
    gen = torch.Generator(device="cuda").manual_seed(dim)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    x, g, w = (r(3, dim) + offset).to(dt), r(3, dim).to(dt), 1 + 0.1 * r(dim)
    _, mean, rstd = se.layer_norm(x, w, return_stats=True)
    dx, dw, db = se.layer_norm_backward(g, x, mean, rstd, w)
    X, G, W, m, q = x.double(), g.double(), w.double(), mean.double()[:, None], rstd.double()[:, None]
    h, wg = (X - m) * q, G * W
    within(dw, (G * h).sum(0), 6.1 * U * (G * h).abs().sum(0) + 1e-30, "dweight")
    within(db, G.sum(0), 3.1 * U * G.abs().sum(0) + 1e-30, "dbias")
    DX = q * (wg - wg.mean(1, keepdim=True) - h * (wg * h).mean(1, keepdim=True))
    size = wg.abs().amax(1, keepdim=True) + h.abs().amax(1, keepdim=True) * (wg * h).abs().mean(1, keepdim=True)
    within(dx, DX, 100 * U * q * size + half(dt) * (DX.abs() + torch.finfo(dt).tiny), "dx")


# Rows enough that every block fills each buffer of its ring several times: vectors with one, two and four loads a
# thread, single values with 16 and 32, a block per row in both; without gaps, with a gap, from an odd address.
RING = [(200_000, 128, torch.float32, 0, 0), (262_144, 256, torch.bfloat16, 0, 0), (100_000, 256, torch.float32, 0, 0),
        (100_000, 512, torch.bfloat16, 0, 0), (100_000, 512, torch.float32, 4, 0), (60_000, 1000, torch.float16, 8, 0),
        (60_000, 301, torch.float32, 0, 1), (120_000, 301, torch.bfloat16, 2, 3), (60_000, 517, torch.float32, 0, 0),
        (60_000, 1001, torch.bfloat16, 0, 1), (60_000, 1037, torch.float32, 3, 1), (90_000, 1037, torch.bfloat16, 0, 0),
        (60_000, 1032, torch.float32, 0, 0), (65_536, 2048, torch.bfloat16, 0, 0), (33_000, 4096, torch.bfloat16, 0, 0),
        (33_000, 4096, torch.float32, 0, 0), (33_000, 4104, torch.float16, 8, 0), (20_000, 8192, torch.bfloat16, 0, 0),
        # more rows than one launch takes
        (1_300_000, 128, torch.float32, 0, 0), (700_000, 301, torch.bfloat16, 2, 3), (3_000_000, 33, torch.bfloat16, 0, 1),
        (160_000, 1037, torch.bfloat16, 0, 0), (160_000, 1032, torch.bfloat16, 8, 0)]


def laid_out(values, pad, offset, dt):
    rows, dim = values.shape
    flat = torch.zeros(rows * (dim + pad) + offset, dtype=dt, device="cuda")
    t = flat[offset:].view(rows, dim + pad)[:, :dim]
    t.copy_(values)
    return t


@pytest.mark.parametrize("rows, dim, dt, pad, offset", RING)
def test_many_tiles_a_block(rows, dim, dt, pad, offset):
    """x and grad are whole numbers from -3 to 3 and mean = 0, rstd = 1 are given, so that h = x and every sum over
    rows stays below 2^24: dweight and dbias are exact, whatever the order of the sums. So are a row's sums; with
    weight 1 dx is g - sum g / D - x sum(g x) / D: two quotients, each rounded twice (1 / D and the product), and two fused
    adds: 4 u (|g| + |mean g| + |x mean(g x)|) before the result's own rounding. y: means of whole numbers, tolerance as
    derived for the other tests (|x| <= 3). Calls repeat bit by bit."""
    gen = torch.Generator(device="cuda").manual_seed(rows + dim)
    ints = lambda: torch.randint(-3, 4, (rows, dim), generator=gen, device="cuda", dtype=torch.int8)  # noqa: E731
    x, g = laid_out(ints(), pad, offset, dt), laid_out(ints(), pad, offset, dt)
    w, zero, one = torch.ones(dim, device="cuda"), torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    first = se.layer_norm_backward(g, x, zero, one, w)
    X, G = x.double(), g.double()
    assert torch.equal(first[1].double(), (G * X).sum(0)) and torch.equal(first[2].double(), G.sum(0))
    c0, c1 = G.mean(1, keepdim=True), X * (G * X).mean(1, keepdim=True)
    DX = G - c0 - c1
    within(first[0], DX, 4 * U * (G.abs() + c0.abs() + c1.abs()) + half(dt) * DX.abs(), "dx")
    y = se.layer_norm(x, w)
    m = X.mean(1, keepdim=True)
    r = 1 / ((X - m).square().mean(1, keepdim=True) + 1e-5).sqrt()
    Y = (X - m) * r
    within(y, Y, U * 100 * 3 * r + half(dt) * Y.abs(), "y")
    del X, G, DX, Y, c1
    for _ in range(10):
        assert all(torch.equal(p, q) for p, q in zip(se.layer_norm_backward(g, x, zero, one, w), first))
        assert torch.equal(se.layer_norm(x, w), y)


# Equal values whose rounding in a long chain of adds goes one way: c lies 0.49 of a step of [256, 512) above the grids of
# [256, 512), [512, 1024) and [1024, 2048).
BIASED = (3276 + 0.49) * 2.0**-15


@pytest.mark.parametrize("dim", [1 << 22, (1 << 23) + 5])
def test_one_very_long_row(dim):
    """A thread's sum is pieces of 64, those in pieces of 64, and at most 5 of those; then 10 levels over the block: 64 + 64 +
    5 + 10 roundings and the quotient's, 150 u of equal values' sum. (One chain of dim / 512 adds is 900 u off and more.)"""
    x = torch.full((1, dim), BIASED, device="cuda")
    c = float(x[0, 0].double())
    _, mean, rstd = se.layer_norm(x, eps=1.0, return_stats=True)
    assert abs(float(mean) - c) <= 150 * U * c and abs(float(rstd) - 1.0) <= 4 * U
    # with x = 1, mean = 0 and rstd = 1 both sums are of equal values: dx = g (1 - 1 - 1)
    one = torch.ones(1, device="cuda")
    dx, _, _ = se.layer_norm_backward(x, torch.ones_like(x), torch.zeros_like(one), one)
    assert float((dx.double() + c).abs().max()) <= (2 * 150 + 4) * U * c


def test_columns_of_many_long_rows():
    """64 splits of the rows: as above, with 64 more adds of the splits."""
    rows, dim = 400_000, 8200
    x = torch.ones(rows, dim, dtype=torch.bfloat16, device="cuda")
    r = torch.full((rows,), BIASED, device="cuda")
    dw = se.layer_norm_backward(x, x, torch.zeros_like(r), r, torch.ones(dim, device="cuda"))[1]
    want = rows * float(r[0].double())
    assert float((dw.double() - want).abs().max()) <= (64 + 64 + 2 + 64) * U * want


def test_columns_of_very_many_rows():
    """A thread adds 512 rows at most, then come 5 levels of a warp, 8 warps, and the launches' blocks in pieces of 64
    by 32 threads: 512 + 5 + 8 + 64 + 64 + 32 roundings at most. (One chain of all rows of a block, 6,700 here, is
    1,200 u off and more.)"""
    rows, dim = 6_000_000, 1032
    x = torch.ones(rows, dim, dtype=torch.bfloat16, device="cuda")
    r = torch.full((rows,), BIASED, device="cuda")
    dw = se.layer_norm_backward(x, x, torch.zeros_like(r), r, torch.ones(dim, device="cuda"))[1]
    want = rows * float(r[0].double())
    assert float((dw.double() - want).abs().max()) <= (512 + 5 + 8 + 64 + 64 + 32) * U * want
