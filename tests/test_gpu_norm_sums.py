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
