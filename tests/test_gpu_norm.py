"""Layer normalisation, forward and backward, against the formulas in 64 bits (GPU).

Tolerances. u = 2^-24 is half a step of fp32, h_t = finfo(t).eps / 2 half a step
of the stored type. A row's sums pass at most 16 adds per thread (40 for rows
beyond 8,192 values) and 10 levels of a tree, under 64 roundings: a mean is off
by at most 64 u max|x|, a variance by 64 u of itself plus the squared error of
the mean, 1 / sqrt by half of that and 2 u. So y is off by at most
u (100 max|x| r |w| + 2 |b|) + h_t |y|, dx by u r 100 (max|q| + max|k| mean|q k|)
+ h_t |dx| with k = (|x| + |mean|) r. A column's sum passes at most 128 adds
(rows per thread, the block's warps, every 16th block, 16) at these sizes:
u 140 sum|g k| + h_t |dw|. Values below the type's normal range round to its
smallest step instead of relatively: h_t finfo.tiny more."""

import ctypes as C

import pytest
import torch

import sparse_embedding_b200 as se
from sparse_embedding_b200 import _native as N
from sparse_embedding_b200 import torch_ops

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]
SHAPES = [(1, 1), (1, 8), (3, 2), (5, 7), (1, 96), (26, 128), (257, 64), (1000, 33), (4100, 96), (63, 129), (130, 1037),
          (64, 512), (9, 1024), (17, 1032), (11, 2048), (7, 4096), (5, 8192), (3, 8191), (2, 8200), (3, 20001)]


def half(t):
    return torch.finfo(t).eps / 2


def inputs(rows, dim, dt, pt, pad=0, offset=0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + rows * 31 + dim)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    out = []
    for scale in (1.0, 0.01):
        v = r(rows, dim) * scale * (0.25 + 2 * torch.rand(rows, 1, generator=g, device="cuda"))
        if scale == 1.0:
            v = v + r(dim)
        flat = torch.zeros(rows * (dim + pad) + offset, dtype=dt, device="cuda")
        t = flat[offset:].view(rows, dim + pad)[:, :dim]
        t.copy_(v)
        out.append(t)
    return out[0], out[1], (1 + 0.1 * r(dim)).to(pt), (0.1 * r(dim)).to(pt)


def within(got, want, tol, what):
    d = (got.double() - want).abs()
    assert got.shape == want.shape and bool((d <= tol).all()), (what, float((d / tol).max()))


def check(x, g, w, b, eps=1e-5):
    dt = x.dtype
    tiny = half(dt) * torch.finfo(dt).tiny
    y, mean, rstd = se.layer_norm(x, w, b, eps=eps, return_stats=True)
    assert y.dtype == dt and mean.dtype == rstd.dtype == torch.float32 and y.is_contiguous()
    X, G = x.double(), g.double()
    W = torch.ones(x.shape[-1], dtype=torch.float64, device="cuda") if w is None else w.double()
    B = torch.zeros_like(W) if b is None else b.double()
    m = X.mean(-1, keepdim=True)
    r = 1 / ((X - m).square().mean(-1, keepdim=True) + eps).sqrt()
    big = X.abs().amax(-1, keepdim=True)
    within(mean, m[:, 0], 64 * U * big[:, 0], "mean")
    within(rstd, r[:, 0], r[:, 0] * U * (40 + 2 * (64 * U * (big * r) ** 2)[:, 0] * 64), "rstd")
    Y = (X - m) * r * W + B
    within(y, Y, U * (100 * big * r * W.abs() + 2 * B.abs()) + half(dt) * Y.abs() + tiny, "y")
    dx, dw, db = se.layer_norm_backward(g, x, mean, rstd, w, with_bias=b is not None)
    m, r = mean.double()[:, None], rstd.double()[:, None]
    h, k, q = (X - m) * r, (X.abs() + m.abs()) * r, G * W
    DX = r * (q - q.mean(-1, keepdim=True) - h * (q * h).mean(-1, keepdim=True))
    tol = U * 100 * r * (q.abs().amax(-1, keepdim=True) + k.amax(-1, keepdim=True) * (q * k).abs().mean(-1, keepdim=True))
    within(dx, DX, tol + half(dt) * DX.abs() + tiny, "dx")
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    for got, want, size in ((dw, (G * h).sum(0), (G * k).abs().sum(0)), (db, G.sum(0), G.abs().sum(0))):
        if got is not None:
            pt = got.dtype
            within(got, want, U * 140 * size + half(pt) * (want.abs() + torch.finfo(pt).tiny), "columns")


@pytest.mark.parametrize("dt, pt", TYPES)
@pytest.mark.parametrize("rows, dim", SHAPES)
def test_against_64_bits(rows, dim, dt, pt):
    check(*inputs(rows, dim, dt, pt))


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pad, offset", [(8, 0), (3, 0), (0, 1), (5, 3), (64, 8)])
@pytest.mark.parametrize("rows, dim", [(1, 64), (37, 64), (50, 100), (19, 1037), (6, 2048)])
def test_strides_and_alignment(rows, dim, pad, offset, dt):
    x, g, w, b = inputs(rows, dim, dt, torch.float32, pad, offset)
    check(x, g, w, b)
    check(x, g.contiguous(), w, None)
    check(x.contiguous(), g, None, None)


def test_many_rows_and_leading_axes():
    x, g, w, b = inputs(70_001, 48, torch.float32, torch.float32)
    y, mean, rstd = se.layer_norm(x, w, b, return_stats=True)
    X = x.double()
    Y = (X - X.mean(1, keepdim=True)) / (X.var(1, keepdim=True, correction=0) + 1e-5).sqrt() * w + b
    assert float((y - Y).abs().max()) < 1e-4 and bool(torch.isfinite(rstd).all())
    y3 = se.layer_norm(x[:70_000].view(100, 700, 48), w, b)
    assert y3.shape == (100, 700, 48) and torch.equal(y3.view(-1, 48), y[:70_000])
    one = se.layer_norm(x[5], w, b, return_stats=True)
    assert one[0].shape == (48,) and one[1].shape == () and torch.equal(one[0], y[5])


@pytest.mark.parametrize("dim", [16, 1, 300, 9000])
def test_no_rows(dim):
    x = torch.empty(0, dim, device="cuda")
    w = torch.ones(dim, device="cuda")
    y, mean, rstd = se.layer_norm(x, w, w, return_stats=True)
    assert y.shape == (0, dim) and mean.shape == rstd.shape == (0,)
    dx, dw, db = se.layer_norm_backward(x, x, mean, rstd, w)
    assert dx.shape == (0, dim) and not dw.any() and not db.any() and dw.shape == db.shape == (dim,)


@pytest.mark.parametrize("dim", [24, 129, 2048, 9001])
def test_constant_infinite_and_nan_rows(dim):
    x, g, w, b = inputs(6, dim, torch.float32, torch.float32)
    x[1] = 3.0
    x[2] = 0.0
    x[3, dim // 2] = float("inf")
    x[4, 0] = float("nan")
    y, mean, rstd = se.layer_norm(x, w, b, return_stats=True)
    # a constant row has no deviation: its mean is exact to 64 u, and eps bounds 1 / sqrt(var + eps)
    assert float((y[1] - b).abs().max()) <= 64 * U * 3 / 1e-5**0.5 * float(w.abs().max()) and torch.equal(y[2], b)
    assert torch.isnan(y[3:5]).all() and torch.isfinite(y[[0, 1, 2, 5]]).all()
    assert float(mean[3]) == float("inf") and torch.isnan(mean[4]) and torch.isnan(rstd[3:5]).all()
    dx, dw, db = se.layer_norm_backward(g, x, mean, rstd, w)
    assert torch.isnan(dx[3:5]).all() and torch.isfinite(dx[[0, 1, 2, 5]]).all()
    assert torch.isnan(dw).all() and torch.isfinite(db).all()
    zero = se.layer_norm(x, w, b, eps=0.0)
    assert torch.isnan(zero[2]).all() and torch.isfinite(zero[[0, 5]]).all()


def test_large_and_offset_values():
    x = torch.randn(33, 256, device="cuda") + 1000.0  # a difference of two sums would lose the variance here
    w = torch.ones(256, device="cuda")
    check(x, torch.randn_like(x), w, w)
    check(x * 1e12, torch.randn_like(x), w, w)
    check(x * 1e-12, torch.randn_like(x) * 1e-3, w, w)


@pytest.mark.parametrize("rows, dim", [(4100, 96), (300, 1037), (500, 4096), (9, 20001)])
def test_equal_calls_give_equal_bits(rows, dim):
    x, g, w, b = inputs(rows, dim, torch.bfloat16, torch.float32)
    y, mean, rstd = se.layer_norm(x, w, b, return_stats=True)
    first = se.layer_norm_backward(g, x, mean, rstd, w)
    for _ in range(3):
        assert torch.equal(se.layer_norm(x, w, b), y)
        assert all(torch.equal(p, q) for p, q in zip(se.layer_norm_backward(g, x, mean, rstd, w), first))


def test_gradients_against_differences():
    # central differences in 64 bits of the 64-bit formula would only test the formula: these difference the kernel's
    # own y. A step d leaves d^2 |f'''| / 6 and roundings of 100 u max|x| r / d per value of y, here below 2e-3.
    x, g, w, b = inputs(3, 10, torch.float32, torch.float32)
    g = g * 100
    _, mean, rstd = se.layer_norm(x, w, b, return_stats=True)
    dx, dw, db = se.layer_norm_backward(g, x, mean, rstd, w)
    d = 2.0**-7
    loss = lambda *a: float((se.layer_norm(*a).double() * g.double()).sum())  # noqa: E731
    for t, grad in ((x, dx), (w, dw), (b, db)):
        for i in range(t.numel()):
            args = [[x, w, b], [x, w, b]]
            for a, sign in zip(args, (1, -1)):
                moved = t.clone()
                moved.view(-1)[i] += sign * d
                a[[id(v) for v in (x, w, b)].index(id(t))] = moved
            diff = (loss(*args[0]) - loss(*args[1])) / (2 * d)
            assert abs(diff - float(grad.view(-1)[i])) <= 5e-3 * max(1.0, float(grad.abs().max()))


def test_autograd_and_broadcast_gradients():
    x, g, w, b = inputs(40, 72, torch.float32, torch.float32)
    x, w, b = (t.clone().requires_grad_() for t in (x, w, b))
    y = torch_ops.layer_norm(x, w, b)
    y.backward(g)
    with torch.no_grad():
        _, mean, rstd = se.layer_norm(x, w, b, return_stats=True)
        want = se.layer_norm_backward(g, x, mean, rstd, w)
    for t, v in zip((x, w, b), want):
        assert torch.equal(t.grad, v)
    x.grad = None
    torch_ops.layer_norm(x, w, b).sum().backward()  # a gradient of stride 0
    ones = se.layer_norm_backward(torch.ones_like(x), x.detach(), mean, rstd, w.detach())
    assert torch.equal(x.grad, ones[0])
    # the same weight twice in one graph: its gradients add; rows in another order are copied first
    w.grad = None
    wide = torch.randn(4, 72, 5, device="cuda", requires_grad=True)
    (torch_ops.layer_norm(wide.transpose(1, 2), w, b) + torch_ops.layer_norm(wide.transpose(1, 2), w)).sum().backward()
    assert wide.grad.shape == wide.shape and w.grad.shape == w.shape
    with torch.no_grad():
        t = wide.transpose(1, 2).contiguous()
        _, mean, rstd = se.layer_norm(t, w, b, return_stats=True)
        one = se.layer_norm_backward(torch.ones_like(t), t, mean, rstd, w)
    assert torch.equal(w.grad, 2 * one[1]) and torch.equal(wide.grad, 2 * one[0].transpose(1, 2))


def test_rows_behind_the_last_are_left_alone():
    rows, dim = 5, 37
    x, g, w, b = inputs(rows, dim, torch.float16, torch.float16)
    big = [torch.full((rows + 2, dim), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    stats = [torch.full((rows + 2,), 7.0, device="cuda") for _ in range(2)]
    cols = [torch.full((dim + 5,), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    st = torch.cuda.current_stream().cuda_stream
    L = N.lib()
    N.check(L.se_layer_norm(1, 1, x.data_ptr(), rows, dim, dim, w.data_ptr(), b.data_ptr(), 1e-5, big[0].data_ptr(),
                            stats[0].data_ptr(), stats[1].data_ptr(), 0, st))
    size = C.c_size_t()
    N.check(L.se_layer_norm_backward_workspace(rows, dim, 0, C.byref(size)))
    work = torch.full((size.value + 64,), 9, dtype=torch.uint8, device="cuda")
    N.check(L.se_layer_norm_backward(1, 1, g.data_ptr(), dim, x.data_ptr(), dim, rows, dim, stats[0].data_ptr(),
                                     stats[1].data_ptr(), w.data_ptr(), big[1].data_ptr(), cols[0].data_ptr(),
                                     cols[1].data_ptr(), work.data_ptr(), size.value, 0, st))
    torch.cuda.synchronize()
    assert all(bool((t[rows:] == 7.0).all()) for t in big + stats) and all(bool((t[dim:] == 7.0).all()) for t in cols)
    assert bool((work[size.value:] == 9).all())
    assert torch.equal(big[0][:rows], se.layer_norm(x, w, b))
    # too small a workspace is refused before anything runs
    assert L.se_layer_norm_backward(1, 1, g.data_ptr(), dim, x.data_ptr(), dim, rows, dim, stats[0].data_ptr(),
                                    stats[1].data_ptr(), w.data_ptr(), big[1].data_ptr(), cols[0].data_ptr(), None,
                                    work.data_ptr(), 4, 0, st) == N.SE_ERR_INVALID_ARGUMENT


def test_streams_and_graphs():
    x, g, w, b = inputs(2000, 256, torch.float32, torch.float32)
    y0, mean, rstd = se.layer_norm(x, w, b, return_stats=True)
    want = [y0, *se.layer_norm_backward(g, x, mean, rstd, w)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([se.layer_norm(x, w, b), *se.layer_norm_backward(g, x, mean, rstd, w)])
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for r in got for p, q in zip(r, want))
    # two graphs captured on one stream and replayed at the same time have workspaces of their own
    xs, graphs, outs = [x.clone(), x.clone() * 3], [], []
    side = torch.cuda.Stream()
    for t in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y, m, r = se.layer_norm(t, w, b, return_stats=True)
            outs.append([y, *se.layer_norm_backward(g, t, m, r, w)])
        graphs.append(graph)
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for t, o in zip(xs, outs):
        y, m, r = se.layer_norm(t, w, b, return_stats=True)
        assert all(torch.equal(p, q) for p, q in zip(o, [y, *se.layer_norm_backward(g, t, m, r, w)]))


def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    s = torch.ones(4, device="cuda")
    for call, msg in [
        (lambda: se.layer_norm(x.double()), "unsupported x dtype"),
        (lambda: se.layer_norm(x.t()), "rows at one stride"),
        (lambda: se.layer_norm(x, w[:7]), "weight must be a contiguous 1D tensor of dim values"),
        (lambda: se.layer_norm(x, torch.ones(16, device="cuda")[::2]), "weight must be a contiguous"),
        (lambda: se.layer_norm(x, w.cpu()), "weight must be a CUDA tensor"),
        (lambda: se.layer_norm(x, w.half()), "weight must have x's dtype or float32"),
        (lambda: se.layer_norm(x.half(), w.half(), w), "same dtype"),
        (lambda: se.layer_norm(x, None, w), "bias needs a weight"),
        (lambda: se.layer_norm(x, eps=-1.0), "eps must be finite"),
        (lambda: se.layer_norm_backward(x.half(), x, s, s), "x's shape and dtype"),
        (lambda: se.layer_norm_backward(x[:3], x, s, s), "x's shape and dtype"),
        (lambda: se.layer_norm_backward(x, x, s[:3], s), "mean must be a contiguous float32"),
        (lambda: se.layer_norm_backward(x, x, s, s.half()), "rstd must be a contiguous float32"),
        (lambda: se.layer_norm_backward(torch.zeros(8, device="cuda").expand(4, 8), x, s, s), "grad must be rows"),
    ]:
        with pytest.raises(ValueError, match=msg):
            call()
    host = torch.zeros(4, 8)
    rc = N.lib().se_layer_norm(0, 0, host.data_ptr(), 4, 8, 8, None, None, 1e-5, x.data_ptr(), None, None, 0, None)
    assert rc == N.SE_ERR_INVALID_ARGUMENT and b"x must be device memory" in N.lib().se_last_error()


def test_more_than_2_31_values():
    rows, dim = 530_000, 4096
    x = torch.empty(rows, dim, dtype=torch.bfloat16, device="cuda")
    x[: rows - 100] = 1.0
    tail = torch.randn(100, dim, device="cuda").bfloat16()
    x[rows - 100 :] = tail
    w = torch.linspace(0.5, 1.5, dim, device="cuda")
    y, mean, rstd = se.layer_norm(x, w, return_stats=True)
    assert torch.equal(y[rows - 100 :], se.layer_norm(tail, w)) and not y[rows - 200].any()
    del y
    dx = se.layer_norm_backward(x, x, mean, rstd, w)[0]
    want = se.layer_norm_backward(tail, tail, mean[rows - 100 :], rstd[rows - 100 :], w)[0]
    assert torch.equal(dx[rows - 100 :], want)


def test_calls_from_two_threads():
    import threading

    x, g, w, b = inputs(3000, 320, torch.bfloat16, torch.float32)
    y0, mean, rstd = se.layer_norm(x, w, b, return_stats=True)
    want = se.layer_norm_backward(g, x, mean, rstd, w)
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got = se.layer_norm_backward(g, x, mean, rstd, w)
                if not all(torch.equal(p, q) for p, q in zip(got, want)) or not torch.equal(se.layer_norm(x, w, b), y0):
                    bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim, pad, offset", [(35, 0, 0), (35, 0, 1), (129, 2, 3), (1037, 0, 5), (513, 9, 1)])
def test_neighbours_of_unaligned_rows(dim, pad, offset, dt):
    # rows are copied in whole 16-byte units: what lies around the matrix, NaN here, must not enter it
    rows = 400
    flat = torch.full((offset + rows * (dim + pad) + 64,), float("nan"), dtype=dt, device="cuda")
    x = flat[offset : offset + rows * (dim + pad)].view(rows, dim + pad)[:, :dim]
    x.copy_(torch.randn(rows, dim, device="cuda"))
    w = torch.ones(dim, dtype=dt, device="cuda")
    y, mean, rstd = se.layer_norm(x, w, return_stats=True)
    assert torch.equal(y, se.layer_norm(x.contiguous(), w)) and torch.isfinite(y).all()
    dx, dw, db = se.layer_norm_backward(x, x, mean, rstd, w)
    assert all(torch.isfinite(t).all() for t in (dx, dw, db))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad", [0, 1, 8])
@pytest.mark.parametrize("dim", [4, 5, 8, 9, 16, 17, 24, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513,
                                 1023, 1024, 1025, 1279])
def test_both_sides_of_each_layout(dim, pad, dt):
    # 301 rows: whole tiles and a last one that ends inside
    check(*inputs(301, dim, dt, torch.float32, pad, 0))


@pytest.mark.parametrize("dim", [1, 5, 12, 20, 33, 40, 65, 104, 129, 300, 600, 1030])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_rows_of_a_warp_do_not_mix(dim, pad):
    x, g, w, b = inputs(40, dim, torch.float32, torch.float32, pad)
    x[7, dim - 1] = float("nan")
    x[18, 0] = float("inf")
    g[30, dim // 2] = float("nan")
    y, mean, rstd = se.layer_norm(x, w, b, return_stats=True)
    dx, dw, db = se.layer_norm_backward(g, x, mean, rstd, w)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[7, 18]] = True
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all() and torch.isfinite(mean[~bad]).all()
    bad[30] = True
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()
    want = torch.zeros(dim, dtype=torch.bool, device="cuda")
    want[dim // 2] = True
    assert torch.equal(torch.isnan(db), want) and torch.isnan(dw).all()
