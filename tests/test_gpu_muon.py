"""Newton-Schulz orthogonalisation and the Muon step against the formulas in 64 bits (GPU).

Tolerances, relative to the norm of the result. A step's map of a singular value,
f(s) = 3.4445 s - 4.775 s^3 + 2.0315 s^5, has |f'| <= 1.6 where the values end up, and
errors of small values grow like the values themselves. Five steps have 15 products, whose
independent relative errors e therefore leave about e sqrt(15) 3.5 = 13.6 e.
 * bf16: f16 operands, rounded by 2^-11 at most and 2^-11 / sqrt(3) in the mean: 13.6 x
   2.8e-4 = 3.9e-3, and 2^-8 for the result's own rounding: 2^-7.
 * fp32, fp16: operands of 22 bits; a sum loses at most 2^-23 in each of the 16 matrix
   instructions between two flushes, half of that in the mean: e = 2^-20, so 2^-16, and
   for fp16 2^-11 more.
A single value may be off by 8 times that, relative to the root mean square. Where a few
directions of the update tower above the rest there is more: X is held as two f16 values,
which rounds entry (i, j) of each X_k by at most 2^-22 |x_ij|. That error has parts along
small singular values, which grow by up to 3.4445 in every step still to come, so a value may
be off by another (3.4445^5 + ... + 3.4445) 2^-22 = 684 x 2^-22 of the largest entry of X_0,
and the whole by that of X_0's norm, which is 1 (fp32 operations in place of the kernel's are
off by a quarter of this: their roundings are 2^-24)."""

import math

import pytest
import torch

import sparse_embedding_b200 as se
from sparse_embedding_b200 import torch_ops

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TOL = {F32: 2.0**-16, F16: 2.0**-16 + 2.0**-11, BF16: 2.0**-7}
SHAPES = [(1, 1), (1, 7), (9, 1), (16, 16), (33, 65), (64, 64), (127, 129), (128, 128), (100, 300), (300, 100),
          (257, 256), (513, 1000), (1000, 517), (640, 640), (1300, 200), (384, 2051)]


def half(t):
    return torch.finfo(t).eps / 2


def matrix(*shape, seed=0, kind="falling"):
    g = torch.Generator(device="cuda").manual_seed(seed * 977 + shape[-1] * 31 + shape[-2])
    r = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float64)  # noqa: E731
    *lead, m, n = shape
    if kind == "flat":
        return r(*shape)
    if kind == "identity":
        return torch.eye(m, n, device="cuda", dtype=torch.float64).expand(shape) + 0.1 * r(*shape) / max(m, n) ** 0.5
    k = min(m, n, 8)
    low = (r(*lead, m, k) / torch.arange(1, k + 1, device="cuda")) @ r(*lead, k, n)
    return 1e-2 * (low + {"falling": 0.3, "strong": 1e-3}[kind] * r(*shape))


def exact(u, steps=5, eps=1e-7):
    x = u.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    wide = x.shape[-2] <= x.shape[-1]
    for _ in range(steps):
        a = x @ x.mT if wide else x.mT @ x
        p = -4.7750 * a + 2.0315 * (a @ a)
        x = 3.4445 * x + (p @ x if wide else x @ p)
    return x


def near(got, want, tol, what="", update=None):
    assert got.shape == want.shape and bool(torch.isfinite(got).all()), what
    d = (got.double() - want).flatten(0, -1)
    norm = float(want.norm())
    noise = 684 * 2.0**-22
    assert float(d.norm()) <= tol * norm + (0.0 if update is None else noise), (what, float(d.norm()) / norm)
    most = 8 * tol * max(norm / want.numel() ** 0.5, float(want.abs().max()) / 8)
    if update is not None:
        most += noise * float(update.double().abs().max() / update.double().norm())
    assert float(d.abs().max()) <= most, (what, float(d.abs().max()), most)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("m, n", SHAPES)
def test_against_64_bits(m, n, dt):
    u = matrix(m, n).to(dt)
    o = se.orthogonalize(u)
    assert o.dtype == dt and o.is_contiguous()
    near(o, exact(u), TOL[dt])


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("kind", ["flat", "identity", "strong"])
@pytest.mark.parametrize("m, n", [(64, 64), (130, 200), (400, 256), (768, 768)])
def test_spectra(m, n, kind, dt):
    u = matrix(m, n, kind=kind).to(dt)
    near(se.orthogonalize(u), exact(u), TOL[dt], update=u)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_other_numbers_of_steps(steps, dt):
    u = matrix(96, 160).to(dt)
    near(se.orthogonalize(u, steps=steps), exact(u, steps), TOL[dt])


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("shape", [(3, 40, 70), (2, 2, 65, 33), (40, 16, 24), (5, 130, 257), (2, 1024, 256), (1, 8, 8)])
def test_batches(shape, dt):
    u = matrix(*shape).to(dt)
    o = se.orthogonalize(u)
    for got, one in zip(o.flatten(0, -3), u.flatten(0, -3)):
        near(got, exact(one), TOL[dt])
    # a matrix's result does not depend on its neighbours
    again = se.orthogonalize(torch.cat([u, u])).flatten(0, -3)
    assert torch.equal(again[: len(again) // 2], o.flatten(0, -3))


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("m, n, pad, offset", [(33, 47, 1, 1), (64, 128, 8, 0), (200, 100, 3, 5), (1, 50, 7, 1)])
def test_strides(m, n, pad, offset, dt):
    flat = torch.full((3 * (m + 2) * (n + pad) + offset,), 5.0, dtype=dt, device="cuda")
    u = flat[offset:].view(3, m + 2, n + pad)[:, 1 : m + 1, :n]
    u.copy_(matrix(3, m, n))
    o = se.orthogonalize(u)
    assert torch.equal(o, se.orthogonalize(u.contiguous()))
    near(o[1], exact(u[1]), TOL[dt])


@pytest.mark.parametrize("dt", [F32, BF16])
def test_scale_of_the_update(dt):
    u = matrix(80, 120).to(dt)
    want = exact(u, eps=0.0)
    for s in (2.0**-60, 2.0**60):
        near(se.orthogonalize((u.double() * s).to(dt), eps=0.0), want, TOL[dt])
    big = matrix(8, 8).to(F32) * 1e25  # its square passes fp32's range
    near(se.orthogonalize(big), exact(big), TOL[F32])


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("m, n", [(70, 40), (300, 190), (130, 2200)])
def test_zero_infinite_and_nan_updates(m, n, dt):
    z = torch.zeros(3, m, n, dtype=dt, device="cuda")
    assert not se.orthogonalize(z).any()
    z[1] = matrix(m, n).to(dt)
    z[2] = z[1]
    z[2, 3, 4] = float("nan")
    o = se.orthogonalize(z)
    assert not o[0].any() and torch.isnan(o[2]).all()
    near(o[1], exact(z[1]), TOL[dt])
    z[2, 3, 4] = float("inf")
    o = se.orthogonalize(z)
    assert torch.isnan(o[2]).any() and torch.isfinite(o[:2]).all()
    for empty in ((0, 5, 5), (2, 0, 5), (2, 5, 0), (0, 0)):
        assert se.orthogonalize(torch.zeros(empty, dtype=dt, device="cuda")).shape == empty


@pytest.mark.parametrize("shape, dt", [((2, 300, 520), F32), ((100, 100), F32), ((200, 4096), F32), ((192, 6000), BF16),
                                       ((1600, 1700), BF16)])
def test_equal_calls_give_equal_bits(shape, dt):
    u = matrix(*shape).to(dt)  # long sides are summed in parts by several blocks
    first = se.orthogonalize(u)
    assert all(torch.equal(se.orthogonalize(u), first) for _ in range(10))
    near(first if first.dim() == 2 else first[1], exact(u if u.dim() == 2 else u[1]), TOL[dt])


@pytest.mark.parametrize("shape, dt", [((2100, 2100), BF16), ((2560, 1536), BF16), ((1100, 1000), F16), ((2, 1100, 1300), F32),
                                       ((1024, 3000), F32), ((3500, 3500), BF16)])
def test_large_matrices(shape, dt):
    u = matrix(*shape).to(dt)
    o = se.orthogonalize(u)
    near(o[-1] if o.dim() == 3 else o, exact(u[-1] if u.dim() == 3 else u), TOL[dt])
    w = torch.zeros(shape, dtype=dt, device="cuda")
    mom = torch.zeros(shape, device="cuda")
    se.muon_step(w, u, mom, lr=1.0, beta=0.0, scale=-1.0)  # from zero weights: the update itself
    assert float((w.double() - o.double()).norm() / o.double().norm()) < 2 * TOL[dt]


def reference_step(w, g, mom, lr, beta, decay, nesterov, steps=5, scale=None):
    mom = beta * mom.double() + g.double()
    o = exact(g.double() + beta * mom if nesterov else mom, steps)
    scale = max(1.0, w.shape[-2] / w.shape[-1]) ** 0.5 if scale is None else scale
    return w.double() * (1 - lr * decay) - lr * scale * o, mom, lr * scale * o


@pytest.mark.parametrize("dt, gt", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("shape", [(1, 1), (24, 40), (130, 66), (3, 64, 100), (520, 300)])
@pytest.mark.parametrize("nesterov, decay", [(True, 0.1), (False, 0.0)])
def test_step_against_64_bits(shape, dt, gt, nesterov, decay):
    lr, beta = 0.5, 0.9
    w, g, mom = matrix(*shape, seed=1, kind="flat").to(dt), matrix(*shape, seed=2).to(gt), matrix(*shape, seed=3).float()
    if shape == (1, 1):
        w, g, mom = w + 2, g + 0.5, mom + 1
    want, mom_want, change = reference_step(w, g, mom, lr, beta, decay, nesterov)
    assert se.muon_step(w, g, mom, lr=lr, beta=beta, weight_decay=decay, nesterov=nesterov) is None
    # momentum: one product and one sum, each within 2^-24 of at most |beta mom| + |g|
    assert bool(((mom.double() - mom_want).abs() <= 2.0**-23 * (mom_want.abs() + g.double().abs())).all())
    # beta and the two factors are rounded to fp32: 2^-23 of each term more
    rms = change.flatten(-2).norm(dim=-1)[..., None, None] / math.sqrt(shape[-1] * shape[-2])
    # (an fp32 step of 16-bit weights rounds its orthogonal part by nothing of its own: TOL without it is not worth a case)
    tol = 8 * TOL[dt] * torch.maximum(rms, change.abs() / 8) + (half(dt) + 2.0**-22) * (want.abs() + change.abs())
    assert bool(((w.double() - want).abs() <= tol).all()), float(((w.double() - want).abs() / tol).max())


def test_step_with_strides_scale_and_repeats():
    base = torch.zeros(2, 70, 90, device="cuda")
    w = base[:, 5:65, 10:50]
    w.copy_(matrix(2, 60, 40, kind="flat"))
    mom = torch.zeros(2, 60, 40, device="cuda")
    ref_w, ref_m = w.double(), mom.double()
    for k in range(4):
        g = matrix(2, 60, 40, seed=10 + k).float()
        ref_w, ref_m, _ = reference_step(ref_w, g, ref_m, 0.1, 0.95, 0.01, True, scale=0.25)
        se.muon_step(w, g, mom, lr=0.1, beta=0.95, weight_decay=0.01, scale=0.25)
    assert float((w.double() - ref_w).norm() / ref_w.norm()) < 4 * 2.0**-16
    base[:, 5:65, 10:50] = 0
    assert not base.any()  # nothing outside the matrices was written


def test_streams_and_graphs():
    u = [matrix(200, 300, seed=k).to(BF16) for k in range(3)]
    want = [se.orthogonalize(x) for x in u]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in u]
    got = []
    for s, x in zip(streams, u):
        with torch.cuda.stream(s):
            got.append([se.orthogonalize(x) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for r, q in zip(got, want) for p in r)
    side, graphs, outs = torch.cuda.Stream(), [], []
    for x in u[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(se.orthogonalize(x))
        graphs.append(graph)
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs, want))


def test_captured_steps_continue():
    w = matrix(96, 64, kind="flat").float()
    g = matrix(96, 64, seed=5).float()
    ref, mom, ref_mom = w.clone(), torch.zeros(96, 64, device="cuda"), torch.zeros(96, 64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        se.muon_step(w, g, mom)
    for _ in range(3):
        graph.replay()
        se.muon_step(ref, g, ref_mom)
    torch.cuda.synchronize()
    assert torch.equal(w, ref) and torch.equal(mom, ref_mom)


def test_calls_from_two_threads():
    import threading

    us = [matrix(150, 300, seed=k).to(BF16) for k in range(3)] + [matrix(60, 90).to(F32)]
    want = [se.orthogonalize(u) for u in us]
    torch.cuda.synchronize()
    bad = []

    def work(u, o):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not torch.equal(se.orthogonalize(u), o):
                    bad.append(1)

    threads = [threading.Thread(target=work, args=a) for a in zip(us, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_first_call_under_capture():
    """A fresh process whose first calls are captured."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch, sparse_embedding_b200 as se
x = torch.randn(300, 200, device="cuda"); w = torch.ones(200, device="cuda"); small = torch.randn(40, 60, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y, m, r = se.layer_norm(x, w, return_stats=True)
    d = se.layer_norm_backward(x, x, m, r, w)
    o, p = se.orthogonalize(x), se.orthogonalize(small)
g.replay(); torch.cuda.synchronize()
assert torch.equal(y, se.layer_norm(x, w)) and torch.equal(o, se.orthogonalize(x)) and torch.equal(p, se.orthogonalize(small))
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_optimizer_state_and_versions():
    p = torch.nn.Parameter(matrix(40, 70, kind="flat").to(BF16))
    opt = torch_ops.Muon([p], lr=0.1)
    p.grad = matrix(40, 70, seed=4).to(BF16)
    version = p._version
    opt.step()
    assert p._version > version
    buffer = opt.state[p]["momentum_buffer"]
    assert buffer.dtype == F32 and torch.equal(buffer, p.grad.float())
    other = torch.nn.Parameter(p.detach().clone())
    resumed = torch_ops.Muon([other], lr=0.3)
    resumed.load_state_dict(opt.state_dict())
    assert resumed.state[other]["momentum_buffer"].dtype == F32 and resumed.param_groups[0]["lr"] == 0.1
    other.grad = p.grad.clone()
    opt.step()
    resumed.step()
    assert torch.equal(p, other) and torch.equal(buffer, resumed.state[other]["momentum_buffer"])
    # a graph that saved the weight before the step refuses to go back through it
    x = torch.randn(3, 70, device="cuda", dtype=BF16, requires_grad=True)
    y = (x @ p.t()).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals():
    w = torch.zeros(6, 8, device="cuda")
    g, mom = torch.zeros_like(w), torch.zeros_like(w)
    for call, msg in [
        (lambda: se.orthogonalize(w.double()), "unsupported update dtype"),
        (lambda: se.orthogonalize(w.t()), "matrices at one stride"),
        (lambda: se.orthogonalize(w[0]), "at least two dimensions"),
        (lambda: se.orthogonalize(w, steps=0), "steps must be in"),
        (lambda: se.orthogonalize(w, eps=-1.0), "eps must be finite"),
        (lambda: se.muon_step(w, g[:5], mom), "grad must have weight's shape"),
        (lambda: se.muon_step(w, g, mom.half()), "momentum must be float32"),
        (lambda: se.muon_step(w, g.half(), mom), "weight's dtype or float32"),
        (lambda: se.muon_step(w, g.cpu(), mom), "grad must be a CUDA tensor"),
        (lambda: se.muon_step(w, w, mom), "must not share memory"),
        (lambda: se.muon_step(w, g, g), "must not share memory"),
        (lambda: se.muon_step(g[:3], w[:3], g[2:5]), "must not share memory"),
        (lambda: se.orthogonalize(torch.zeros(70000, 1, 1, device="cuda")), "batch must be at most"),
        (lambda: se.muon_step(w.t(), g.t(), mom.t()), "matrices at one stride"),
        (lambda: se.muon_step(w, g, mom, beta=1.0), "beta must be in"),
        (lambda: se.muon_step(w, g, mom, lr=float("nan")), "must be finite"),
    ]:
        with pytest.raises(ValueError, match=msg):
            call()
    assert not w.any() and not mom.any()


def test_a_training_step_over_the_store():
    """embedding_bag -> layer_norm -> two matrices -> loss, backward, then the store's Adagrad and Muon: against the
    same step in 64-bit torch operations. Every quantity is a few fp32 operations from the last, so 1e-4 of its norm
    is over 100 times their rounding; the Muon changes have the tolerance above."""
    dim, hidden, bags = 64, 96, 200
    store = se.EmbeddingStore(se.EmbeddingConfig(dims=[dim], key_dtype="int64", device=0), se.Uniform(-0.5, 0.5),
                              se.Adagrad(lr=0.05, eps=1e-8, initial_accumulator_value=0.1))
    gen = torch.Generator(device="cuda").manual_seed(3)
    pool = torch.arange(1000, 1300, device="cuda")
    counts = torch.randint(1, 5, (bags,), generator=gen, device="cuda")
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), counts.cumsum(0)])
    keys = pool[torch.randint(0, 300, (int(offsets[-1]),), generator=gen, device="cuda")]
    rows0 = store.lookup_or_insert(pool, dim)[0].view(-1, dim).double()
    param = lambda *s: torch.nn.Parameter(torch.randn(s, generator=gen, device="cuda") / s[-1] ** 0.5)  # noqa: E731
    w1, w2 = param(hidden, dim), param(32, hidden)
    scale, shift = torch.nn.Parameter(torch.ones(dim, device="cuda")), torch.nn.Parameter(torch.zeros(dim, device="cuda"))
    target = torch.randn(bags, 32, generator=gen, device="cuda")
    wide = [t.detach().double().requires_grad_() for t in (w1, w2, scale, shift)]
    muon = torch_ops.Muon([w1, w2], lr=0.1)

    x = torch_ops.embedding_bag(store, keys, offsets, dim)
    y = torch_ops.layer_norm(x, scale, shift)
    loss = ((torch.relu(y @ w1.t()) @ w2.t()) - target).square().mean()
    loss.backward()
    muon.step()
    store.optimizer_step(1)

    rows = rows0.clone().requires_grad_()
    bag = torch.repeat_interleave(torch.arange(bags, device="cuda"), counts)
    px = torch.zeros(bags, dim, dtype=torch.float64, device="cuda").index_add(0, bag, rows[keys - 1000])
    m = px.mean(1, keepdim=True)
    py = (px - m) / ((px - m).square().mean(1, keepdim=True) + 1e-5).sqrt() * wide[2] + wide[3]
    ploss = ((torch.relu(py @ wide[0].t()) @ wide[1].t()) - target.double()).square().mean()
    ploss.backward()
    off = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert abs(float(loss) - float(ploss)) < 1e-4 * float(ploss)
    for t, p in zip((w1, w2, scale, shift), wide):
        assert off(t.grad, p.grad) < 1e-4
    for t, p in zip((w1, w2), wide):
        want, _, change = reference_step(p.detach(), p.grad, torch.zeros_like(p), 0.1, 0.95, 0.0, True)
        # the gradients' own 1e-4 passes into the change; 485 = 3.4445^5 is the most the iteration can magnify it
        assert off(t.detach(), want) < 1e-2 * float(change.norm() / want.norm()) + 1e-6
    used = torch.zeros(300, dtype=torch.bool, device="cuda")
    used[keys - 1000] = True
    acc = 0.1 + rows.grad.square()
    want = torch.where(used[:, None], rows0 - 0.05 * rows.grad / (acc.sqrt() + 1e-8), rows0)
    got = store.lookup(pool, dim)[0].view(-1, dim)
    assert off(got, want) < 1e-4 and torch.equal(got[~used].double(), rows0[~used])
