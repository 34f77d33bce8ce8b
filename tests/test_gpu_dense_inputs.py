"""Inputs of the dense operators that are not plain fp32 torch tensors (GPU): DLPack objects, 16-bit autograd."""

import pytest
import torch

import sparse_embedding_b200 as se
from sparse_embedding_b200 import torch_ops

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


class Foreign:
    """Another library's array: nothing but the DLPack protocol."""

    def __init__(self, t):
        self.t = t

    def __dlpack__(self, **kw):
        return self.t.__dlpack__(**kw)

    def __dlpack_device__(self):
        return self.t.__dlpack_device__()


def rand(*shape, dt=F32, seed=0):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dt)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_dlpack_objects(dt):
    x, g, w, b = rand(30, 77, dt=dt), rand(30, 77, dt=dt, seed=1), rand(77, dt=dt, seed=2), rand(77, dt=dt, seed=3)
    wide = rand(30, 80, dt=dt)[:, 2:79]
    for t in (x, wide):
        y, mean, rstd = se.layer_norm(t, w, b, return_stats=True)
        got = se.layer_norm(Foreign(t), Foreign(w), Foreign(b), return_stats=True)
        assert all(torch.equal(p, q) for p, q in zip(got, (y, mean, rstd)))
        want = se.layer_norm_backward(g, t, mean, rstd, w)
        got = se.layer_norm_backward(Foreign(g), Foreign(t), mean, rstd, Foreign(w))
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert torch.equal(se.orthogonalize(Foreign(x)), se.orthogonalize(x))
    one, two, mom, mom2 = x.clone(), x.clone(), torch.zeros(30, 77, device="cuda"), torch.zeros(30, 77, device="cuda")
    se.muon_step(one, g, mom)
    se.muon_step(Foreign(two), Foreign(g), Foreign(mom2))  # in place, in the other library's memory
    assert torch.equal(one, two) and torch.equal(mom, mom2) and not torch.equal(one, x)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        se.layer_norm(Foreign(x.cpu()))


@pytest.mark.parametrize("dt, pt", [(F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("shape", [(40, 72), (3, 5, 33), (2000, 256), (7, 4100)])
def test_autograd_of_16_bit_rows(shape, dt, pt):
    x, g = rand(*shape, dt=dt).requires_grad_(), rand(*shape, dt=dt, seed=1)
    w, b = rand(shape[-1], dt=pt, seed=2).requires_grad_(), rand(shape[-1], dt=pt, seed=3).requires_grad_()
    y = torch_ops.layer_norm(x, w, b)
    assert y.dtype == dt and y.shape == x.shape
    y.backward(g)
    with torch.no_grad():
        z, mean, rstd = se.layer_norm(x, w, b, return_stats=True)
        want = se.layer_norm_backward(g, x, mean, rstd, w)
    assert torch.equal(y, z)
    for t, v in zip((x, w, b), want):
        assert t.grad.dtype == t.dtype and torch.equal(t.grad, v)
    # frozen parameters, and rows without a gradient
    x2 = x.detach().clone().requires_grad_()
    torch_ops.layer_norm(x2, w.detach(), b.detach()).backward(g)
    assert torch.equal(x2.grad, want[0])
    w2 = w.detach().clone().requires_grad_()
    torch_ops.layer_norm(x.detach(), w2).backward(g)
    assert torch.equal(w2.grad, want[1])


@pytest.mark.parametrize("dt", [F16, BF16])
def test_a_small_tower_of_16_bit_matrices(dt):
    """Rows -> layer_norm -> matrix -> loss, in 16 bits, against the same formulas in 64: every quantity is a few
    operations of relative error finfo.eps / 2 and sums of 32 bits from the last; gradients within 16 of those."""
    x, w, s = rand(300, 64, dt=dt).requires_grad_(), (rand(48, 64, seed=1) / 8).to(dt).requires_grad_(), rand(64, seed=2).requires_grad_()
    c = rand(300, 48, seed=3)
    (torch.nn.functional.linear(torch_ops.layer_norm(x, s), w).float() * c).sum().backward()
    X, W, S = (t.detach().double().requires_grad_() for t in (x, w, s))
    m = X.mean(1, keepdim=True)
    Y = (X - m) / ((X - m).square().mean(1, keepdim=True) + 1e-5).sqrt() * S
    ((Y @ W.t()) * c.double()).sum().backward()
    for got, want in ((x, X), (w, W), (s, S)):
        assert float((got.grad.double() - want.grad).norm() / want.grad.norm()) < 16 * torch.finfo(dt).eps / 2


def test_captured_optimizer_steps():
    """Replays go on with the momentum; a first step, whose zeros a graph would replay, is refused."""
    params = [torch.nn.Parameter(rand(96, 64, seed=k)) for k in range(2)]
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    grads = [rand(96, 64, seed=k + 5) for k in range(2)]
    opt, twin = torch_ops.Muon(params, lr=0.1), torch_ops.Muon(twins, lr=0.1)
    for p, q, g in zip(params, twins, grads):
        p.grad, q.grad = g.clone(), g.clone()
    with pytest.raises(RuntimeError, match="step once before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert not opt.state[params[0]] and all(torch.equal(p, q) for p, q in zip(params, twins))
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
    for _ in range(4):
        twin.step()
    torch.cuda.synchronize()
    for p, q in zip(params, twins):
        assert torch.equal(p, q) and torch.equal(opt.state[p]["momentum_buffer"], twin.state[q]["momentum_buffer"])
