"""The Newton-Schulz products in every form that plan_for chooses (GPU): tile widths, single CTAs and pairs, sums over k
whole and in parts, against the formulas in 64 bits.

Tolerances, relative to the norm. The last step's X' = a X + B X has |X'| >= 0.68 |X| where |B X| <= 2.75 |X|, so a
relative error e of its product is one of 4 e at most in the result, the error of the step before passes f' <= 1.6, and
those of earlier steps shrink against the values' growth: 4 e sqrt(1 + 1.6^2) = 7.6 e in all.
 * bf16: both f16 operands are rounded, each by 2.1e-4 in the mean square (an eighth of bf16's 1.7e-3): e = 2.9e-4 where
   B's values lie off its diagonal, which they do by less than their half: 1.1e-3, and 1.7e-3 for the result's own
   rounding. 2^-8 is twice their sum in squares; operands of two bits less would be off by 4.7e-3.
 * fp32, f16: a sum loses 2^-24 in the mean in each of the 16 instructions between two flushes: e = 2^-20, 7.6 e < 2^-17;
   f16's own rounding 2^-12 in the mean square, 2^-11 at most, more."""

import pytest
import torch

import sparse_embedding_b200 as se

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TOL = {F32: 2.0**-17, F16: 2.0**-17 + 2.0**-11, BF16: 2.0**-8}
# the tile of single products (CTAs, columns) and whether X X^T is summed in parts; three products have one tile
FORMS = [((130, 133), BF16, "1x64"), ((2710, 255), BF16, "1x64"), ((193, 3080), BF16, "1x64 parts"),
         ((3, 770, 774), BF16, "1x128"), ((8, 715, 517), BF16, "1x128"), ((773, 4077), BF16, "1x128 parts"),
         ((8, 402, 869), BF16, "2x128"), ((3, 4109, 389), BF16, "2x128 parts"), ((2, 1616, 2187), BF16, "2x256"),
         ((4, 649, 8078), BF16, "2x256 parts"), ((4, 1029, 2891), BF16, "1x256"), ((3, 8207, 779), BF16, "1x256 parts"),
         ((874, 938), F32, "three"), ((2, 1561, 129), F32, "three parts"), ((668, 1851), F32, "three parts"),
         ((1100, 700), F16, "three"), ((129, 1561), F16, "three parts"), ((4100, 1000), F32, "three parts")]


def matrix(*shape):
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    r = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float64)  # noqa: E731
    *lead, m, n = shape
    low = (r(*lead, m, 8) / torch.arange(1, 9, device="cuda")) @ r(*lead, 8, n)
    return 1e-2 * (low + 0.3 * r(*shape))


def exact(u, steps=5):
    x = u.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + 1e-7)
    wide = x.shape[-2] <= x.shape[-1]
    for _ in range(steps):
        a = x @ x.mT if wide else x.mT @ x
        p = -4.7750 * a + 2.0315 * (a @ a)
        x = 3.4445 * x + (p @ x if wide else x @ p)
    return x


def off(got, want):
    return float(((got.double() - want).flatten(-2).norm(dim=-1) / want.flatten(-2).norm(dim=-1)).max())


@pytest.mark.parametrize("shape, dt, form", FORMS)
def test_form(shape, dt, form):
    u = matrix(*shape).to(dt)
    want = exact(u)
    o = se.orthogonalize(u)
    assert off(o, want) <= TOL[dt]
    for _ in range(3):
        assert torch.equal(se.orthogonalize(u), o)
    w, mom = torch.zeros_like(u), torch.zeros(shape, device="cuda")
    se.muon_step(w, u, mom, lr=1.0, beta=0.0, scale=-1.0)  # from zero weights: the update itself
    assert off(w, want) <= TOL[dt]
    again = torch.zeros_like(u)
    se.muon_step(again, u, torch.zeros_like(mom), lr=1.0, beta=0.0, scale=-1.0)
    assert torch.equal(again, w)


@pytest.mark.parametrize("shape", [(40, 70), (3, 128, 200), (300, 520), (2, 1561, 129), (1300, 1200)])
def test_full_products_for_bf16(shape):
    """The same products as for fp32: the bf16 result is the fp32 one's rounding, bit by bit; a step's weights are within
    half a step of bf16 of those from it, with 2^-22 |O| for its pair of f16 and fp32 roundings of lr and decay."""
    u = matrix(*shape).to(BF16)
    full = se.orthogonalize(u.float())
    o = se.orthogonalize(u, precise=True)
    assert o.dtype == BF16 and torch.equal(o, full.to(BF16))
    assert not torch.equal(o, se.orthogonalize(u))
    for grad in (u, u.float()):
        w = matrix(*reversed(shape)).mT.reshape(shape).to(BF16).contiguous()
        before, mom = w.double(), torch.zeros(shape, device="cuda")
        se.muon_step(w, grad, mom, lr=0.5, beta=0.0, weight_decay=0.1, scale=2.0, precise=True)
        want = before * 0.95 - full.double()
        tol = 2.0**-8 * want.abs() + 2.0**-22 * (before.abs() + 2 * full.double().abs())
        assert bool(((w.double() - want).abs() <= tol).all())


def test_optimizer_takes_full_products():
    from sparse_embedding_b200 import torch_ops

    p = [torch.nn.Parameter(matrix(96, 64).to(BF16)) for _ in range(2)]
    step = matrix(96, 65)[:, 1:].to(BF16).contiguous()
    want = p[0].detach().clone()
    se.muon_step(want, step, torch.zeros(96, 64, device="cuda"), lr=0.1, precise=True)
    old = torch_ops.Muon([p[1]], lr=0.1)
    state = old.state_dict()
    del state["param_groups"][0]["precise"]  # a state from before
    old.load_state_dict(state)
    for q in p:
        q.grad = step.clone()
    torch_ops.Muon([p[0]], lr=0.1, precise=True).step()
    old.step()
    assert torch.equal(p[0], want) and not torch.equal(p[1], want)


def test_matrices_on_chip_need_no_workspace():
    from sparse_embedding_b200 import _native as N

    u = matrix(50, 40, 96).float()
    out, st = torch.empty_like(u), torch.cuda.current_stream().cuda_stream
    N.check(N.lib().se_orthogonalize(0, u.data_ptr(), 50, 40, 96, 40 * 96, 96, 5, 1e-7, out.data_ptr(), None, 0, 0, st))
    assert torch.equal(out, se.orthogonalize(u))
    big = matrix(130, 300).float()
    rc = N.lib().se_orthogonalize(0, big.data_ptr(), 1, 130, 300, 39000, 300, 5, 1e-7, big.data_ptr(), None, 0, 0, st)
    assert rc == N.SE_ERR_INVALID_ARGUMENT and b"workspace is null" in N.lib().se_last_error()
    # 20,000 small matrices: 80 MB of them, and no more than their result beside them
    many = torch.ones(20000, 32, 32, device="cuda")
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    se.orthogonalize(many)
    assert torch.cuda.max_memory_allocated() - before < many.numel() * 4 + (1 << 20)
