"""Waits inside the dense operators' kernels that run out (GPU): with a limit of one clock the first wait for a copy, a
matrix instruction or another block that is not done gives up, the kernel lets what it has in flight land and returns."""

import contextlib

import pytest
import torch

import sparse_embedding_b200 as se
from sparse_embedding_b200 import _native as N

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
# one CTA on chip; over the grid with single and with three products; pairs of CTAs; sums in parts
SHAPES = [((40, 96), F32), ((3, 128, 200), BF16), ((300, 520), F32), ((300, 520), BF16), ((2048, 2048), BF16),
          ((200, 4096), F32)]


@contextlib.contextmanager
def brief_waits():
    N.check(N.lib().se_set_wait_limit(1))
    try:
        yield
        torch.cuda.synchronize()
    finally:
        N.check(N.lib().se_set_wait_limit(0))


def rand(*shape, dt=F32, seed=0):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dt)


@pytest.mark.parametrize("shape, dt", SHAPES)
def test_a_step_that_gave_up_leaves_the_weights(shape, dt):
    w, g, mom = rand(*shape, dt=dt), rand(*shape, dt=dt, seed=1), torch.zeros(shape, device="cuda")
    before, want, want_mom = w.clone(), w.clone(), mom.clone()
    se.muon_step(want, g, want_mom)
    with brief_waits():
        se.muon_step(w, g, mom)
    assert torch.equal(w, before) and torch.equal(mom, g.float())
    with pytest.raises(RuntimeError, match="gave up waiting"):
        se.muon_step(w, g, mom)
    assert torch.equal(w, before)
    mom.zero_()
    se.muon_step(w, g, mom)
    assert torch.equal(w, want) and torch.equal(mom, want_mom)


@pytest.mark.parametrize("shape, dt", SHAPES)
def test_an_orthogonalisation_that_gave_up(shape, dt):
    u = rand(*shape, dt=dt)
    want = se.orthogonalize(u)
    with brief_waits():
        se.orthogonalize(u)
    with pytest.raises(RuntimeError, match="gave up waiting"):
        se.orthogonalize(u)
    assert torch.equal(se.orthogonalize(u), want)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("dim", [128, 301, 700, 1037, 4096])
def test_normalisations_that_gave_up(dim, dt):
    rows = (1 << 27) // dim  # more than L2 holds: the blocks do wait for their copies
    x, g, w = rand(rows, dim, dt=dt), rand(rows, dim, dt=dt, seed=1), torch.ones(dim, device="cuda")
    y, mean, rstd = se.layer_norm(x, w, return_stats=True)
    want = se.layer_norm_backward(g, x, mean, rstd, w)
    for call, right in ((lambda: [se.layer_norm(x, w)], [y]), (lambda: se.layer_norm_backward(g, x, mean, rstd, w), want)):
        with brief_waits():
            got = call()
        try:
            call()
        except RuntimeError as e:
            assert "gave up waiting" in str(e)
        else:  # rows that take longer to work on than to copy: no wait need run out
            assert dim != 128 and all(torch.equal(p, q) for p, q in zip(got, right))
    assert torch.equal(se.layer_norm(x, w), y)
    assert all(torch.equal(p, q) for p, q in zip(se.layer_norm_backward(g, x, mean, rstd, w), want))


def test_limits_are_checked():
    assert N.lib().se_set_wait_limit(8_000_000_001) == N.SE_ERR_INVALID_ARGUMENT
    assert b"at most 8e9" in N.lib().se_last_error()


def test_reports_stay_with_their_stream():
    u = rand(40, 96)
    x, w = rand(2000, 128), torch.ones(128, device="cuda")
    want, y = se.orthogonalize(u), se.layer_norm(x, w)
    bad, other = torch.cuda.Stream(), torch.cuda.Stream()
    with brief_waits(), torch.cuda.stream(bad):
        se.orthogonalize(u)
    with torch.cuda.stream(other):  # nobody else is refused
        assert torch.equal(se.orthogonalize(u), want) and torch.equal(se.layer_norm(x, w), y)
    assert torch.equal(se.orthogonalize(u), want)
    with torch.cuda.stream(bad):
        with pytest.raises(RuntimeError, match="gave up waiting"):
            se.layer_norm(x, w)
        assert torch.equal(se.layer_norm(x, w), y)


def test_replayed_graphs_report():
    w, g, mom = rand(300, 200), rand(300, 200, seed=1), torch.zeros(300, 200, device="cuda")
    before = w.clone()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with brief_waits(), torch.cuda.graph(graph, stream=side):  # a graph keeps the limit of its capture
        se.muon_step(w, g, mom)
    se.check_waits()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, before)
        for device in (None, torch.device("cuda", 0)):
            if device is None:
                with pytest.raises(RuntimeError, match="gave up waiting"):
                    se.check_waits()
            else:
                se.check_waits(device)  # taken once
    se.check_waits(0)
    se.check_waits("cuda:0")
