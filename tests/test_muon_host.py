"""Argument checks of the Muon update that need no GPU (CPU only)."""

import ctypes as C

import numpy as np
import pytest
import torch

import sparse_embedding_b200 as se
from sparse_embedding_b200 import _native as N
from sparse_embedding_b200 import dense, torch_ops


def test_host_inputs_are_refused():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="update must be a CUDA tensor"):
        se.orthogonalize(x)
    with pytest.raises(ValueError, match="update must be a CUDA tensor"):
        se.orthogonalize(np.zeros((4, 8), np.float32))
    with pytest.raises(TypeError, match="update must be a CUDA tensor"):
        se.orthogonalize(3)
    with pytest.raises(ValueError, match="weight must be a CUDA tensor"):
        se.muon_step(x, x, x)


def test_matrices_of_strided_tensors():
    base = torch.zeros(3, 4, 6, 16)
    assert dense._matrices(base, "x") == (12, 6, 16, 96, 16)
    assert dense._matrices(base[..., :5], "x") == (12, 6, 5, 96, 16)
    assert dense._matrices(base[:, 1, ::2, 2:9], "x") == (3, 3, 7, 384, 32)
    assert dense._matrices(base[0, 0], "x") == (1, 6, 16, 96, 16)
    assert dense._matrices(base[0, 0, :1, :3], "x") == (1, 1, 3, 3, 3)
    assert dense._matrices(torch.zeros(0, 4, 5), "x")[0] == 0
    assert dense._matrices(torch.zeros(2, 0, 5), "x")[0] == 0
    for bad in (base[:, ::3, :, 1:], base.transpose(2, 3), base[..., ::2], torch.zeros(4, 5).expand(3, 4, 5),
                torch.zeros(5).expand(4, 5), base.transpose(0, 1)):
        with pytest.raises(ValueError, match="x must be matrices at one stride"):
            dense._matrices(bad, "x")
    with pytest.raises(ValueError, match="at least two dimensions"):
        dense._matrices(torch.zeros(3), "x")


def orth(dtype=0, batch=1, m=4, n=4, bs=16, rs=4, steps=5, eps=1e-7):
    return N.lib().se_orthogonalize(dtype, None, batch, m, n, bs, rs, steps, eps, None, None, 0, 0, None)


@pytest.mark.parametrize("kw, msg", [
    (dict(dtype=3), b"unsupported dtype"), (dict(m=-1), b"m and n must be in"), (dict(n=(1 << 20) + 1), b"m and n must be in"),
    (dict(batch=65536), b"batch must be at most"), (dict(steps=0), b"steps must be in"), (dict(steps=101), b"steps must be in"),
    (dict(eps=-1.0), b"eps must be finite"), (dict(eps=float("nan")), b"eps must be finite"),
    (dict(rs=3), b"overlap"), (dict(batch=2, bs=15), b"overlap"), (dict(batch=2, rs=8, bs=24), b"overlap"),
])
def test_c_abi_argument_errors(kw, msg):
    assert orth(**kw) == N.SE_ERR_INVALID_ARGUMENT
    assert msg in N.lib().se_last_error()


def step(**kw):
    a = dict(lr=0.1, beta=0.9, wd=0.0, scale=1.0)
    a.update(kw)
    return N.lib().se_muon_step(0, 0, None, 16, 4, None, 16, 4, None, 16, 4, 1, 4, 4, a["lr"], a["beta"], a["wd"],
                                a["scale"], 1, 5, 1e-7, None, 0, 0, None)


@pytest.mark.parametrize("kw", [dict(lr=float("inf")), dict(beta=1.0), dict(beta=-0.1), dict(beta=float("nan")),
                                dict(wd=float("nan")), dict(scale=float("inf"))])
def test_step_values_are_checked(kw):
    assert step(**kw) == N.SE_ERR_INVALID_ARGUMENT


def test_nothing_to_do_needs_no_device():
    assert orth(batch=0) == orth(m=0, rs=4) == orth(n=0) == N.SE_OK
    size = C.c_size_t(7)
    for args in ((0, 0, 4, 4), (0, 3, 0, 4), (2, 3, 4, 0)):
        N.check(N.lib().se_muon_workspace(*args, C.byref(size)))
        assert size.value == 0
    N.check(N.lib().se_muon_workspace(2, 1, 100, 200, C.byref(size)))
    single = size.value
    N.check(N.lib().se_muon_workspace(2, 1, 200, 100, C.byref(size)))
    assert size.value == single >= 4 * 2 * 100 * 200  # X twice as pairs of 16-bit values
    N.check(N.lib().se_muon_workspace(0, 1, 100, 200, C.byref(size)))
    assert size.value > single
    assert N.lib().se_muon_workspace(0, 1, 4, 4, None) == N.SE_ERR_INVALID_ARGUMENT


def test_optimizer_refuses_vectors():
    with pytest.raises(ValueError, match="at least two dimensions"):
        torch_ops.Muon([torch.nn.Parameter(torch.zeros(4))])
    opt = torch_ops.Muon([torch.nn.Parameter(torch.zeros(4, 4))])
    opt.step()  # no gradients: nothing to do
    with pytest.raises(ValueError, match="at least two dimensions"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4))]})


def test_full_products_flag():
    full = dense._FULL_PRODUCTS
    size = [C.c_size_t() for _ in range(4)]
    for out, code in zip(size, (0, 2, 2 | full, full)):
        N.check(N.lib().se_muon_workspace(code, 1, 1000, 2000, C.byref(out)))
    assert size[1].value < size[2].value == size[0].value == size[3].value
    assert orth(dtype=3 | full) == orth(dtype=2 | full << 1) == N.SE_ERR_INVALID_ARGUMENT
    assert b"unsupported dtype" in N.lib().se_last_error()


def test_matrices_on_chip_ask_for_no_more_in_a_batch():
    def ask(code, batch, m, n):
        size = C.c_size_t()
        N.check(N.lib().se_muon_workspace(code, batch, m, n, C.byref(size)))
        return size.value

    for code in (0, 1, 2, 2 | dense._FULL_PRODUCTS):
        for m, n in ((128, 256), (256, 128), (16, 16), (1, 1)):
            assert 0 < ask(code, 65535, m, n) == ask(code, 1, m, n) < 1 << 20
        assert ask(code, 3, 129, 256) > 2 * ask(code, 1, 129, 256)


def test_optimizer_refuses_a_group_whole():
    param = lambda t: torch.nn.Parameter(t)  # noqa: E731
    opt = torch_ops.Muon([param(torch.zeros(4, 4))])
    base = torch.zeros(70000, 1, 1)
    for bad, msg in ((torch.zeros(4), "at least two dimensions"), (torch.zeros(8, 4).t(), "every parameter must be matrices"),
                     (base, "batch must be at most 65535"), (torch.zeros(1).expand(1, (1 << 20) + 1), "must be")):
        with pytest.raises(ValueError, match=msg):
            opt.add_param_group({"params": [param(torch.zeros(3, 5)), param(bad)]})
        assert len(opt.param_groups) == 1 and len(opt.param_groups[0]["params"]) == 1
        opt.step()  # nothing of the refused group is left
    opt.add_param_group({"params": [param(torch.zeros(2, 3, 5)), param(torch.zeros(6, 9)[:, 2:7])], "lr": 0.5})
    assert opt.param_groups[1]["lr"] == 0.5 and opt.param_groups[1]["precise"] is False


def test_sparse_gradients_are_refused_before_any_step():
    first, second = torch.nn.Parameter(torch.zeros(4, 4)), torch.nn.Parameter(torch.zeros(4, 4))
    opt = torch_ops.Muon([first, second])
    first.grad, second.grad = torch.ones(4, 4), torch.ones(4, 4).to_sparse()
    with pytest.raises(ValueError, match="dense gradients"):  # not the first parameter's refusal (a host tensor)
        opt.step()
    assert not opt.state
