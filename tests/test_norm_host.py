"""Layer normalisation's argument checks that need no GPU (CPU only)."""

import ctypes as C

import numpy as np
import pytest
import torch

import sparse_embedding_b200 as se
from sparse_embedding_b200 import _native as N
from sparse_embedding_b200 import dense


def test_host_inputs_are_refused():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        se.layer_norm(x)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        se.layer_norm(np.zeros((4, 8), np.float32))
    with pytest.raises(TypeError, match="x must be a CUDA tensor"):
        se.layer_norm([[1.0, 2.0]])
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        se.layer_norm_backward(x, x, x, x)


def test_rows_of_strided_tensors():
    base = torch.zeros(6, 5, 16)
    assert dense._rows(base, "x") == (30, 16, 16)
    assert dense._rows(base[:, :, :7], "x") == (30, 7, 16)
    assert dense._rows(base[:, 2, 3:9], "x") == (6, 6, 80)
    assert dense._rows(base[::2, 0], "x") == (3, 16, 160)
    assert dense._rows(base[2, 1], "x") == (1, 16, 16)
    assert dense._rows(base[0, :1, ::1], "x") == (1, 16, 16)
    assert dense._rows(torch.zeros(0, 8), "x") == (0, 8, 8)
    assert dense._rows(torch.zeros(4, 1), "x") == (4, 1, 1)
    for bad in (base[:, ::2, :7], base[:, :4, :], base.transpose(0, 1), base[..., ::2], base[0].t(),
                torch.zeros(8).expand(3, 8)):
        with pytest.raises(ValueError, match="x must be rows at one stride"):
            dense._rows(bad, "x")
    with pytest.raises(ValueError, match="dim must be > 0"):
        dense._rows(torch.zeros(3, 0), "x")
    with pytest.raises(ValueError, match="at least one dimension"):
        dense._rows(torch.zeros(()), "x")


def call(**kw):
    a = dict(value=0, param=0, x=None, rows=1, dim=8, stride=8, eps=1e-5)
    a.update(kw)
    return N.lib().se_layer_norm(a["value"], a["param"], a["x"], a["rows"], a["dim"], a["stride"], None, None, a["eps"],
                                 None, None, None, 0, None)


@pytest.mark.parametrize("kw, msg", [
    (dict(value=3), b"unsupported value_dtype"), (dict(value=-1), b"unsupported value_dtype"),
    (dict(param=7), b"unsupported param_dtype"), (dict(dim=0), b"dim must be > 0"),
    (dict(dim=-4), b"dim must be > 0"), (dict(dim=1 << 31, stride=1 << 31), b"dim must be at most 2^30"),
    (dict(eps=-1.0), b"eps must be finite"), (dict(eps=float("nan")), b"eps must be finite"),
    (dict(eps=float("inf")), b"eps must be finite"), (dict(rows=2, stride=7), b"x_stride must be at least dim"),
])
def test_c_abi_argument_errors(kw, msg):
    assert call(**kw) == N.SE_ERR_INVALID_ARGUMENT
    assert msg in N.lib().se_last_error()


def test_no_rows_need_no_device():
    assert call(rows=0) == N.SE_OK
    assert N.lib().se_layer_norm_backward_workspace(1, 8, 0, None) == N.SE_ERR_INVALID_ARGUMENT
    size = C.c_size_t()
    assert N.lib().se_layer_norm_backward_workspace(1, 0, 0, C.byref(size)) == N.SE_ERR_INVALID_ARGUMENT


def test_waits_of_a_device():
    N.check(N.lib().se_check_waits(0))  # nothing ran: nothing to report
    se.check_waits(0)
    with pytest.raises(ValueError, match="must be a CUDA device"):
        se.check_waits("cpu")
