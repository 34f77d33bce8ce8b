"""Dense operators that run next to the store: layer normalisation of its rows
(pooled bags, looked-up rows) with the backward pass, and the Muon update of the
matrices that read them, beside the store's own row optimizers. They have no
counterpart in the reference, whose users run the dense part of a model outside
it.

Inputs are CUDA tensors (or DLPack objects in CUDA memory) whose last axis is
contiguous; rows may lie further apart than their length, as slices of wider
tensors do. The work runs on the current torch stream of the tensors' device,
allocates from torch's allocator only and never waits for the GPU, so calls can
be captured into CUDA graphs. `torch_ops` has the autograd forms. A kernel
whose waits gave up is reported by the next call on its stream (RuntimeError),
or by `check_waits`.
"""

from __future__ import annotations

import ctypes as C
import functools
import math

from . import _native as N
from ._tensors import _torch_dtype_name, is_torch_tensor, torch_mod

_FLOATS = {}  # torch dtype -> code of the C ABI


def _code(dtype) -> int:
    if not _FLOATS:
        torch = torch_mod()
        _FLOATS.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    return _FLOATS.get(dtype, -1)


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    """An entry point of the library (looked up once)."""
    return getattr(N.lib(), name)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(name: str, *args) -> int:
    size = C.c_size_t()
    N.check(_entry(name)(*args, C.byref(size)))
    return size.value


def _cuda_tensor(x, what: str):
    """x as a CUDA tensor of a supported dtype."""
    if not is_torch_tensor(x):
        if not hasattr(x, "__dlpack__"):
            raise TypeError(f"{what} must be a CUDA tensor")
        x = torch_mod().from_dlpack(x)
    if not x.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if _code(x.dtype) < 0:
        raise ValueError(f"unsupported {what} dtype: {_torch_dtype_name(x)}")
    return x


def _strided(x, last: int):
    """(count, stride) of the blocks that x's last `last` axes form, over its
    leading axes; None where no single stride covers them."""
    count, stride = 1, None
    for size, step in zip(reversed(x.shape[: x.dim() - last]), reversed(x.stride()[: x.dim() - last])):
        if size != 1:
            if stride is None:
                stride = step
            elif step != stride * count:
                return None
        count *= size
    return count, stride or 0


def _rows(x, what: str):
    """(rows, dim, row stride) of x as rows of its last axis."""
    if x.dim() < 1:
        raise ValueError(f"{what} must have at least one dimension")
    dim = x.shape[-1]
    if dim == 0:
        raise ValueError("dim must be > 0")
    if x.is_contiguous():
        return x.numel() // dim, dim, dim
    if x.numel() == 0:
        return 0, dim, dim
    found = _strided(x, 1)
    if (dim > 1 and x.stride(-1) != 1) or found is None or (found[0] > 1 and found[1] < dim):
        raise ValueError(f"{what} must be rows at one stride with a contiguous last dimension")
    rows, stride = found
    return rows, dim, max(stride, dim)


def _same_device(a, b, what: str) -> None:
    if a.device != b.device:
        raise ValueError(f"{what} is on {b.device}, the call on {a.device}")


def _param(x, dim: int, p, what: str):
    p = _cuda_tensor(p, what)
    _same_device(x, p, what)
    if p.dim() != 1 or p.shape[0] != dim or not p.is_contiguous():
        raise ValueError(f"{what} must be a contiguous 1D tensor of dim values")
    if p.dtype != x.dtype and p.dtype != torch_mod().float32:
        raise ValueError(f"{what} must have x's dtype or float32")
    return p


def _affine(x, dim: int, weight, bias):
    if weight is None:
        if bias is not None:
            raise ValueError("bias needs a weight")
        return None, None, 0
    weight = _param(x, dim, weight, "weight")
    if bias is not None:
        bias = _param(x, dim, bias, "bias")
        if bias.dtype != weight.dtype:
            raise ValueError("weight and bias must have the same dtype")
    return weight, bias, _code(weight.dtype)


def _like(x):
    # empty_like is torch's quickest allocation (1.3 us of host time; new_empty 2.3), but it keeps the order of the axes
    return torch_mod().empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _bytes(x, nbytes: int):
    """A workspace on x's device (torch's allocations are aligned to 512 bytes)."""
    torch = torch_mod()
    return torch.empty(nbytes, dtype=torch.uint8, device=x.device)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(t) -> int:
    # what torch.cuda.current_stream(t.device).cuda_stream gives, without building a Stream object
    return torch_mod()._C._cuda_getCurrentRawStream(t.device.index)


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, return_stats: bool = False):
    """Normalises the rows of x [..., dim] (float32, float16 or bfloat16):
    y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis, with
    fp32 statistics. weight and bias [dim] have x's dtype or float32. Returns
    y, or with return_stats (y, mean, rstd): fp32, of x's leading shape, as
    layer_norm_backward takes them. Outside autograd."""
    x = _cuda_tensor(x, "x")
    rows, dim, stride = _rows(x, "x")
    weight, bias, pcode = _affine(x, dim, weight, bias)
    eps = float(eps)
    if not math.isfinite(eps) or eps < 0.0:
        raise ValueError("eps must be finite and non-negative")
    y = _like(x)
    mean = rstd = None
    if return_stats:
        torch = torch_mod()
        mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
    N.check(_entry("se_layer_norm")(_code(x.dtype), pcode, x.data_ptr(), rows, dim, stride, _ptr(weight), _ptr(bias), eps,
                                    y.data_ptr(), _ptr(mean), _ptr(rstd), x.device.index, _stream(x)))
    return (y, mean, rstd) if return_stats else y


def layer_norm_backward(grad, x, mean, rstd, weight=None, with_bias: bool = True):
    """(dx, dweight, dbias) of layer_norm for the gradient of its y: `grad` has
    x's shape and dtype, mean and rstd come from the forward pass. Without a
    weight dweight and dbias are None; dbias also without with_bias. They have
    the weight's dtype, are summed in fp32, and equal calls on one device give
    equal bits."""
    x = _cuda_tensor(x, "x")
    grad = _cuda_tensor(grad, "grad")
    _same_device(x, grad, "grad")
    if grad.shape != x.shape or grad.dtype != x.dtype:
        raise ValueError("grad must have x's shape and dtype")
    rows, dim, stride = _rows(x, "x")
    _, _, gstride = _rows(grad, "grad")
    weight, _, pcode = _affine(x, dim, weight, None)
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        if not is_torch_tensor(t) or t.dtype != torch_mod().float32 or t.numel() != rows or not t.is_contiguous():
            raise ValueError(f"{what} must be a contiguous float32 tensor with a value per row")
        _same_device(x, t, what)
    dx = _like(x)
    dw = db = work = None
    nbytes = 0
    if weight is not None:
        dw = _like(weight)
        db = _like(weight) if with_bias else None
        nbytes = _workspace_bytes("se_layer_norm_backward_workspace", rows, dim, x.device.index)
        work = _bytes(x, nbytes)
    N.check(_entry("se_layer_norm_backward")(_code(x.dtype), pcode, grad.data_ptr(), gstride, x.data_ptr(), stride, rows,
                                             dim, mean.data_ptr(), rstd.data_ptr(), _ptr(weight), dx.data_ptr(),
                                             _ptr(dw), _ptr(db), _ptr(work), nbytes, x.device.index, _stream(x)))
    return dx, dw, db


def check_waits(device=None) -> None:
    """Raises RuntimeError where a wait inside a dense operator's kernel on the
    device (an index, a torch.device; the current one by default) has given up
    and no call has reported it: the results of that call are not valid. The
    host does not wait for the GPU, so synchronise first where it matters, as
    after the last replay of a graph."""
    torch = torch_mod()
    if device is None or isinstance(device, int):
        index = device
    else:
        where = torch.device(device)
        if where.type != "cuda":
            raise ValueError("device must be a CUDA device")
        index = where.index
    N.check(_entry("se_check_waits")(torch.cuda.current_device() if index is None else index))


def _matrices(x, what: str):
    """(batch, m, n, batch stride, row stride) of x as matrices of its last two axes."""
    if x.dim() < 2:
        raise ValueError(f"{what} must have at least two dimensions")
    m, n = x.shape[-2:]
    if x.is_contiguous():
        return (x.numel() // (m * n) if m * n else 0), m, n, m * n, n
    if x.numel() == 0:
        return 0, m, n, m * n, n
    found = _strided(x, 2)
    rs = x.stride(-2) if m > 1 else n
    if (n > 1 and x.stride(-1) != 1) or found is None or rs < n or (found[0] > 1 and found[1] < (m - 1) * rs + n):
        raise ValueError(f"{what} must be matrices at one stride with contiguous rows")
    batch, bs = found
    return batch, m, n, (bs if batch > 1 else m * rs), rs


def _check_sizes(batch: int, m: int, n: int) -> None:
    """The C ABI's limits, before there is a call."""
    if m > 1 << 20 or n > 1 << 20:
        raise ValueError("m and n must be in [0, 2^20]")
    if batch > 65535:
        raise ValueError("batch must be at most 65535")


_FULL_PRODUCTS = 0x100  # SE_FULL_PRODUCTS


def _muon_code(x, precise: bool) -> int:
    return _code(x.dtype) | (_FULL_PRODUCTS if precise else 0)


def _muon_work(x, code: int, batch: int, m: int, n: int):
    nbytes = _workspace_bytes("se_muon_workspace", code, batch, m, n)
    return _bytes(x, nbytes), nbytes


def orthogonalize(update, steps: int = 5, eps: float = 1e-7, precise: bool = False):
    """Newton-Schulz orthogonalisation of update [..., m, n] (float32, float16
    or bfloat16), as the Muon optimizer applies it: X = U / (|U| + eps), then
    `steps` times X = 3.4445 X + (-4.7750 A + 2.0315 A A) X with A = X X^T
    (from the smaller side). Leading axes are a batch of separate matrices.
    Returns a new tensor of update's shape and dtype. A bfloat16 result comes
    from products of 11-bit values, within about its own rounding; with
    `precise` from products of 22 bits, as float32 and float16 results do, at
    about three times the matrix work."""
    u = _cuda_tensor(update, "update")
    batch, m, n, bs, rs = _matrices(u, "update")
    out = _like(u)
    code = _muon_code(u, precise)
    work, nbytes = _muon_work(u, code, batch, m, n)
    N.check(_entry("se_orthogonalize")(code, u.data_ptr(), batch, m, n, bs, rs, int(steps), float(eps),
                                       out.data_ptr(), work.data_ptr(), nbytes, u.device.index, _stream(u)))
    return out


def _span(x):
    """First and last byte of x's storage range that its elements reach."""
    size = sum((s - 1) * st for s, st in zip(x.shape, x.stride())) + 1
    return x.data_ptr(), x.data_ptr() + size * x.element_size()


def muon_step(weight, grad, momentum, lr: float = 0.02, beta: float = 0.95, weight_decay: float = 0.0,
              nesterov: bool = True, steps: int = 5, eps: float = 1e-7, scale: float | None = None,
              precise: bool = False) -> None:
    """One Muon step of weight [..., m, n], in place (outside autograd):

        momentum = beta momentum + grad
        U = grad + beta momentum if nesterov else momentum
        weight = (1 - lr weight_decay) weight - lr scale orthogonalize(U)

    momentum is float32 of weight's shape; grad has weight's dtype or float32.
    scale is sqrt(max(1, m / n)) unless given, `precise` as in orthogonalize
    (for bfloat16 weights). The three lie in memory of their
    own: ranges that overlap, slices of one tensor among them, are refused."""
    w, g, mom = (_cuda_tensor(t, what) for t, what in ((weight, "weight"), (grad, "grad"), (momentum, "momentum")))
    torch = torch_mod()
    for t, what in ((g, "grad"), (mom, "momentum")):
        _same_device(w, t, what)
        if t.shape != w.shape:
            raise ValueError(f"{what} must have weight's shape")
    if mom.dtype != torch.float32:
        raise ValueError("momentum must be float32")
    if g.dtype != w.dtype and g.dtype != torch.float32:
        raise ValueError("grad must have weight's dtype or float32")
    batch, m, n, wbs, wrs = _matrices(w, "weight")
    _, _, _, gbs, grs = _matrices(g, "grad")
    _, _, _, mbs, mrs = _matrices(mom, "momentum")
    if w.numel():
        spans = sorted(_span(t) for t in (w, g, mom))
        if spans[0][1] > spans[1][0] or spans[1][1] > spans[2][0]:
            raise ValueError("weight, grad and momentum must not share memory")
    if scale is None:
        scale = math.sqrt(max(1.0, m / n)) if n else 1.0
    code = _muon_code(w, precise)
    work, nbytes = _muon_work(w, code, batch, m, n)
    N.check(_entry("se_muon_step")(code, _code(g.dtype), w.data_ptr(), wbs, wrs, g.data_ptr(), gbs, grs,
                                   mom.data_ptr(), mbs, mrs, batch, m, n, float(lr), float(beta), float(weight_decay),
                                   float(scale), int(bool(nesterov)), int(steps), float(eps), work.data_ptr(), nbytes,
                                   w.device.index, _stream(w)))
    # written behind autograd's back: a graph that saved either notices
    torch.autograd.graph.increment_version([t for t in (w, mom) if not t.is_inference()])
