"""PyTorch autograd wrappers: the store's embedding bag (the forward is
EmbeddingStore.embedding_bag, the backward accumulates the pooled gradients
into the store, EmbeddingStore.embedding_bag_backward; the parameters are
updated by EmbeddingStore.optimizer_step, outside autograd), the layer
normalisation of its rows (dense.layer_norm), and an optimizer for the dense
matrices behind them (dense.muon_step).
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import dense


class EmbeddingBagFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, anchor, store, keys, offsets, dim, insert):
        ctx.store, ctx.keys, ctx.offsets = store, keys, offsets
        return store.embedding_bag(keys, offsets, dim, insert=insert)

    @staticmethod
    def backward(ctx, grad):
        ctx.store.embedding_bag_backward(ctx.keys, ctx.offsets, grad.contiguous())
        return None, None, None, None, None, None


def embedding_bag(store, keys: torch.Tensor, offsets: torch.Tensor, dim: int, insert: bool = True) -> torch.Tensor:
    """Sum-pooled bag rows [num_bags, dim] that take part in autograd: calling
    backward on a loss built from them accumulates the bags' gradients into
    `store` for its next optimizer_step."""
    anchor = torch.empty(0, device=keys.device, requires_grad=True)
    return EmbeddingBagFunction.apply(anchor, store, keys, offsets, dim, insert)


class LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = dense.layer_norm(x, weight, bias, eps=eps, return_stats=True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.with_bias = bias is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = dense.layer_norm_backward(grad.contiguous(), x, mean, rstd, weight, with_bias=ctx.with_bias)
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """dense.layer_norm that takes part in autograd: gradients of x, weight and
    bias by dense.layer_norm_backward. An x whose rows are not at one stride is
    copied first."""
    if x.is_cuda and not x.is_contiguous():
        try:
            dense._rows(x, "x")
        except ValueError:
            x = x.contiguous()
    return LayerNormFunction.apply(x, weight, bias, eps)


class Muon(torch.optim.Optimizer):
    """Muon for the dense matrices of a model, next to the store's own row
    optimizers: each parameter [..., m, n] takes dense.muon_step with a float32
    momentum (leading axes are separate matrices: stacked layers or experts; a
    convolution's [out, in, 3, 3] is out x in matrices of 3 x 3). Vectors (biases,
    normalisation weights) need another optimizer; they, parameters without
    contiguous rows (transposed ones) and batches of more than 65,535 matrices
    are refused when they are added. A captured step keeps the lr and the other
    values of its capture; the first step, which makes the momentum, is not
    captured (RuntimeError). `precise`:
    full products for bfloat16 parameters too (dense.orthogonalize)."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, weight_decay: float = 0.0,
                 nesterov: bool = True, steps: int = 5, eps: float = 1e-7, precise: bool = False):
        super().__init__(params, dict(lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov,
                                      steps=steps, eps=eps, precise=precise))

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("precise", False)  # states from before it was there

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        try:
            for p in self.param_groups[-1]["params"]:
                if p.dim() < 2:
                    raise ValueError("Muon steps matrices: every parameter needs at least two dimensions")
                dense._check_sizes(*dense._matrices(p, "every parameter")[:3])
        except ValueError:  # the group is not taken, and the optimizer goes on with those that it had
            self.param_groups.pop()
            raise

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        # torch casts an optimizer's state to its parameters' dtype: put the float32 momentum back
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        own = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, own):
            buffer = state_dict["state"].get(i, {}).get("momentum_buffer")
            if buffer is not None:
                self.state[p]["momentum_buffer"] = buffer.to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if any(p.grad is not None and p.grad.is_sparse for group in self.param_groups for p in group["params"]):
            raise ValueError("Muon needs dense gradients")  # before any parameter is stepped
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if "momentum_buffer" not in state:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("Muon's first step cannot be captured: a replayed graph would zero the "
                                           "momentum every time; step once before the capture")
                    state["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                dense.muon_step(p, p.grad.contiguous(), state["momentum_buffer"], lr=group["lr"],
                                beta=group["momentum"], weight_decay=group["weight_decay"],
                                nesterov=group["nesterov"], steps=group["steps"], eps=group["eps"],
                                precise=group["precise"])
        return loss
