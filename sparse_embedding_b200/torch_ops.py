"""PyTorch autograd wrappers: the store's embedding bag (the forward is
EmbeddingStore.embedding_bag, the backward accumulates the pooled gradients
into the store, EmbeddingStore.embedding_bag_backward; the parameters are
updated by EmbeddingStore.optimizer_step, outside autograd), and the layer
normalisation of its rows (dense.layer_norm).
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
