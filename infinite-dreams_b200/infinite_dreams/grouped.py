"""Products grouped by expert as a differentiable function.

``grouped_linear`` runs ``infinite_dreams_ext.grouped_gemm`` forward and, for
the gradients, the same kernel on the transposed weights (dx) and
``grouped_gemm_wgrad`` (dweight).  Nothing is synchronised with the host, so a
training step can be captured into a CUDA graph.
"""
from __future__ import annotations

import torch

from . import infinite_dreams_ext as ext


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets):
        ctx.save_for_backward(x, weight, offsets)
        return ext.grouped_gemm(x, weight, offsets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, offsets = ctx.saved_tensors
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = ext.grouped_gemm(dy, weight.transpose(1, 2), offsets)
        if ctx.needs_input_grad[1]:
            E, K, N = weight.shape
            if weight.stride(1) == 1 and weight.stride(2) != 1:   # stored N x K: so is its gradient
                out = torch.empty((E, N, K), dtype=dy.dtype, device=dy.device).transpose(1, 2)
            else:
                out = None
            dw = ext.grouped_gemm_wgrad(x, dy, offsets, out=out)
        return dx, dw, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """y[r] = x[r] @ weight[e] for the rows offsets[e] <= r < offsets[e + 1], differentiable in x and weight.

    x is [T, K] with its rows sorted by group, weight [E, K, N] (row-major or a
    transposed view), offsets E + 1 row numbers on the device, as for
    ``infinite_dreams_ext.grouped_gemm``.  Rows outside the groups give zeros
    and receive zero gradients; an empty group's weight gradient is zero.
    It can be differentiated once.
    """
    if ext._fast is not None:
        return ext._fast.grouped_linear(x, weight, offsets)
    return _GroupedLinear.apply(x, weight, offsets)


__all__ = ["grouped_linear"]
