"""Layer norm of feature rows, differentiable in the rows, the weight and the
bias (no reference counterpart)."""

from __future__ import annotations

import torch

from mlx_lattice_amd._native import ext
from mlx_lattice_amd.core import SparseTensor

__all__ = ['layer_norm']


def layer_norm(x: SparseTensor | torch.Tensor,
               weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, *, eps: float = 1e-5,
               active_rows: torch.Tensor | None = None
               ) -> SparseTensor | torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the channels of
    each row of a sparse tensor or of ``(N, C)`` rows.

    ``weight`` and ``bias`` have shape ``(C,)`` and the rows' dtype (``None``:
    1 and 0).  Rows at and past the device count ``active_rows`` (a sparse
    tensor's own) become zeros and take no part in the gradients.  Statistics
    and sums are float32; float32, float16 and bfloat16 rows.
    """
    if isinstance(x, SparseTensor):
        if active_rows is not None:
            raise ValueError('a sparse tensor has its own active_rows.')
        return x.replace(feats=layer_norm(x.feats, weight, bias, eps=eps,
                                          active_rows=x.active_rows))
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, eps, active_rows)
    return ext.layer_norm(x, weight, bias, eps, active_rows, False)[0]


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, active_rows):
        y, statistics = ext.layer_norm(x, weight, bias, eps, active_rows, True)
        ctx.save_for_backward(x, weight, statistics, active_rows)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        x, weight, statistics, active_rows = ctx.saved_tensors
        _, need_weight, need_bias, _, _ = ctx.needs_input_grad
        grad_x, grad_weight, grad_bias = ext.layer_norm_grad(
            grad_y, x, weight, statistics, active_rows, need_weight, need_bias)
        return (grad_x, grad_weight if need_weight else None,
                grad_bias if need_bias else None, None, None)
