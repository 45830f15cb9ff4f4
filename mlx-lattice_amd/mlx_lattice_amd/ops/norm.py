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
    if torch.is_grad_enabled() and (
            x.requires_grad or weight is not None and weight.requires_grad
            or bias is not None and bias.requires_grad):
        return ext.layer_norm_node(x, weight, bias, eps, active_rows)
    return ext.layer_norm(x, weight, bias, eps, active_rows, False)[0]
