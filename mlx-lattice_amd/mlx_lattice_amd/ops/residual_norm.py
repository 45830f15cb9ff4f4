"""The junction of two parts of a block: gated residual sum and norms,
differentiable in the rows and the vectors (no reference counterpart)."""

from __future__ import annotations

import torch

from mlx_lattice_amd._native import ext
from mlx_lattice_amd.core import SparseTensor

__all__ = ['residual_norm']


def residual_norm(x: SparseTensor | torch.Tensor,
                  residual: SparseTensor | torch.Tensor,
                  weight: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, *,
                  gate: torch.Tensor | None = None, scale: float = 1.0,
                  post_norm: bool = False,
                  post_weight: torch.Tensor | None = None,
                  post_bias: torch.Tensor | None = None, rms: bool = False,
                  eps: float = 1e-5, active_rows: torch.Tensor | None = None
                  ) -> tuple[SparseTensor, SparseTensor] | tuple[
                      torch.Tensor, torch.Tensor]:
    """``(sum, normed)`` of what a part of a block gives, ``x``, and its
    residual stream, two sparse tensors or ``(N, C)`` rows::

        part   = norm(x) * post_weight + post_bias   (post_norm; else x)
        sum    = residual + scale * gate * part
        normed = norm(sum) * weight + bias

    where ``norm`` is over the channels of a row, ``(z - mean) / sqrt(var +
    eps)``, or ``z / sqrt(mean(z ** 2) + eps)`` with ``rms``.  ``sum`` is
    rounded to the rows' dtype first, and ``normed`` is of what it holds, as an
    addition and :func:`layer_norm` give it.  The vectors have shape ``(C,)``
    and the rows' dtype (``None``: 1 for weights and gate, 0 for biases).  Rows at and past the device count ``active_rows`` (a sparse
    tensor's own) become zeros and take no part in the gradients.  Statistics
    and sums are float32; float32, float16 and bfloat16 rows.
    """
    if isinstance(x, SparseTensor):
        if not isinstance(residual, SparseTensor):
            raise ValueError('a sparse tensor needs a sparse residual.')
        if not x.same_coords(residual):
            raise ValueError('sparse tensor coordinates must match.')
        if active_rows is not None:
            raise ValueError('a sparse tensor has its own active_rows.')
        rows = residual_norm(
            x.feats, residual.feats, weight, bias, gate=gate, scale=scale,
            post_norm=post_norm, post_weight=post_weight, post_bias=post_bias,
            rms=rms, eps=eps, active_rows=x.active_rows)
        return x.replace(feats=rows[0]), x.replace(feats=rows[1])
    if isinstance(residual, SparseTensor):
        raise ValueError('a sparse residual needs a sparse tensor.')
    vectors = (weight, bias, gate, post_weight, post_bias)
    how = (vectors, scale, post_norm, rms, eps, active_rows)
    if torch.is_grad_enabled():
        for t in (x, residual, *vectors):
            if t is not None and t.requires_grad:
                return ext.residual_norm_node(x, residual, *how)
    return ext.residual_norm(x, residual, *how, False)[:2]
