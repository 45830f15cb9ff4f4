"""Dropout from a counter-based generator, whose mask is never stored (no
reference counterpart)."""

from __future__ import annotations

import torch

from mlx_lattice_amd._native import ext
from mlx_lattice_amd.core import SparseTensor

__all__ = ['dropout']

_WORD = 0xFFFFFFFFFFFFFFFF


def dropout(x: SparseTensor | torch.Tensor, p: float, *, seed: int,
            offset: int = 0,
            residual: SparseTensor | torch.Tensor | None = None
            ) -> SparseTensor | torch.Tensor:
    """Each value of ``x`` dropped with probability ``p`` or divided by
    ``1 - p``, and ``residual`` added.

    The mask is a function of ``seed``, ``offset`` (64 bits each) and the
    value's place in row-major order: element ``e`` is kept when word ``e % 4``
    of Philox 4x32-10 over the counter ``(e // 4, offset)`` and the key
    ``seed`` is at least ``round(p * 2**32)``.  The gradient makes it again, so
    nothing but the two numbers is kept; a layer counts ``offset`` up call by
    call.  A captured graph repeats its mask.
    """
    if isinstance(x, SparseTensor):
        if isinstance(residual, SparseTensor):
            if not x.same_coords(residual):
                raise ValueError('sparse tensor coordinates must match.')
            residual = residual.feats
        return x.replace(feats=dropout(x.feats, p, seed=seed, offset=offset,
                                       residual=residual))
    if isinstance(residual, SparseTensor):
        raise ValueError('a sparse residual needs a sparse tensor.')
    if not 0.0 <= p <= 1.0:
        raise ValueError('p must be between 0 and 1.')
    threshold = round(p * 2 ** 32)
    scale = 0.0 if p == 1.0 else 1.0 / (1.0 - p)
    key = (int(seed) & _WORD, int(offset) & _WORD, threshold, scale)
    if torch.is_grad_enabled() and (
            x.requires_grad or residual is not None and residual.requires_grad):
        return ext.dropout_node(x, residual, *key)
    return ext.dropout(x, residual, *key)
