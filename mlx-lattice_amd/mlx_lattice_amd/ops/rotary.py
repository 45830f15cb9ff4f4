"""Rotary positions of several axes, for heads of rows with voxel coordinates
(no reference counterpart)."""

from __future__ import annotations

from collections.abc import Sequence

import torch

from mlx_lattice_amd._native import ext

__all__ = ['rotary_frequencies', 'rotary_positions']


def rotary_frequencies(dims: Sequence[int], base: float = 10000.0, *,
                       device=None) -> torch.Tensor:
    """Radians a unit of position, ``base ** (-2 i / dims[a])`` for pair ``i``
    of axis ``a``: float64 ``(sum(dims) / 2,)``, made once for a layer."""
    if any(d < 0 or d % 2 for d in dims):
        raise ValueError('rotary dims must be even and non-negative.')
    if not base > 0:
        raise ValueError('base must be positive.')
    return torch.tensor([base ** (-2.0 * i / d) for d in dims
                         for i in range(d // 2)],
                        dtype=torch.float64, device=device)


def rotary_positions(x: torch.Tensor, positions: torch.Tensor,
                     frequencies: torch.Tensor, *, dims: Sequence[int],
                     interleaved: bool = False) -> torch.Tensor:
    """Turn the channel pairs of ``x`` ``(N, heads, dim)`` by the row's
    ``positions`` ``(N, axes)`` (int32, as ``coords[:, 1:]``, or float32).

    The first ``sum(dims)`` channels of a head are cut into one section per
    axis (1 to 4), ``dims[a]`` channels each; pair ``i`` of a section turns by
    ``position * frequency`` radians, the other channels stay.  A pair is
    channels ``(i, i + dims[a] / 2)`` of its section, or ``(2 i, 2 i + 1)``
    with ``interleaved``.  ``x`` may be a slice of packed rows (any row and
    head stride).  Differentiable in ``x``; the positions get no gradient.
    """
    dims = [int(d) for d in dims]
    if torch.is_grad_enabled() and x.requires_grad:
        return ext.rotary_positions_node(x, positions, frequencies, dims,
                                         interleaved)
    return ext.rotary_positions(x, positions, frequencies, dims, interleaved,
                                False)
