"""Attention over a sliding window of rows, with first rows that stay visible
(no reference counterpart)."""

from __future__ import annotations

import torch

from mlx_lattice_amd._native import ext
from mlx_lattice_amd.core import SparseTensor

__all__ = ['batch_offsets', 'window_attention']

_ALL = 2 ** 31 - 1


def batch_offsets(x: SparseTensor, batches: int | None = None) -> torch.Tensor:
    """Row offsets ``(B + 1,)`` of the scans of ``x``, int32 on its device.

    From ``batch_counts`` where ``x`` has them; else its active rows hold the
    scans 0 to ``batches - 1`` (a strided conv's output has no counts).  Without
    ``batches`` their number is read from the last active row's batch column,
    which waits for the device; layers of a level can share the offsets.  Rows
    of a scan are adjacent and scans in order, as ``sparse_collate`` lays them
    and strided convs keep them.  Rows past the active ones are in no scan.
    """
    counts = x.batch_counts
    if counts is not None and len(counts) > 1:
        offsets = [0]
        for count in counts:
            offsets.append(offsets[-1] + count)
        return torch.minimum(_on_device(offsets, x.device), x.active_rows)
    if batches is None:
        batches = 1 if counts is not None else _scans(x)
    if batches < 1:
        raise ValueError('batches must be positive.')
    if counts is not None or batches == 1:
        return torch.cat([torch.zeros_like(x.active_rows), x.active_rows])
    rows = torch.arange(x.capacity, device=x.device)
    scan = torch.where(rows < x.active_rows, x.batch_indices, batches)
    return torch.searchsorted(
        scan, torch.arange(batches + 1, dtype=scan.dtype, device=x.device),
        out_int32=True)


def _refuse_capture(device: torch.device, what: str) -> None:
    if device.type == 'cuda' and torch.cuda.is_current_stream_capturing():
        raise ValueError(f'{what}, which a captured graph cannot: give '
                         'offsets made before.')


def _on_device(offsets: list[int], device: torch.device) -> torch.Tensor:
    """Copied from pinned memory: the host does not wait for the device."""
    _refuse_capture(device, 'offsets of batch_counts are copied from the host')
    return torch.tensor(offsets, dtype=torch.int32,
                        pin_memory=device.type == 'cuda').to(
                            device, non_blocking=True)


def _scans(x: SparseTensor) -> int:
    if x.capacity == 0:
        return 1
    _refuse_capture(x.device, 'without batch_counts the number of scans is '
                    'read from the device')
    last = (x.active_rows - 1).clamp(min=0).long()
    scan = torch.where(x.active_rows > 0, x.batch_indices[last], 0)
    return max(0, int(scan)) + 1


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                     offsets: torch.Tensor,
                     key_offsets: torch.Tensor | None = None,
                     key_lengths: torch.Tensor | None = None,
                     left: int | None = None, right: int | None = None,
                     sinks: int = 0, scale: float | None = None
                     ) -> torch.Tensor:
    """Softmax attention of packed sequences, ``(queries, heads, dim)``.

    ``q`` has shape ``(queries, heads, dim)``, ``k`` and ``v`` ``(keys,
    kv_heads, dim)`` with ``heads`` a multiple of ``kv_heads``; each may be a
    slice of packed rows.  float32, float16 or bfloat16, ``dim`` up to 128;
    ``scale`` is ``dim ** -0.5`` by default.

    Sequence ``s`` holds the query rows ``offsets[s] : offsets[s + 1]`` and the
    key rows of ``key_offsets`` (``offsets`` by default), of which
    ``key_lengths[s]`` are filled (all by default): a cache of ``B`` sequences
    of ``L`` rows has ``key_offsets = arange(B + 1) * L``.  All three are int32
    on the device and are not read back; offsets must not decrease, and are
    clamped to the rows there are.

    Query ``i`` of ``nq``, in a sequence of ``nk`` keys, has position ``p = i +
    nk - nq``: queries sit at the end of the keys.  It sees key ``j`` where
    ``j <= p + right`` and either ``j >= p - left`` or ``j < sinks``; ``None``
    is no bound, ``right=0`` is causal.  A query that sees nothing gives zeros
    and no gradient, as do rows in no sequence; what a query does not see never
    reaches it, be it infinite or NaN.

    Differentiable in ``q``, ``k`` and ``v``; the gradients of a shared key
    head are summed over its query heads, in a fixed order.
    """
    left, right = (_ALL if b is None else int(b) for b in (left, right))
    if scale is None:  # a head without channels is refused below
        scale = max([1, *q.shape[-1:]]) ** -0.5
    if key_offsets is None:
        key_offsets = offsets
    layout = (offsets, key_offsets, key_lengths)
    window = (left, right, int(sinks), float(scale))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad
                                    or v.requires_grad):
        return ext.window_attention_node(q, k, v, *layout, *window)
    return ext.window_attention(q, k, v, *layout, *window, False)[0]
